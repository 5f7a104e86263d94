// Host side of the split products (split_mm.cuh): the workspace of split matrices, the choice of
// tile and contraction split, and the gated feed-forward block and orthogonalised update that are
// built from them. Part of the library's one translation unit (mfk_api.cu includes it).
#pragma once

namespace {

constexpr int kXKinds = 72;  // kernel instantiations (and cluster sizes) with per-device set-up

struct XDevice {
    bool ready[kXKinds] = {};
    int slots[kXKinds] = {};  // CTAs (or pairs) resident at once
};
XDevice g_xdevices[kMaxDevices];

// A matrix held split in the workspace.
struct XMat {
    int64_t rows = 0, cols = 0, batch = 1;  // as stored
    int rb = 0, cb = 0;                     // blocks
    int64_t first = 0;                      // index of its first block in the workspace
    int64_t inv = 0;                        // and of its first 1/s
    bool by_row = false;                    // a scale for every row of a block
    bool transposed = false;                // stored as the logical matrix's transpose

    int64_t blocks() const { return static_cast<int64_t>(rb) * cb; }
};

// One stream-ordered allocation: all split blocks, their 1/s, sums of squares, and what else a call
// asks for.
struct XWorkspace {
    cudaStream_t stream;
    uint8_t* base = nullptr;
    uint8_t* blocks = nullptr;
    float* inv = nullptr;
    double* sumsq = nullptr;
    float* extra = nullptr;
    int64_t total_blocks = 0, total_inv = 0;
    CUtensorMap mk, mm;
    int dev = 0;
    DeviceInfo* info = nullptr;

    explicit XWorkspace(cudaStream_t s) : stream(s) {}
    XWorkspace(const XWorkspace&) = delete;
    XWorkspace& operator=(const XWorkspace&) = delete;
    ~XWorkspace() {
        if (base != nullptr) cudaFreeAsync(base, stream);
    }
};

XMat x_mat(XWorkspace& ws, int64_t rows, int64_t cols, int64_t batch = 1, bool by_row = false) {
    XMat m;
    m.by_row = by_row;
    m.rows = rows;
    m.cols = cols;
    m.batch = batch;
    m.rb = static_cast<int>((rows + mfk::kXBlk - 1) / mfk::kXBlk);
    m.cb = static_cast<int>((cols + mfk::kXBlk - 1) / mfk::kXBlk);
    m.first = ws.total_blocks;
    m.inv = ws.total_inv;
    ws.total_blocks += m.blocks() * batch;
    ws.total_inv += m.blocks() * batch * (by_row ? mfk::kXBlk : 1);
    return m;
}

// Whether (rs, cs) of a rows x cols matrix has a unit stride, and which.
bool x_orientation(int64_t rows, int64_t cols, int64_t rs, int64_t cs, bool* transposed) {
    *transposed = false;
    if (cs == 1 || cols <= 1) return true;
    if (rs == 1 || rows <= 1) {
        *transposed = true;
        return true;
    }
    return false;
}

int x_allocate(XWorkspace& ws, size_t extra_floats) {
    if (ws.total_blocks > (int64_t(1) << 25)) return MFK_ERR_UNSUPPORTED;  // 2 TB of blocks
    const size_t block_bytes = static_cast<size_t>(ws.total_blocks) * mfk::kXBlockBytes;
    const size_t inv_bytes = (static_cast<size_t>(ws.total_inv) * 4 + 255) / 256 * 256;
    const size_t sum_bytes = (static_cast<size_t>(ws.total_blocks) * 8 + 255) / 256 * 256;
    const size_t total = block_bytes + inv_bytes + sum_bytes + extra_floats * 4 + 1024;
    MFK_CUDA(cudaMallocAsync(reinterpret_cast<void**>(&ws.base), total, ws.stream));
    uint8_t* p = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ws.base) + 1023) &
                                            ~static_cast<uintptr_t>(1023));
    ws.blocks = p;
    p += block_bytes;
    ws.inv = reinterpret_cast<float*>(p);
    p += inv_bytes;
    ws.sumsq = reinterpret_cast<double*>(p);
    p += sum_bytes;
    ws.extra = reinterpret_cast<float*>(p);
    // The blocks as 2 KB lines of 256 eight-byte units. K-major stages take 8 whole lines,
    // MN-major ones the same 1 KB of 16 lines.
    auto fn = encode_fn();
    if (fn == nullptr) return MFK_ERR_CUDA;
    const cuuint64_t dims[2] = {256, static_cast<cuuint64_t>(ws.total_blocks) * mfk::kXBlockLines};
    const cuuint64_t strides[1] = {mfk::kXLineBytes};
    const cuuint32_t box_k[2] = {256, 8}, box_m[2] = {128, 16}, estr[2] = {1, 1};
    for (int i = 0; i < 2; ++i) {
        if (fn(i ? &ws.mm : &ws.mk, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, 2, ws.blocks, dims, strides,
               i ? box_m : box_k, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return MFK_ERR_CUDA;
    }
    return MFK_OK;
}

// Adds logical matrix (rows x cols at p, strides rs, cs; batch matrices bs apart) to the split
// pass and to the workspace. False: neither stride is 1.
bool x_source(XWorkspace& ws, mfk::XSources& list, XMat* out, const float* p, int64_t rows,
              int64_t cols, int64_t rs, int64_t cs, int64_t batch = 1, int64_t bs = 0,
              bool by_row = false) {
    bool t = false;
    if (!x_orientation(rows, cols, rs, cs, &t) || (by_row && t)) return false;
    *out = x_mat(ws, t ? cols : rows, t ? rows : cols, batch, by_row);
    out->transposed = t;
    mfk::XSource& s = list.s[list.count++];
    s = mfk::XSource{};
    s.src = p;
    s.rs = t ? cs : rs;
    s.bs = batch > 1 ? bs : 0;
    s.rows = static_cast<int>(out->rows);
    s.cols = static_cast<int>(out->cols);
    s.rb = out->rb;
    s.cb = out->cb;
    s.by_row = by_row ? 1 : 0;
    s.vec = aligned16(p) && (s.rs % 4 == 0 || out->rows <= 1) && s.bs % 4 == 0;
    return true;
}

int x_split(XWorkspace& ws, mfk::XSources& list, const XMat* const* mats, bool sums) {
    int64_t at = 0;
    for (int i = 0; i < list.count; ++i) {
        mfk::XSource& s = list.s[i];
        s.first = static_cast<int>(at);
        s.data = ws.blocks + mats[i]->first * mfk::kXBlockBytes;
        s.inv = ws.inv + mats[i]->inv;
        s.sumsq = sums ? ws.sumsq + mats[i]->first : nullptr;
        at += mats[i]->blocks() * mats[i]->batch;
    }
    if (at == 0) return MFK_OK;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(static_cast<unsigned>(at), 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = ws.stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = list.s[0].live != nullptr ? 1 : 0;  // beside the launch that finds the live rows
    MFK_CUDA(cudaLaunchKernelEx(&cfg, mfk::split_blocks_kernel, list));
    g_launches.fetch_add(1);
    return MFK_OK;
}

// Matrix m as an operand whose contraction runs over its logical columns, or rows.
mfk::XOperand x_operand(const XWorkspace& ws, const XMat& m, bool over_columns, bool sym = false) {
    mfk::XOperand o{};
    o.line0 = static_cast<int>(m.first * mfk::kXBlockLines);
    o.ldb = m.cb;
    o.bstride = m.batch > 1 ? static_cast<int>(m.blocks()) : 0;
    o.flip = over_columns == m.transposed ? 1 : 0;
    o.sym = sym ? 1 : 0;
    o.by_row = m.by_row ? 1 : 0;
    o.inv = ws.inv + m.inv;
    return o;
}

mfk::XOut x_out(const XWorkspace& ws, const XMat& m) {
    mfk::XOut o{};
    o.data = ws.blocks + m.first * mfk::kXBlockBytes;
    o.inv = ws.inv + m.inv;
    o.ldb = m.cb;
    o.bstride = m.batch > 1 ? static_cast<int>(m.blocks()) : 0;
    return o;
}

// CTAs, pairs or clusters of `cluster` CTAs of a kernel that the device holds at once.
template <int CG, int NB, int EPI, bool SPL>
int x_slots(XWorkspace& ws, int kind, int cluster, int* slots) {
    using C = mfk::XConfig<CG, NB>;
    auto kernel = mfk::split_mm_kernel<CG, NB, EPI, SPL>;
    std::lock_guard<std::mutex> lock(g_mutex);
    XDevice& d = g_xdevices[ws.dev];
    if (!d.ready[kind]) {
        MFK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      C::kSmemBytes));
        int n = ws.info->sm_count / cluster;
        if (cluster > 1) {
            cudaLaunchConfig_t cfg = {};
            cudaLaunchAttribute attr[1];
            cfg.blockDim = dim3(mfk::kXThreads, 1, 1);
            cfg.gridDim = dim3(static_cast<unsigned>(n * cluster), 1, 1);
            cfg.dynamicSmemBytes = C::kSmemBytes;
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
            attr[0].val.clusterDim.y = 1;
            attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int clusters = 0;
            if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess &&
                clusters > 0)
                n = clusters;
            cudaGetLastError();
        }
        d.slots[kind] = n;
        d.ready[kind] = true;
    }
    *slots = d.slots[kind];
    return MFK_OK;
}

// Time of a launch in SM cycles: whole waves of tiles, and the part of the epilogue that no product
// hides. A chunk of 128 takes 24 MMAs, of 128 cycles for a pair's 256 x 256, which it reaches (its
// 128 KB per CTA come at 42 bytes a cycle). One CTA's 128 x 128 would take 24 x 64, but 128 KB in
// that time is more than an SM gets from L2: 2500 measured (4 to 50 chunks), 4200 for 128 x 256.
// Sharing a contraction costs 9000 cycles (128 x 128) or 17000 per wave (1024 x 1024 over a depth
// of 1024: 15.6 us by clusters of 3 single CTAs, 24.5 us by clusters of 4 pairs).
double x_cost(int64_t tiles, int slots, double chunk, int kc, double epilogue) {
    const int64_t waves = (tiles + slots - 1) / slots;
    return static_cast<double>(waves) * (kc * chunk + epilogue);
}

template <int CG, int NB, int EPI, bool SPL>
int x_launch(XWorkspace& ws, mfk::XArgs& g, int slots, int64_t batch, int64_t tm, int64_t tn,
             int64_t tiles, int splits) {
    using C = mfk::XConfig<CG, NB>;
    auto kernel = mfk::split_mm_kernel<CG, NB, EPI, SPL>;
    g.tiles_m = static_cast<int>(tm);
    g.tiles_n = static_cast<int>(tn);
    g.tiles = static_cast<int>(tiles);
    g.splits = splits;
    g.units = static_cast<int>(tiles * batch) * splits;
    const int cluster = CG * splits;
    const int units = SPL ? g.units : std::min(g.units, slots);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.blockDim = dim3(mfk::kXThreads, 1, 1);
    cfg.gridDim = dim3(static_cast<unsigned>(units * CG), 1, 1);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = ws.stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    {
        TimedLaunch timed(ws.stream);
        MFK_CUDA(cudaLaunchKernelEx(&cfg, kernel, ws.mk, ws.mm, g));
    }
    g_launches.fetch_add(1);
    return MFK_OK;
}

// Launches out[mb x nb blocks] = A B over kc0 (+ kc1) chunks. k0, k1: the segments' depths. The
// third product of kXWeights has the others' blocks, or those of their transposes: as many tiles.
template <int EPI>
int x_product(XWorkspace& ws, mfk::XArgs& g, int64_t k0, int64_t k1, int64_t batch) {
    constexpr int kNb1 = EPI == mfk::kXGated ? 2 : 1;  // the one-CTA kernel's blocks per tile
    g.kc0 = static_cast<int>((k0 + mfk::kXBlk - 1) / mfk::kXBlk);
    g.kc = g.kc0 + static_cast<int>((k1 + mfk::kXBlk - 1) / mfk::kXBlk);
    g.last0 = (k0 - 1) % mfk::kXBlk < 64 ? 1 : 2;
    g.last1 = k1 > 0 ? ((k1 - 1) % mfk::kXBlk < 64 ? 1 : 2) : g.last0;
    const int per_tile_n = EPI == mfk::kXGated ? 1 : 2;
    const int64_t tm2 = (g.mb + 1) / 2, tn2 = (g.nb + per_tile_n - 1) / per_tile_n;
    const int64_t tm1 = g.mb, tn1 = g.nb;
    const int64_t tiles2 = g.sym ? tm2 * (tm2 + 1) / 2 : tm2 * tn2;
    const int64_t tiles1 = g.sym ? tm1 * (tm1 + 1) / 2 : tm1 * tn1;
    if (tiles1 * batch > (int64_t(1) << 26)) return MFK_ERR_UNSUPPORTED;
    // What the epilogue adds to a wave, measured at 8 chunks. The backward one has three outputs
    // and two inputs, and no registers to spare beside a pair's 128 sums a thread: 4096 x 1024 x
    // 4096 takes 163 us by pairs and 154 by single CTAs (at 32 chunks the pairs win).
    constexpr double kEpi1 = EPI == mfk::kXGatedBwd ? 10000.0 : EPI == mfk::kXGated ? 7000.0
                                                                                    : 3000.0;
    constexpr double kEpi2 = EPI == mfk::kXGatedBwd ? 30000.0 : EPI == mfk::kXGated ? 7000.0
                                                                                    : 6000.0;
    // 256 x 256 by pairs of CTAs where there are tiles enough, 128-row tiles of one CTA where there
    // are not, and either with the contraction shared by a cluster where that leaves SMs idle.
    int slots = 0, best_slots = 0, pairs = 0, splits = 0, rc = MFK_OK;
    double least = 0.0;
    auto consider = [&](int cta_group, int s, int64_t tiles, double chunk, double epilogue,
                        double exchange) {
        double t = x_cost(tiles * batch, slots, chunk, (g.kc + s - 1) / s, epilogue / s);
        if (s > 1) t += exchange * static_cast<double>((tiles * batch + slots - 1) / slots);
        if (splits == 0 || t < least) {
            least = t;
            pairs = cta_group - 1;
            splits = s;
            best_slots = slots;
        }
    };
    for (int s = 1; s <= 4 && s <= g.kc; ++s) {
        rc = s == 1 ? x_slots<2, 2, EPI, false>(ws, EPI * 12 + s - 1, 2, &slots)
                    : x_slots<2, 2, EPI, true>(ws, EPI * 12 + s - 1, 2 * s, &slots);
        if (rc != MFK_OK) return rc;
        consider(2, s, tiles2, 24 * 128.0, kEpi2, 17000.0);
    }
    for (int s = 1; s <= 8 && s <= g.kc; ++s) {
        rc = s == 1 ? x_slots<1, kNb1, EPI, false>(ws, EPI * 12 + 3 + s, 1, &slots)
                    : x_slots<1, kNb1, EPI, true>(ws, EPI * 12 + 3 + s, s, &slots);
        if (rc != MFK_OK) return rc;
        consider(1, s, tiles1, kNb1 == 2 ? 4200.0 : 2500.0, kEpi1, kNb1 == 2 ? 17000.0 : 9000.0);
    }
    g.third.tiles_m = pairs ? (g.third.mb + 1) / 2 : g.third.mb;
    g.third.tiles_n = pairs ? (g.third.nb + 1) / 2 : g.third.nb;
    if (pairs)
        return splits == 1
                   ? x_launch<2, 2, EPI, false>(ws, g, best_slots, batch, tm2, tn2, tiles2, 1)
                   : x_launch<2, 2, EPI, true>(ws, g, best_slots, batch, tm2, tn2, tiles2, splits);
    return splits == 1
               ? x_launch<1, kNb1, EPI, false>(ws, g, best_slots, batch, tm1, tn1, tiles1, 1)
               : x_launch<1, kNb1, EPI, true>(ws, g, best_slots, batch, tm1, tn1, tiles1, splits);
}

int x_zero(float* out, int64_t rows, int64_t cols, int64_t ld, cudaStream_t stream) {
    if (out == nullptr || rows == 0 || cols == 0) return MFK_OK;
    MFK_CUDA(cudaMemset2DAsync(out, static_cast<size_t>(ld) * 4, 0, static_cast<size_t>(cols) * 4,
                               static_cast<size_t>(rows), stream));
    return MFK_OK;
}

}  // namespace

#include "rows_host.cuh"

namespace {

// ---- the gated feed-forward block ------------------------------------------------------------

constexpr int64_t kXMaxDim = int64_t(1) << 30;  // 32-bit indexes may run a few tiles further

int check_gated(const mfk_gated_ffn_desc* d) {
    if (d == nullptr) return MFK_ERR_INVALID_ARGUMENT;
    if (d->rows < 0 || d->d < 0 || d->f < 0) return MFK_ERR_INVALID_ARGUMENT;
    if (d->activation < MFK_ACT_NONE || d->activation > MFK_ACT_SILU)
        return MFK_ERR_INVALID_ARGUMENT;
    if (d->rows > kXMaxDim || d->d > kXMaxDim || d->f > kXMaxDim) return MFK_ERR_UNSUPPORTED;
    if (d->rows > 0 && d->d > 0 && d->x == nullptr) return MFK_ERR_INVALID_ARGUMENT;
    if (d->d > 0 && d->f > 0 &&
        (d->w_gate == nullptr || d->w_up == nullptr || d->w_down == nullptr))
        return MFK_ERR_INVALID_ARGUMENT;
    return MFK_OK;
}

int64_t gated_saved_floats(int64_t rows, int64_t f) {
    const int64_t blocks = ((rows + 127) / 128) * ((f + 127) / 128);
    return blocks * (2 * 128 * 128 + 4 * 128);
}

// gate and up (and h, when `h` is given) of x: one product whose tiles hold both projections.
int gated_forward(XWorkspace& ws, const mfk_gated_ffn_desc* d, const XMat& x, const XMat& wg,
                  const XMat& wu, const XMat* h, float* saved) {
    mfk::XArgs g{};
    g.a[0] = g.a[1] = x_operand(ws, x, true);
    g.b[0] = x_operand(ws, wg, false);
    g.b[1] = x_operand(ws, wu, false);
    g.mb = static_cast<int>((d->rows + 127) / 128);
    g.nb = static_cast<int>((d->f + 127) / 128);
    g.m = static_cast<int>(d->rows);
    g.n = static_cast<int>(d->f);
    g.act = d->activation;
    if (h != nullptr) {
        g.o[0] = x_out(ws, *h);
        g.store_h = 1;
    }
    g.o[0].ldb = g.nb;
    if (saved != nullptr) {
        const int64_t blocks = static_cast<int64_t>(g.mb) * g.nb;
        g.gate = saved;
        g.up = saved + blocks * 128 * 128;
        g.gmax = saved + blocks * 2 * 128 * 128;
    }
    return x_product<mfk::kXGated>(ws, g, d->d, 0, 1);
}

int run_gated_ffn(const mfk_gated_ffn_desc* d, float* y, int64_t ldy, float* saved,
                  cudaStream_t stream) {
    int rc = check_gated(d);
    if (rc != MFK_OK) return rc;
    if (d->rows > 0 && d->d > 0 && (y == nullptr || ldy < d->d)) return MFK_ERR_INVALID_ARGUMENT;
    if (d->rows == 0 || (d->d == 0 && saved == nullptr)) return MFK_OK;
    if (saved != nullptr && !aligned16(saved)) return MFK_ERR_INVALID_ARGUMENT;
    if (d->d > 1 && d->x_cs != 1) return MFK_ERR_UNSUPPORTED;
    XWorkspace ws(stream);
    rc = current_device(&ws.dev, &ws.info);
    if (rc != MFK_OK) return rc;
    if (d->f == 0 || d->d == 0) {
        if (saved != nullptr && d->f > 0)
            MFK_CUDA(cudaMemsetAsync(saved, 0, gated_saved_floats(d->rows, d->f) * 4, stream));
        return x_zero(y, d->rows, d->d, ldy, stream);
    }
    if (d->rows <= mfk::kRowsMax && saved == nullptr)
        return run_gated_rows(d, y, ldy, ws.info, ws.dev, stream);
    mfk::XSources list{};
    XMat x, wg, wu, wd;
    if (!x_source(ws, list, &x, d->x, d->rows, d->d, d->x_rs, d->x_cs, 1, 0, true) ||
        !x_source(ws, list, &wg, d->w_gate, d->d, d->f, d->w_gate_rs, d->w_gate_cs) ||
        !x_source(ws, list, &wu, d->w_up, d->d, d->f, d->w_up_rs, d->w_up_cs) ||
        !x_source(ws, list, &wd, d->w_down, d->f, d->d, d->w_down_rs, d->w_down_cs))
        return MFK_ERR_UNSUPPORTED;
    if (wg.transposed != wu.transposed) return MFK_ERR_UNSUPPORTED;
    const XMat h = x_mat(ws, d->rows, d->f, 1, true);
    rc = x_allocate(ws, 0);
    if (rc != MFK_OK) return rc;
    const XMat* mats[4] = {&x, &wg, &wu, &wd};
    rc = x_split(ws, list, mats, false);
    if (rc != MFK_OK) return rc;
    rc = gated_forward(ws, d, x, wg, wu, &h, saved);
    if (rc != MFK_OK) return rc;
    mfk::XArgs g{};
    g.a[0] = g.a[1] = x_operand(ws, h, true);
    g.b[0] = g.b[1] = x_operand(ws, wd, false);
    g.mb = h.rb;
    g.nb = static_cast<int>((d->d + 127) / 128);
    g.m = static_cast<int>(d->rows);
    g.n = static_cast<int>(d->d);
    g.out = y;
    g.ld = ldy;
    return x_product<mfk::kXF32>(ws, g, d->f, 0, 1);
}

// The weights' gradients in one launch, so that the last tiles of one run beside the first of the
// next: (dw_gate, dw_up) = x^T (dgate, dup) and dw_down = h^T dy, all over the rows. A column-major
// result is the transposed product with the operands exchanged. (1531 rows, 1003 x 2731: 88 and 44
// tiles on 74 pairs are three waves, 132 are two.)
int x_weight_grads(XWorkspace& ws, const mfk_gated_ffn_desc* d, const mfk_gated_ffn_grads* o,
                   const XMat& x, const XMat& dg, const XMat& h, const XMat& dy) {
    bool t = false, td = false;
    if (!x_orientation(d->d, d->f, o->dw_rs, o->dw_cs, &t) ||
        !x_orientation(d->f, d->d, o->dw_down_rs, o->dw_down_cs, &td))
        return MFK_ERR_UNSUPPORTED;
    mfk::XOperand ox = x_operand(ws, x, false), odg = x_operand(ws, dg, false);
    const mfk::XOperand oh = x_operand(ws, h, false), ody = x_operand(ws, dy, false);
    odg.bstride = static_cast<int>(dg.blocks());   // dup lies behind dgate
    mfk::XArgs g{};
    g.a[0] = t ? odg : ox;
    g.b[0] = t ? ox : odg;
    g.m = static_cast<int>(t ? d->f : d->d);
    g.n = static_cast<int>(t ? d->d : d->f);
    g.mb = (g.m + 127) / 128;
    g.nb = (g.n + 127) / 128;
    g.out = o->dw_gate;
    g.ld = t ? o->dw_cs : o->dw_rs;
    g.out_bs = o->dw_up - o->dw_gate;
    g.a[1] = td ? ody : oh;
    g.b[1] = td ? oh : ody;
    g.third.m = static_cast<int>(td ? d->d : d->f);
    g.third.n = static_cast<int>(td ? d->f : d->d);
    g.third.mb = (g.third.m + 127) / 128;
    g.third.nb = (g.third.n + 127) / 128;
    g.third.out = o->dw_down;
    g.third.ld = td ? o->dw_down_cs : o->dw_down_rs;
    return x_product<mfk::kXWeights>(ws, g, d->rows, 0, 3);
}

int run_gated_ffn_backward(const mfk_gated_ffn_desc* d, const mfk_gated_ffn_grads* o,
                           const float* saved, cudaStream_t stream) {
    int rc = check_gated(d);
    if (rc != MFK_OK) return rc;
    if (o == nullptr) return MFK_ERR_INVALID_ARGUMENT;
    const bool need_w = o->dw_gate != nullptr || o->dw_up != nullptr || o->dw_down != nullptr;
    const bool need_x = o->dx != nullptr;
    if (need_w && (o->dw_gate == nullptr || o->dw_up == nullptr || o->dw_down == nullptr))
        return MFK_ERR_INVALID_ARGUMENT;
    if (d->rows > 0 && d->d > 0 && o->grad == nullptr) return MFK_ERR_INVALID_ARGUMENT;
    if (need_x && o->ld_dx < d->d) return MFK_ERR_INVALID_ARGUMENT;
    if (saved != nullptr && !aligned16(saved)) return MFK_ERR_INVALID_ARGUMENT;
    bool t = false;
    if (need_w && (!x_orientation(d->d, d->f, o->dw_rs, o->dw_cs, &t) ||
                   !x_orientation(d->f, d->d, o->dw_down_rs, o->dw_down_cs, &t)))
        return MFK_ERR_UNSUPPORTED;
    if ((!need_x && !need_w) || d->d == 0) return MFK_OK;
    XWorkspace ws(stream);
    rc = current_device(&ws.dev, &ws.info);
    if (rc != MFK_OK) return rc;
    if (d->f == 0) return need_x ? x_zero(o->dx, d->rows, d->d, o->ld_dx, stream) : MFK_OK;
    if (d->rows == 0) {
        if (!need_w) return MFK_OK;
        x_orientation(d->d, d->f, o->dw_rs, o->dw_cs, &t);
        const int64_t r = t ? d->f : d->d, c = t ? d->d : d->f, ld = t ? o->dw_cs : o->dw_rs;
        rc = x_zero(o->dw_gate, r, c, std::max(ld, c), stream);
        if (rc == MFK_OK) rc = x_zero(o->dw_up, r, c, std::max(ld, c), stream);
        x_orientation(d->f, d->d, o->dw_down_rs, o->dw_down_cs, &t);
        const int64_t r2 = t ? d->d : d->f, c2 = t ? d->f : d->d,
                      ld2 = t ? o->dw_down_cs : o->dw_down_rs;
        if (rc == MFK_OK) rc = x_zero(o->dw_down, r2, c2, std::max(ld2, c2), stream);
        return rc;
    }
    mfk::XSources list{};
    // x twice where the projections are computed again: by rows for them, in blocks for the sums
    // over rows.
    XMat x, wg, wu, wd, dy, x_rows;
    if (!x_source(ws, list, &x, d->x, d->rows, d->d, d->x_rs, d->x_cs) ||
        !x_source(ws, list, &wg, d->w_gate, d->d, d->f, d->w_gate_rs, d->w_gate_cs) ||
        !x_source(ws, list, &wu, d->w_up, d->d, d->f, d->w_up_rs, d->w_up_cs) ||
        !x_source(ws, list, &wd, d->w_down, d->f, d->d, d->w_down_rs, d->w_down_cs) ||
        !x_source(ws, list, &dy, o->grad, d->rows, d->d, o->grad_rs, o->grad_cs) || x.transposed)
        return MFK_ERR_UNSUPPORTED;
    if (wg.transposed != wu.transposed) return MFK_ERR_UNSUPPORTED;
    if (saved == nullptr &&
        !x_source(ws, list, &x_rows, d->x, d->rows, d->d, d->x_rs, d->x_cs, 1, 0, true))
        return MFK_ERR_UNSUPPORTED;
    const XMat dg = x_mat(ws, d->rows, d->f);
    const XMat du = x_mat(ws, d->rows, d->f);  // directly behind dg: a batch of two
    const XMat h = x_mat(ws, d->rows, d->f);
    const int64_t saved_floats = gated_saved_floats(d->rows, d->f);
    const size_t again = saved == nullptr ? static_cast<size_t>(saved_floats) : 0;
    const size_t live_words = (static_cast<size_t>(d->rows) + 3) / 4 * 4;
    const int64_t top_words = h.blocks() * 4;
    rc = x_allocate(ws, again + live_words + static_cast<size_t>(top_words));
    if (rc != MFK_OK) return rc;
    int* live = reinterpret_cast<int*>(ws.extra + again);
    uint32_t* tops = reinterpret_cast<uint32_t*>(live + live_words);
    mfk::live_rows_kernel<<<static_cast<unsigned>((d->rows + 7) / 8), 256, 0, stream>>>(
        o->grad, o->grad_rs, o->grad_cs, static_cast<int>(d->rows), static_cast<int>(d->d), live,
        tops, top_words);
    g_launches.fetch_add(1);
    MFK_CUDA(cudaGetLastError());
    list.s[0].live = live;
    const XMat* mats[6] = {&x, &wg, &wu, &wd, &dy, &x_rows};
    rc = x_split(ws, list, mats, false);
    if (rc != MFK_OK) return rc;
    const float* pre = saved;
    if (pre == nullptr) {
        rc = gated_forward(ws, d, x_rows, wg, wu, nullptr, ws.extra);
        if (rc != MFK_OK) return rc;
        pre = ws.extra;
    }
    {   // dh = dy w_down^T, and from it dgate, dup and h
        mfk::XArgs g{};
        g.a[0] = g.a[1] = x_operand(ws, dy, true);
        g.b[0] = g.b[1] = x_operand(ws, wd, true);
        g.mb = h.rb;
        g.nb = h.cb;
        g.m = static_cast<int>(d->rows);
        g.n = static_cast<int>(d->f);
        g.act = d->activation;
        const int64_t blocks = h.blocks();
        float* p = const_cast<float*>(pre);
        g.gate = p;
        g.up = p + blocks * 128 * 128;
        g.gmax = p + blocks * 2 * 128 * 128;
        g.live = live;
        g.tops = tops;
        g.o[0] = x_out(ws, dg);
        g.o[1] = x_out(ws, du);
        g.o[2] = x_out(ws, h);
        rc = x_product<mfk::kXGatedBwd>(ws, g, d->d, 0, 1);
        if (rc != MFK_OK) return rc;
        // the blocks that it stored under loose scales, by tiles of one CTA
        int slots = 0;
        rc = x_slots<1, 1, mfk::kXGatedAgain, false>(ws, mfk::kXGatedAgain * 12 + 4, 1, &slots);
        if (rc != MFK_OK) return rc;
        rc = x_launch<1, 1, mfk::kXGatedAgain, false>(ws, g, slots, 1, g.mb, g.nb, blocks, 1);
        if (rc != MFK_OK) return rc;
    }
    if (need_x) {  // dx = dgate w_gate^T + dup w_up^T: one product over 2 f
        mfk::XArgs g{};
        g.a[0] = x_operand(ws, dg, true);
        g.a[1] = x_operand(ws, du, true);
        g.b[0] = x_operand(ws, wg, true);
        g.b[1] = x_operand(ws, wu, true);
        g.mb = h.rb;
        g.nb = static_cast<int>((d->d + 127) / 128);
        g.m = static_cast<int>(d->rows);
        g.n = static_cast<int>(d->d);
        g.out = o->dx;
        g.ld = o->ld_dx;
        rc = x_product<mfk::kXF32>(ws, g, d->f, d->f, 1);
        if (rc != MFK_OK) return rc;
    }
    if (need_w) return x_weight_grads(ws, d, o, x, dg, h, dy);
    return MFK_OK;
}

// ---- the orthogonalised update ---------------------------------------------------------------

int run_orthogonalize(const float* u, int64_t batch, int64_t rows, int64_t cols, int64_t rs,
                      int64_t bs, float* out, int64_t ld, int64_t out_bs, int32_t steps, float ca,
                      float cb, float cc, float eps, cudaStream_t stream) {
    if (batch < 0 || rows < 0 || cols < 0 || steps < 1) return MFK_ERR_INVALID_ARGUMENT;
    if (!(eps >= 0.0f)) return MFK_ERR_INVALID_ARGUMENT;
    if (rows > kXMaxDim || cols > kXMaxDim || batch > kXMaxDim) return MFK_ERR_UNSUPPORTED;
    if (batch == 0 || rows == 0 || cols == 0) return MFK_OK;
    if (u == nullptr || out == nullptr || ld < cols) return MFK_ERR_INVALID_ARGUMENT;
    XWorkspace ws(stream);
    int rc = current_device(&ws.dev, &ws.info);
    if (rc != MFK_OK) return rc;
    const bool tall = rows > cols;
    const int64_t k = tall ? cols : rows;  // the Gram matrix is k x k
    const int64_t depth = tall ? rows : cols;
    // One launch where a cluster holds the matrix: 48 of 64 x 128 in 115 us by the launches below.
    if (k <= mfk::kXBlk && depth <= mfk::kXBlk * mfk::kOrthMaxRanks &&
        batch <= (int64_t(1) << 27)) {
        mfk::OrthSmallArgs s{};
        s.u = u;
        s.rs = rs;
        s.bs = bs;
        s.out = out;
        s.ld = ld;
        s.out_bs = out_bs;
        s.rows = static_cast<int>(rows);
        s.cols = static_cast<int>(cols);
        s.tall = tall ? 1 : 0;
        s.steps = steps;
        s.a = ca;
        s.b = cb;
        s.c = cc;
        s.eps = eps;
        static std::atomic<uint64_t> ready{0};  // a bit per device
        if ((ready.load() >> ws.dev & 1u) == 0u) {
            MFK_CUDA(cudaFuncSetAttribute(mfk::orth_small_kernel,
                                          cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          mfk::kOrthSmem));
            ready.fetch_or(uint64_t(1) << ws.dev);
        }
        const int64_t ranks = (depth + mfk::kXBlk - 1) / mfk::kXBlk;
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        cfg.gridDim = dim3(static_cast<unsigned>(batch * ranks), 1, 1);
        cfg.blockDim = dim3(mfk::kOrthThreads, 1, 1);
        cfg.dynamicSmemBytes = mfk::kOrthSmem;
        cfg.stream = stream;
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        MFK_CUDA(cudaLaunchKernelEx(&cfg, mfk::orth_small_kernel, s));
        g_launches.fetch_add(1);
        return MFK_OK;
    }
    mfk::XSources list{};
    XMat x0;
    if (!x_source(ws, list, &x0, u, rows, cols, rs, 1, batch, bs)) return MFK_ERR_UNSUPPORTED;
    XMat x1 = steps > 1 ? x_mat(ws, rows, cols, batch) : x0;
    const XMat gram = x_mat(ws, k, k, batch), poly = x_mat(ws, k, k, batch);
    rc = x_allocate(ws, 0);
    if (rc != MFK_OK) return rc;
    const XMat* mats[1] = {&x0};
    rc = x_split(ws, list, mats, true);
    if (rc != MFK_OK) return rc;
    if (x0.blocks() > (int64_t(1) << 30)) return MFK_ERR_UNSUPPORTED;
    {
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        cfg.blockDim = dim3(256, 1, 1);
        cfg.gridDim = dim3(static_cast<unsigned>(batch), 1, 1);
        cfg.stream = stream;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        MFK_CUDA(cudaLaunchKernelEx(&cfg, mfk::split_normalize_kernel,
                                    static_cast<const double*>(ws.sumsq + x0.first),
                                    ws.inv + x0.inv, static_cast<int>(x0.blocks()), eps));
        g_launches.fetch_add(1);
    }
    XMat *x = &x0, *next = &x1;
    for (int step = 0; step < steps; ++step) {
        {   // gram = x x^T (or x^T x): symmetric, lower blocks only
            mfk::XArgs g{};
            g.a[0] = g.a[1] = g.b[0] = g.b[1] = x_operand(ws, *x, !tall);
            g.mb = g.nb = gram.rb;
            g.m = g.n = static_cast<int>(k);
            g.sym = 1;
            g.alpha = 1.0f;
            g.o[0] = x_out(ws, gram);
            rc = x_product<mfk::kXSplit>(ws, g, depth, 0, batch);
            if (rc != MFK_OK) return rc;
        }
        {   // poly = cb gram + cc gram gram
            mfk::XArgs g{};
            g.a[0] = g.a[1] = g.b[0] = g.b[1] = x_operand(ws, gram, true, true);
            g.mb = g.nb = gram.rb;
            g.m = g.n = static_cast<int>(k);
            g.sym = 1;
            g.alpha = cc;
            g.beta = cb;
            g.c = x_out(ws, gram);
            g.o[0] = x_out(ws, poly);
            rc = x_product<mfk::kXSplit>(ws, g, k, 0, batch);
            if (rc != MFK_OK) return rc;
        }
        // x = ca x + poly x (or x poly). (With ca on poly's diagonal no third matrix is read, but
        // then the largest term is rounded toward zero with the rest: 2.2e-6 off after five steps,
        // not 8e-7.)
        mfk::XArgs g{};
        if (tall) {
            g.a[0] = g.a[1] = x_operand(ws, *x, true);
            g.b[0] = g.b[1] = x_operand(ws, poly, true, true);
        } else {
            g.a[0] = g.a[1] = x_operand(ws, poly, true, true);
            g.b[0] = g.b[1] = x_operand(ws, *x, false);
        }
        g.mb = x->rb;
        g.nb = x->cb;
        g.m = static_cast<int>(rows);
        g.n = static_cast<int>(cols);
        g.alpha = 1.0f;
        g.beta = ca;
        g.c = x_out(ws, *x);
        if (step + 1 < steps) {
            g.o[0] = x_out(ws, *next);
            rc = x_product<mfk::kXSplit>(ws, g, k, 0, batch);
            std::swap(x, next);
        } else {
            g.out = out;
            g.ld = ld;
            g.out_bs = out_bs;
            rc = x_product<mfk::kXF32>(ws, g, k, 0, batch);
        }
        if (rc != MFK_OK) return rc;
    }
    return MFK_OK;
}

}  // namespace

extern "C" {

int mfk_gated_ffn_f32(const mfk_gated_ffn_desc* desc, float* y, int64_t ldy, float* saved,
                      void* stream) {
    return run_gated_ffn(desc, y, ldy, saved, static_cast<cudaStream_t>(stream));
}

int64_t mfk_gated_ffn_saved_floats(int64_t rows, int64_t f) {
    return rows < 0 || f < 0 || rows > kXMaxDim || f > kXMaxDim ? -1 : gated_saved_floats(rows, f);
}

int mfk_gated_ffn_backward_f32(const mfk_gated_ffn_desc* desc, const mfk_gated_ffn_grads* grads,
                               const float* saved, void* stream) {
    return run_gated_ffn_backward(desc, grads, saved, static_cast<cudaStream_t>(stream));
}

int mfk_orthogonalize_f32(const float* update, int64_t batch, int64_t rows, int64_t cols,
                          int64_t row_stride, int64_t batch_stride, float* out, int64_t ld,
                          int64_t out_batch_stride, int32_t steps, float a, float b, float c,
                          float eps, void* stream) {
    return run_orthogonalize(update, batch, rows, cols, row_stride, batch_stride, out, ld,
                             out_batch_stride, steps, a, b, c, eps,
                             static_cast<cudaStream_t>(stream));
}

}  // extern "C"
