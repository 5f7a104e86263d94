// Host side of the few-rows kernels (rows.cuh). Part of the library's one translation unit.
#pragma once

namespace {

// One product of few rows: picks the kernel by the weights' orientation and alignment, the tile
// width and the depth's shares (a cluster of 1 to 8 CTAs).
struct RowsLaunch {
    cudaStream_t stream;
    const DeviceInfo* info;
    int device;
    bool dependent;  // may start while the launch before still runs

    // Bytes on the longest path of a launch of `tiles` x ranks CTAs, two per SM: whole waves of
    // a share of the depth, plus about 4 us of start and finish a wave (90 KB at a CTA's share of
    // HBM). Fewer, longer waves beat an even number of shares: 8 rows, 4096 x 11008, gate and up
    // in 86 tiles: 106 us as 8 shares (2.3 waves), 80 us as 3 (0.9 waves).
    int64_t cost(int64_t tiles, int64_t depth, int64_t row_bytes, int* ranks) const {
        int64_t best = 0;
        *ranks = 1;
        for (int r = 1; r <= mfk::kRowsRanks && (r == 1 || depth >= r * 32); ++r) {
            const int64_t slots = int64_t(info->sm_count) * 2;
            const int64_t waves = (tiles * r + slots - 1) / slots;
            const int64_t c = waves * ((depth + r - 1) / r * row_bytes + 90000);
            if (best == 0 || c < best) {
                best = c;
                *ranks = r;
            }
        }
        return best;
    }

    template <void (*kernel)(mfk::RowsArgs)>
    int go(const mfk::RowsArgs& g, int64_t tiles, int ranks) const {
        static std::atomic<uint64_t> ready{0};  // a bit per device
        if ((ready.load() >> device & 1u) == 0u) {
            MFK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          mfk::kRowsSmem));
            ready.fetch_or(uint64_t(1) << device);
        }
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[2];
        cfg.gridDim = dim3(static_cast<unsigned>(tiles * ranks), 1, 1);
        cfg.blockDim = dim3(256, 1, 1);
        cfg.dynamicSmemBytes = mfk::kRowsSmem;
        cfg.stream = stream;
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.numAttrs = 1;
        if (dependent) {
            attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[1].val.programmaticStreamSerializationAllowed = 1;
            cfg.numAttrs = 2;
        }
        cfg.attrs = attr;
        MFK_CUDA(cudaLaunchKernelEx(&cfg, kernel, g));
        g_launches.fetch_add(1);
        return MFK_OK;
    }

    template <int MT, int W>
    int run(const mfk::RowsArgs& g, bool depth_contiguous) const {
        const bool same4 = aligned16(g.w0) && g.ld0 % 4 == 0 &&
                           (W == 1 || (aligned16(g.w1) && g.ld1 % 4 == 0));
        int ranks = 1;
        if (depth_contiguous) {
            const int64_t tiles = (g.cols + 15) / 16;
            cost(tiles, g.depth, 64 * W, &ranks);
            if (same4 && g.depth % 4 == 0)
                return go<mfk::rows_k_kernel<MT, 4, W>>(g, tiles, ranks);
            return go<mfk::rows_k_kernel<MT, 1, W>>(g, tiles, ranks);
        }
        // tiles of 128, 64 or 32 columns by that cost, narrow ones a little dearer per byte
        const int64_t t4 = (g.cols + 127) / 128, t2 = (g.cols + 63) / 64, t1 = (g.cols + 31) / 32;
        int r4 = 1, r2 = 1, r1 = 1;
        const double c4 = static_cast<double>(cost(t4, g.depth, 512 * W, &r4));
        const double c2 = 1.1 * static_cast<double>(cost(t2, g.depth, 256 * W, &r2));
        const double c1 = 1.3 * static_cast<double>(cost(t1, g.depth, 128 * W, &r1));
        constexpr bool kWide = MT * W <= 16;  // 64 sums a lane at most
        const bool can4 = kWide && same4 && g.cols % 4 == 0;
        const bool can2 = same4 && g.cols % 2 == 0;
        if constexpr (kWide) {
            if (can4 && c4 <= c2 && c4 <= c1)
                return go<mfk::rows_n_kernel<MT, 4, W>>(g, t4, r4);
        }
        if (can2 && c2 <= c1) return go<mfk::rows_n_kernel<MT, 2, W>>(g, t2, r2);
        return go<mfk::rows_n_kernel<MT, 1, W>>(g, t1, r1);
    }

    template <int W>
    int product(const mfk::RowsArgs& g, bool depth_contiguous) const {
        if (g.rows == 1) return run<1, W>(g, depth_contiguous);
        if (g.rows == 2) return run<2, W>(g, depth_contiguous);
        if (g.rows <= 4) return run<4, W>(g, depth_contiguous);
        if (g.rows <= 8) return run<8, W>(g, depth_contiguous);
        return run<16, W>(g, depth_contiguous);
    }
};

// The block for at most kRowsMax rows.
int run_gated_rows(const mfk_gated_ffn_desc* d, float* y, int64_t ldy, const DeviceInfo* info,
                   int device, cudaStream_t stream) {
    bool tg = false, tu = false, td = false;
    if (!x_orientation(d->d, d->f, d->w_gate_rs, d->w_gate_cs, &tg) ||
        !x_orientation(d->d, d->f, d->w_up_rs, d->w_up_cs, &tu) ||
        !x_orientation(d->f, d->d, d->w_down_rs, d->w_down_cs, &td) || tg != tu)
        return MFK_ERR_UNSUPPORTED;
    float* h = nullptr;
    const int64_t ldh = (d->f + 3) / 4 * 4;
    MFK_CUDA(cudaMallocAsync(reinterpret_cast<void**>(&h), static_cast<size_t>(d->rows * ldh) * 4,
                             stream));
    struct Free {
        void* p;
        cudaStream_t s;
        ~Free() { cudaFreeAsync(p, s); }
    } release{h, stream};
    mfk::RowsArgs g{};
    g.x = d->x;
    g.x_rs = d->x_rs;
    g.w0 = d->w_gate;
    g.w1 = d->w_up;
    g.ld0 = tg ? d->w_gate_cs : d->w_gate_rs;
    g.ld1 = tu ? d->w_up_cs : d->w_up_rs;
    g.rows = static_cast<int>(d->rows);
    g.depth = static_cast<int>(d->d);
    g.cols = static_cast<int>(d->f);
    g.out = h;
    g.ldo = ldh;
    g.act = d->activation;
    const int rc = RowsLaunch{stream, info, device, false}.product<2>(g, tg);
    if (rc != MFK_OK) return rc;
    mfk::RowsArgs o{};
    o.x = h;
    o.x_rs = ldh;
    o.w0 = d->w_down;
    o.ld0 = td ? d->w_down_cs : d->w_down_rs;
    o.rows = g.rows;
    o.depth = g.cols;
    o.cols = g.depth;
    o.out = y;
    o.ldo = ldy;
    o.wait = 1;
    return RowsLaunch{stream, info, device, true}.product<1>(o, td);
}

}  // namespace
