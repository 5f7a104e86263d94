// fp32 matrix products on the fp16 tensor cores, for the language-model operators (the gated
// feed-forward block and its backward pass, the orthogonalised update).
//
// Mathematics. A matrix is cut into blocks of 128 x 128. With s the power of two that brings a
// block's largest magnitude into [2^14, 2^15), each entry x of the block is held as two halves,
//     hi = fp16(s x),  lo = fp16(s x - hi),
// so s x = hi + lo to 2^-23 of itself (and never worse than 2^-40 of the block's largest entry:
// lo's spacing ends at 2^-24). An operand whose rows are the result's rows may have one s per row
// of a block instead (`by_row`): then no row's accuracy depends on another's size. A product of two
// such matrices takes three fp16 products,
//     (s_a a)(s_b b) ~ lo hi + hi lo + hi hi,
// summed in fp32; the term left out, lo lo, is below 2^-22 of the product. fp16 tensor products
// run at twice the tf32 rate, so this is twice as fast as a tf32 three-way split of the same 22
// bits; the price is the block scale.
//
// Accumulation. tcgen05 rounds its fp32 accumulator toward zero on every instruction: each one
// loses about 3.4e-8 of the running sum, always towards zero (measured: 3.8e-6 relative to the
// result after 192 instructions, 1.2e-5 after sixteen times as many spread over stream-K parts). So
// a tensor-memory accumulator only ever holds one 128-deep chunk (24 instructions, the small lo
// products of a stage first), and the epilogue warps add the chunks, scaled by the two blocks' 1/s,
// in fp32 registers with round to nearest.
//
// Layout. A block is 64 KB: hi then lo, each as 16 columns-of-eight ("lines"), a line holding
// 128 rows x 8 halves (16 bytes a row, 2 KB). 8 rows x 16 bytes are one core matrix of the
// unswizzled operand layouts, and the same bytes serve as a K-major operand (contraction along
// the stored columns) and as an MN-major one (along the stored rows): no operand is ever
// transposed or split twice. The epilogues write blocks with full 128-byte rows of 16-byte
// stores, one per lane.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "mfk_ptx.cuh"

namespace mfk {

constexpr int kXBlk = 128;                 // block side
constexpr int kXBlockBytes = 65536;        // hi 32 KB, lo 32 KB
constexpr int kXLineBytes = 2048;          // 128 rows x 8 halves
constexpr int kXBlockLines = 32;
constexpr int kXThreads = 320;             // TMA warp, MMA warp, eight epilogue warps
constexpr int kXEpiWarp0 = 2;
constexpr int kXEpiThreads = 256;
constexpr int kXBoxFloats = 32 * 32;

// kXWeights: fp32 results of three products in one launch, two of one shape (a batch) and a third
// with sizes and operands of its own over the same depth. kXGatedAgain: kXGatedBwd for the blocks
// that it stored under loose scales.
enum XEpi : int {
    kXF32 = 0, kXSplit = 1, kXGated = 2, kXGatedBwd = 3, kXWeights = 4, kXGatedAgain = 5
};

template <int EPI>
__host__ __device__ constexpr bool x_fp32() {
    return EPI == kXF32 || EPI == kXWeights;
}

template <int EPI>
__host__ __device__ constexpr bool x_backward() {
    return EPI == kXGatedBwd || EPI == kXGatedAgain;
}

// A split matrix as an operand: block (mn, k) of matrix z.
struct XOperand {
    int line0;        // first line of block 0 in the tensor maps
    int ldb;          // blocks per stored block row
    int bstride;      // blocks from one matrix of a batch to the next
    int flip;         // 0: contraction along the stored columns, 1: along the stored rows
    int sym;          // symmetric: only blocks (i, j) with i >= j are stored
    int by_row;       // a scale for every row of a block
    const float* inv; // 1/s per block, or per row of a block
};

struct XOut {
    uint8_t* data;
    float* inv;
    int ldb, bstride;
};

struct XArgs {
    XOperand a[2], b[2];   // two segments of the contraction, or (gated) b = gate and up, or
                           // (weights) the batch's and the third product's
    int kc0, kc;           // chunks of 128 in segment 0, in all
    int last0, last1;      // stages of 64 in each segment's last chunk (1 or 2)
    int mb, nb;            // output blocks
    int m, n;              // output entries
    int tiles_m, tiles_n, splits, units, sym;
    int tiles;             // per matrix
    float alpha, beta;     // acc * alpha + C * beta (kXF32 without C: acc)
    XOut c;                // C as a split matrix (beta != 0)
    float* out;            // fp32 output, row stride ld, batch stride out_bs
    long long ld, out_bs;
    struct {               // the third product of kXWeights
        int tiles_m, tiles_n, mb, nb, m, n;
        float* out;
        long long ld;
    } third;
    XOut o[3];             // split outputs: result / h; dgate, dup, h
    float* gate;           // saved pre-activations in accumulator order (null: not saved)
    float* up;
    float* gmax;           // largest |gate| and |up| of 64 columns: per block [2][2 halves][128]
    const int* live;       // backward: 0 for the rows whose gradient is all zero
    uint32_t* tops;        // backward, per block: fp16 bits of the largest |hi| of dgate, dup, h
    int act;
    int store_h;
};

// ---- PTX forms this kernel adds --------------------------------------------------------------

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int32_t x, int32_t y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y)
        : "memory");
}

__device__ __forceinline__ void tma_load_2d_cg2(void* dst, const CUtensorMap* map,
                                                uint32_t bar_cluster_addr, int32_t x, int32_t y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster_addr), "r"(x), "r"(y)
        : "memory");
}

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                        uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
            : "memory");
    }
}

// 32 lanes x 16 consecutive columns, landed when it returns.
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, float (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]),
          "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]),
          "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(taddr)
        : "memory");
}

// a0 += r0 f, a1 += r1 f: one instruction for the pair.
__device__ __forceinline__ void fma2(float& a0, float& a1, float r0, float r1, float f) {
    asm("{\n\t.reg .b64 a, r, f;\n\t"
        "mov.b64 a, {%0, %1};\n\t"
        "mov.b64 r, {%2, %3};\n\t"
        "mov.b64 f, {%4, %4};\n\t"
        "fma.rn.f32x2 a, r, f, a;\n\t"
        "mov.b64 {%0, %1}, a;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "f"(r0), "f"(r1), "f"(f));
}

// kind::f16 with fp16 operands and an fp32 accumulator (fields as idesc_tf32; formats 0 = F16).
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool a_mn_major, bool b_mn_major) {
    return (1u << 4) | ((a_mn_major ? 1u : 0u) << 15) | ((b_mn_major ? 1u : 0u) << 16) |
           ((static_cast<uint32_t>(n) >> 3) << 17) | ((static_cast<uint32_t>(m) >> 4) << 24);
}

__device__ __forceinline__ uint32_t cluster_nctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

// Programmatic dependent launch: the launches of one call start while the one before still runs,
// set themselves up, and wait for its results here.
__device__ __forceinline__ void grid_dependents_go() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ void grid_wait() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
    asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

__device__ __forceinline__ void epi_bar() {
    asm volatile("bar.sync 1, 256;" ::: "memory");
}

// ---- the split -------------------------------------------------------------------------------

// s (a power of two) for a block whose largest finite magnitude is amax, and 1/s. s stays a
// normal number with a normal reciprocal: below 2^-112 the scaled values merely get smaller.
__device__ __forceinline__ void split_scale(float amax, float& s, float& inv) {
    const int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;  // amax >= 0
    const int sh = amax == 0.0f ? 0 : min(14 - e, 126);
    s = __uint_as_float(static_cast<uint32_t>(sh + 127) << 23);
    inv = __uint_as_float(static_cast<uint32_t>(127 - sh) << 23);
}

__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.0f;  // infinities and NaN do not set a block's scale
}

// The largest finite |v[i]|: one instruction a value (a NaN is passed over), and only if an
// infinity turns up a second look without them.
template <int N>
__device__ __forceinline__ float largest(const float* v) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, fabsf(v[i]));
    if (m > 3.402823466e38f) {
        m = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, finite_abs(v[i]));
    }
    return m;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ unsigned long long pack2(float2 a) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
    return r;
}

__device__ __forceinline__ float2 unpack2(unsigned long long a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)));
    return unpack2(r);
}

__device__ __forceinline__ float2 sub2(float2 a, float2 b) {
    unsigned long long r;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)));
    return unpack2(r);
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)));
    return unpack2(r);
}

__device__ __forceinline__ float2 fma2v(float2 a, float2 b, float2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)), "l"(pack2(c)));
    return unpack2(r);
}

// (hi, lo) of s x0 and s x1, packed. A non-finite x makes lo NaN.
__device__ __forceinline__ void split_pair(float x0, float x1, float s, uint32_t& hi,
                                           uint32_t& lo) {
    const float2 xs = mul2(make_float2(x0, x1), make_float2(s, s));
    const __half2 h = __floats2half2_rn(xs.x, xs.y);
    const float2 lf = sub2(xs, __half22float2(h));   // exact
    const __half2 l = __floats2half2_rn(lf.x, lf.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Eight consecutive columns (16-byte line `chunk`) of one row of a block; `top` gathers the largest
// |hi| of even and odd columns.
__device__ __forceinline__ void store_split8(uint8_t* block, int chunk, int row, const float* v,
                                             float s, __half2* top = nullptr) {
    uint4 h, l;
    split_pair(v[0], v[1], s, h.x, l.x);
    split_pair(v[2], v[3], s, h.y, l.y);
    split_pair(v[4], v[5], s, h.z, l.z);
    split_pair(v[6], v[7], s, h.w, l.w);
    if (top != nullptr) {
        const uint32_t hs[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *top = __hmax2(*top, __habs2(*reinterpret_cast<const __half2*>(&hs[i])));
    }
    uint8_t* p = block + chunk * kXLineBytes + row * 16;
    *reinterpret_cast<uint4*>(p) = h;
    *reinterpret_cast<uint4*>(p + kXBlockBytes / 2) = l;
}

struct XSource {
    const float* src;      // rows x cols, unit column stride
    long long rs, bs;      // row stride, batch stride (elements)
    int rows, cols;
    int rb, cb;            // blocks of a matrix
    int vec;               // every row starts on 16 bytes
    int first;             // index of this matrix's first block in the launch
    uint8_t* data;
    float* inv;
    double* sumsq;         // per-block sum of squares, or null
    const int* live;       // rows to leave out (0) as if they were zero, or null
    int by_row;            // a scale for every row
};

constexpr int kXMaxSources = 6;
struct XSources {
    XSource s[kXMaxSources];
    int count;
};

// One 128 x 128 block per CTA of 256 threads: 64 entries per thread in registers, the block's
// largest magnitude, then hi and lo. Lanes take 8 rows x 4 eight-column lines, so a warp reads
// 128-byte row pieces and writes whole 128-byte core matrices. Bound by HBM: 4 bytes read, 4
// written per entry.
__global__ void __launch_bounds__(256) split_blocks_kernel(const __grid_constant__ XSources list) {
    grid_dependents_go();
    int which = 0;
#pragma unroll
    for (int i = 1; i < kXMaxSources; ++i)
        if (i < list.count && static_cast<int>(blockIdx.x) >= list.s[i].first) which = i;
    const XSource& t = list.s[which];
    const int local = static_cast<int>(blockIdx.x) - t.first;
    const int per = t.rb * t.cb;
    const int z = local / per;
    const int ij = local - z * per;
    const int bi = ij / t.cb, bj = ij - bi * t.cb;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r8 = lane >> 2, c4 = lane & 3;
    const float* base = t.src + z * t.bs;
    // only the blocks that leave rows out read what the launch before writes (and with them the
    // whole launch ends after that one)
    if (t.live != nullptr) grid_wait();
    float v[2][4][8];
    if (t.vec) {
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int row = bi * kXBlk + (warp * 2 + a) * 8 + r8;
            const bool row_ok = row < t.rows && (t.live == nullptr || t.live[row] != 0);
            const float* p = base + static_cast<long long>(row_ok ? row : 0) * t.rs;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int col = bj * kXBlk + (b * 4 + c4) * 8;
#pragma unroll
                for (int j = 0; j < 8; j += 4) {
                    float4 q = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (row_ok) {
                        if (col + j + 4 <= t.cols) {
                            q = *reinterpret_cast<const float4*>(p + col + j);
                        } else {
                            if (col + j < t.cols) q.x = p[col + j];
                            if (col + j + 1 < t.cols) q.y = p[col + j + 1];
                            if (col + j + 2 < t.cols) q.z = p[col + j + 2];
                        }
                    }
                    v[a][b][j] = q.x;
                    v[a][b][j + 1] = q.y;
                    v[a][b][j + 2] = q.z;
                    v[a][b][j + 3] = q.w;
                }
            }
        }
    } else {
        // Rows that start anywhere: read along, 128 bytes an instruction, eight rows of the warp's
        // sixteen at a time, and handed to their lanes through shared memory. (Each lane's columns
        // one by one: 1531 x 1003 and three of 1003 x 2731 in 22.9 us, 20.6 so.)
        __shared__ __align__(16) float lines[8][8][kXBlk + 4];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int row0 = bi * kXBlk + (warp * 2 + a) * 8;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const int row = row0 + r;
                const bool row_ok = row < t.rows && (t.live == nullptr || t.live[row] != 0);
                const float* p = base + static_cast<long long>(row_ok ? row : 0) * t.rs;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int col = bj * kXBlk + b * 32 + lane;
                    v[a][r / 2][(r & 1) * 4 + b] = row_ok && col < t.cols ? p[col] : 0.0f;
                }
            }
        }
#pragma unroll
        for (int a = 0; a < 2; ++a) {
#pragma unroll
            for (int r = 0; r < 8; ++r)
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    lines[warp][r][b * 32 + lane] = v[a][r / 2][(r & 1) * 4 + b];
            __syncwarp();
#pragma unroll
            for (int b = 0; b < 4; ++b) {
#pragma unroll
                for (int j = 0; j < 8; j += 4) {
                    const float4 q = *reinterpret_cast<const float4*>(
                        &lines[warp][r8][(b * 4 + c4) * 8 + j]);
                    v[a][b][j] = q.x;
                    v[a][b][j + 1] = q.y;
                    v[a][b][j + 2] = q.z;
                    v[a][b][j + 3] = q.w;
                }
            }
            __syncwarp();
        }
    }
    const float amax = largest<64>(&v[0][0][0]);
    double sum = 0.0;
    if (t.sumsq != nullptr) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    sum += static_cast<double>(v[a][b][j]) * static_cast<double>(v[a][b][j]);
    }
    __shared__ uint32_t wmax[8];
    __shared__ double wsum[8];
    const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));
    if (t.sumsq != nullptr) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (lane == 0) {
        wmax[warp] = m;
        wsum[warp] = sum;
    }
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) all = max(all, wmax[w]);
    float s, inv;
    split_scale(__uint_as_float(all), s, inv);
    if (threadIdx.x == 0) {
        if (!t.by_row) t.inv[local] = inv;
        if (t.sumsq != nullptr) {
            double total = 0.0;
#pragma unroll
            for (int w = 0; w < 8; ++w) total += wsum[w];
            t.sumsq[local] = total;
        }
    }
    uint8_t* block = t.data + static_cast<long long>(local) * kXBlockBytes;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        const int row = (warp * 2 + a) * 8 + r8;
        if (t.by_row) {  // a row's 128 columns lie in four lanes
            float m = largest<32>(&v[a][0][0]);
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            split_scale(m, s, inv);
            if (c4 == 0) t.inv[static_cast<long long>(local) * kXBlk + row] = inv;
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) store_split8(block, b * 4 + c4, row, v[a][b], s);
    }
}

// live[r] = whether row r of the rows x cols matrix has an entry other than zero: a warp per row,
// which stops at the first 32 columns that have one. Clears `words` words at `clear`.
__global__ void __launch_bounds__(256)
    live_rows_kernel(const float* __restrict__ p, long long rs, long long cs, int rows, int cols,
                     int* __restrict__ live, uint32_t* __restrict__ clear, long long words) {
    grid_dependents_go();
    const long long t = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    for (long long i = t; i < words; i += static_cast<long long>(gridDim.x) * 256) clear[i] = 0u;
    const int lane = threadIdx.x & 31;
    const int r = static_cast<int>(t >> 5);
    if (r >= rows) return;
    bool any = false;
    for (int c = 0; c < cols && !any; c += 32) {
        const bool mine = c + lane < cols && !(p[r * rs + (c + lane) * cs] == 0.0f);
        any = __any_sync(0xffffffffu, mine);
    }
    if (lane == 0) live[r] = any ? 1 : 0;
}

// Divides matrix z of a batch by its Frobenius norm (+ eps) by scaling the blocks' 1/s: exact up
// to the factor's own rounding, since every 1/s is a power of two. The blocks' sums of squares
// are added in one fixed order, in double.
__global__ void __launch_bounds__(256) split_normalize_kernel(const double* sumsq, float* inv,
                                                              int blocks, float eps) {
    __shared__ double part[256];
    grid_dependents_go();
    grid_wait();
    const double* p = sumsq + static_cast<long long>(blockIdx.x) * blocks;
    double sum = 0.0;
    for (int i = threadIdx.x; i < blocks; i += 256) sum += p[i];
    part[threadIdx.x] = sum;
    __syncthreads();
#pragma unroll
    for (int o = 128; o > 0; o >>= 1) {
        if (static_cast<int>(threadIdx.x) < o) part[threadIdx.x] += part[threadIdx.x + o];
        __syncthreads();
    }
    // in double: the factor alone leaves fp32's normal range where the norm is above 2^126
    const double f = 1.0 / (sqrt(part[0]) + static_cast<double>(eps));
    float* q = inv + static_cast<long long>(blockIdx.x) * blocks;
    for (int i = threadIdx.x; i < blocks; i += 256) q[i] = static_cast<float>(q[i] * f);
}

// ---- activations of the gated block ----------------------------------------------------------

enum XAct : int { kXActNone = 0, kXActRelu = 1, kXActGelu = 2, kXActGeluTanh = 3, kXActSilu = 4 };

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// v within [-16, 16], NaN as it is.
__device__ __forceinline__ float clamp16(float v) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;\n\tmin.NaN.f32 %0, %0, %3;"
        : "=&f"(y)
        : "f"(v), "f"(-16.0f), "f"(16.0f));
    return y;
}

// 1 / (1 + exp(-z)): 2^(-z log2 e) is off by |z| 2^-24 relative at most, which the 1 it is added
// to hides wherever the result is not tiny.
__device__ __forceinline__ float logistic(float z) {
    return rcp(1.0f + ex2(z * -1.4426950408889634f));
}

// act(v) and act'(v) in fp32. silu and the tanh form of GELU go through the logistic function s:
// 0.5 (1 + tanh z) = s(2 z). The kind is a template parameter and the epilogues branch on it once
// per tile: with the branch inside the unrolled loops the code of all kinds lies between one
// element and the next, and fetching it took half of the kernels' time (4096 x 1024 x 4096: forward
// 380 us, 192 without it; backward 435 and 190).
template <int ACT>
__device__ __forceinline__ float2 act_slope(float v) {
    if constexpr (ACT == kXActSilu) {
        const float s = logistic(v);
        return make_float2(v * s, s * (1.0f + v * (1.0f - s)));
    } else if constexpr (ACT == kXActRelu) {
        const float rest = v == v ? 0.0f : v;  // NaN stays NaN, the derivative's too
        return v > 0.0f ? make_float2(v, 1.0f) : make_float2(rest, rest);
    } else if constexpr (ACT == kXActGelu) {
        // The normal distribution's tail: 0.5 erfc(|v| / sqrt 2) = exp(-v^2 / 2) t q(t) with
        // t = 1 / (1 + |v| / 4) and q a polynomial of degree 9, fitted to 3.4e-8 of the value
        // for all |v| by reweighted least squares. Within 4e-7 of Phi for |v| < 3, and to
        // v^2 2^-24 in the tail. The exponential serves the derivative's density too.
        const float t = rcp(fmaf(fabsf(v), 0.25f, 1.0f));
        const float e = ex2(v * v * -0.72134752044448170f);
        float q = 1.978445737e-02f;
        q = fmaf(q, t, -8.088806416e-02f);
        q = fmaf(q, t, 9.561682330e-02f);
        q = fmaf(q, t, -3.173717236e-02f);
        q = fmaf(q, t, 6.371062601e-02f);
        q = fmaf(q, t, 5.897111475e-02f);
        q = fmaf(q, t, 8.160392950e-02f);
        q = fmaf(q, t, 9.346626611e-02f);
        q = fmaf(q, t, 9.973643596e-02f);
        q = fmaf(q, t, 9.973556666e-02f);
        const float tail = e * t * q;
        const float phi = v < 0.0f ? tail : 1.0f - tail;
        return make_float2(v * phi, fmaf(v * 0.39894228040143268f, e, phi));
    } else if constexpr (ACT == kXActGeluTanh) {
        const float w = clamp16(v);  // the logistic is 0 or 1 beyond
        const float s = logistic(1.5957691216057308f * (w + 0.044715f * w * w * w));
        const float dz2 = 1.5957691216057308f * (1.0f + 0.134145f * w * w);
        return make_float2(v * s, s + w * s * (1.0f - s) * dz2);
    } else {
        return make_float2(v, 1.0f);
    }
}

// Two values at a time: (act, act') of v; the silu in packed arithmetic.
template <int ACT>
__device__ __forceinline__ void act_slope2(float2 v, float2& a, float2& slope) {
    if constexpr (ACT == kXActSilu) {
        const float2 one = make_float2(1.0f, 1.0f);
        const float2 z = mul2(v, make_float2(-1.4426950408889634f, -1.4426950408889634f));
        const float2 d = add2(make_float2(ex2(z.x), ex2(z.y)), one);
        const float2 s = make_float2(rcp(d.x), rcp(d.y));
        a = mul2(v, s);
        slope = mul2(s, fma2v(v, sub2(one, s), one));
    } else {
        const float2 p = act_slope<ACT>(v.x), q = act_slope<ACT>(v.y);
        a = make_float2(p.x, q.x);
        slope = make_float2(p.y, q.y);
    }
}

// Calls f with the activation as a compile-time constant.
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
    switch (act) {
    case kXActSilu: f(std::integral_constant<int, kXActSilu>{}); break;
    case kXActRelu: f(std::integral_constant<int, kXActRelu>{}); break;
    case kXActGelu: f(std::integral_constant<int, kXActGelu>{}); break;
    case kXActGeluTanh: f(std::integral_constant<int, kXActGeluTanh>{}); break;
    default: f(std::integral_constant<int, kXActNone>{}); break;
    }
}

// The largest |act'| over all inputs (GELU's is 1.1290): bounds the gate's gradient.
constexpr float kXMaxSlope = 1.13f;

// fp16 bits of 2^11: a block whose scale brought a bound into [2^14, 2^15) and whose largest |hi|
// is below, or infinite, has a scale that is more than three powers of two off, or unknown.
constexpr uint32_t kXTight = 0x6800u;
constexpr float kXMostScale = 8.507059173e37f;  // 2^126, the largest that split_scale gives

__device__ __forceinline__ bool x_loose(uint32_t top) {
    return top < kXTight || top >= 0x7c00u;
}

// ---- the product -----------------------------------------------------------------------------

template <int CG, int NB>
struct XConfig {
    static constexpr int kBBlocks = CG == 2 ? 1 : NB;   // blocks of B this CTA loads
    static constexpr int kStageBytes = 32768 * (1 + kBBlocks);
    static constexpr int kStages = kBBlocks == 2 ? 2 : 3;
    static constexpr int kTmemCols = NB * 256;          // two accumulators
    static constexpr int kStageArea = kStages * kStageBytes;
    static constexpr int kEpiBytes = 8 * kXBoxFloats * 4;  // one box per epilogue warp
    static constexpr int kSmemBytes = kStageArea + kEpiBytes + 1024 + 512;
};

struct XUnit {
    int z, tm, tn, s, c0, c1;
};

template <int EPI>
__device__ __forceinline__ bool x_third(int z) {
    return EPI == kXWeights && z == 2;
}

template <int EPI>
__device__ __forceinline__ XUnit x_unit(const XArgs& g, int u) {
    XUnit w;
    const int t = u / g.splits;
    w.s = u - t * g.splits;
    w.z = t / g.tiles;
    int q = t - w.z * g.tiles;
    if (g.sym) {  // lower triangle, row by row
        int i = static_cast<int>((sqrtf(8.0f * static_cast<float>(q) + 1.0f) - 1.0f) * 0.5f);
        while (i * (i + 1) / 2 > q) --i;
        while ((i + 1) * (i + 2) / 2 <= q) ++i;
        w.tm = i;
        w.tn = q - i * (i + 1) / 2;
    } else {  // bands of eight tile rows, column by column, so the operands in flight stay in L2
        const int tiles_m = x_third<EPI>(w.z) ? g.third.tiles_m : g.tiles_m;
        const int tiles_n = x_third<EPI>(w.z) ? g.third.tiles_n : g.tiles_n;
        const int band = q / (8 * tiles_n);
        const int first = band * 8;
        const int height = min(8, tiles_m - first);
        q -= first * tiles_n;
        w.tn = q / height;
        w.tm = first + q - w.tn * height;
    }
    w.c0 = static_cast<int>(static_cast<long long>(g.kc) * w.s / g.splits);
    w.c1 = static_cast<int>(static_cast<long long>(g.kc) * (w.s + 1) / g.splits);
    return w;
}

// Whether a launch has nothing to do in this tile.
template <int EPI>
__device__ __forceinline__ bool x_skips(const XArgs& g, const XUnit& w) {
    if constexpr (EPI == kXGatedAgain) {
        const uint4 t = __ldcg(reinterpret_cast<const uint4*>(g.tops) +
                               (static_cast<long long>(w.tm) * g.nb + w.tn));
        return !x_loose(t.x) && !x_loose(t.y) && !x_loose(t.z);
    } else {
        return false;
    }
}

// Whether a tile whose first block along the operand's mn is `mn0` reads chunk k along the
// blocks' stored rows (MN-major). A symmetric matrix stores only its lower blocks: a chunk right
// of the tile's first block comes from (k, mn), transposed. All blocks of one MMA agree: for
// k > mn0 every block of the tile has mn <= k or is one below (k >= mn0 + 1), and a diagonal
// block reads either way.
__device__ __forceinline__ int x_flip(const XOperand& o, int mn0, int k) {
    return o.sym ? (k > mn0 ? 1 : 0) : o.flip;
}

__device__ __forceinline__ int x_block(const XOperand& o, int z, int mn, int k, int flip) {
    return z * o.bstride + (flip ? k * o.ldb + mn : mn * o.ldb + k);
}

// The 128 x 64 (or 64 x 128) half of a block that stage `half` of a chunk reads: hi, then lo.
template <int CG>
__device__ __forceinline__ void x_load(uint8_t* dst, const CUtensorMap* mk, const CUtensorMap* mm,
                                       uint64_t* bar, uint32_t bar0, const XOperand& o, int z,
                                       int mn0, int mn, int k, int half) {
    const int flip = x_flip(o, mn0, k);
    const int line = o.line0 + x_block(o, z, mn, k, flip) * kXBlockLines;
    const CUtensorMap* map = flip ? mm : mk;
    const int x = flip ? half * 128 : 0;           // rows 64 half.. of every line (8-byte units)
    const int y = flip ? line : line + half * 8;   // lines 8 half..
    if constexpr (CG == 1) {
        tma_load_2d(dst, map, bar, x, y);
        tma_load_2d(dst + 16384, map, bar, x, y + 16);
    } else {
        tma_load_2d_cg2(dst, map, bar0, x, y);
        tma_load_2d_cg2(dst + 16384, map, bar0, x, y + 16);
    }
}

template <int CG, int NB, int EPI>
__device__ __forceinline__ void x_producer(const XArgs& g, const CUtensorMap* mk,
                                           const CUtensorMap* mm, uint8_t* stages, uint64_t* full,
                                           uint64_t* empty, uint32_t rank, uint32_t leader,
                                           int first, int step) {
    using C = XConfig<CG, NB>;
    int stage = 0;
    uint32_t phase = 0;
    for (int u = first; u < g.units; u += step) {
        const XUnit w = x_unit<EPI>(g, u);
        if (x_skips<EPI>(g, w)) continue;
        const int nb = x_third<EPI>(w.z) ? g.third.nb : g.nb;
        const int i = min(w.tm * CG + static_cast<int>(rank),
                          (x_third<EPI>(w.z) ? g.third.mb : g.mb) - 1);
        for (int c = w.c0; c < w.c1; ++c) {
            const int seg = x_third<EPI>(w.z) || (EPI == kXF32 && c >= g.kc0) ? 1 : 0;
            const int k = EPI == kXF32 && seg ? c - g.kc0 : c;
            const int halves = c == g.kc0 - 1 ? g.last0 : (c == g.kc - 1 ? g.last1 : 2);
            for (int h = 0; h < halves; ++h) {
                if (!mbar_wait(&empty[stage], phase ^ 1u, 1u << 0)) {
                    // the copies in flight land before this CTA may leave
                    const uint64_t t0 = global_timer();
                    while (global_timer() - t0 < 1000000ull) {
                    }
                    return;
                }
                uint8_t* s = stages + stage * C::kStageBytes;
                uint32_t bar0 = 0;
                if constexpr (CG == 1) {
                    mbar_arrive_expect_tx(&full[stage], C::kStageBytes);
                } else {
                    if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * C::kStageBytes);
                    bar0 = mapa_shared(&full[stage], leader);
                }
                x_load<CG>(s, mk, mm, &full[stage], bar0, g.a[seg], w.z, w.tm * CG, i,
                           k, h);
#pragma unroll
                for (int b = 0; b < C::kBBlocks; ++b) {
                    const int bb = CG == 2 ? static_cast<int>(rank) : b;
                    if constexpr (EPI == kXGated) {
                        x_load<CG>(s + 32768 * (1 + b), mk, mm, &full[stage], bar0, g.b[bb], w.z,
                                   w.tn, w.tn, k, h);
                    } else {
                        x_load<CG>(s + 32768 * (1 + b), mk, mm, &full[stage], bar0, g.b[seg], w.z,
                                   w.tn * NB, min(w.tn * NB + bb, nb - 1), k, h);
                    }
                }
                if (++stage == C::kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
    }
}

// One lane of the (pair's first) CTA.
template <int CG, int NB, int EPI>
__device__ __forceinline__ void x_mma(const XArgs& g, uint32_t tmem, uint8_t* stages,
                                      uint64_t* full, uint64_t* empty, uint64_t* tfull,
                                      uint64_t* tempty, uint32_t leader, int first, int step) {
    using C = XConfig<CG, NB>;
    constexpr int kM = 128 * CG;
    constexpr int kN = CG == 2 ? 128 * NB : 128;
    int stage = 0, buf = 0;
    uint32_t phase = 0, tphase = 0;
    const uint32_t stage0 = smem_u32(stages);
    for (int u = first; u < g.units; u += step) {
        const XUnit w = x_unit<EPI>(g, u);
        if (x_skips<EPI>(g, w)) continue;
        const int i = w.tm * CG, j = EPI == kXGated ? w.tn : w.tn * NB;
        for (int c = w.c0; c < w.c1; ++c) {
            const int seg = x_third<EPI>(w.z) || (EPI == kXF32 && c >= g.kc0) ? 1 : 0;
            const int k = EPI == kXF32 && seg ? c - g.kc0 : c;
            const int halves = c == g.kc0 - 1 ? g.last0 : (c == g.kc - 1 ? g.last1 : 2);
            const int fa = x_flip(g.a[seg], i, k), fb = x_flip(g.b[seg], j, k);
            // K-major: core matrices 2 KB apart along k, 128 B along rows; 16 deep = two lines.
            // MN-major (a line keeps 64 rows, 1 KB): 128 B apart along k, 1 KB along the other.
            const uint32_t a_lbo = fa ? 128u : 2048u, a_sbo = fa ? 1024u : 128u;
            const uint32_t b_lbo = fb ? 128u : 2048u, b_sbo = fb ? 1024u : 128u;
            const uint32_t a_step = fa ? 256u : 4096u, b_step = fb ? 256u : 4096u;
            const uint32_t idesc = idesc_f16(kM, kN, fa != 0, fb != 0);
            if (!mbar_wait(&tempty[buf], tphase ^ 1u, 1u << 1)) return;
            tc_fence_after();
            const uint32_t d = tmem + static_cast<uint32_t>(buf * NB * 128);
            for (int h = 0; h < halves; ++h) {
                if (!mbar_wait(&full[stage], phase, 1u << 1)) return;
                tc_fence_after();
                const uint32_t sa = stage0 + stage * C::kStageBytes;
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    const uint64_t ah = smem_desc(sa + ks * a_step, a_lbo, a_sbo, kSwizzleNone);
                    const uint64_t al =
                        smem_desc(sa + 16384 + ks * a_step, a_lbo, a_sbo, kSwizzleNone);
#pragma unroll
                    for (int b = 0; b < C::kBBlocks; ++b) {
                        const uint32_t sb = sa + 32768 * (1 + b) + ks * b_step;
                        const uint64_t bh = smem_desc(sb, b_lbo, b_sbo, kSwizzleNone);
                        const uint64_t bl = smem_desc(sb + 16384, b_lbo, b_sbo, kSwizzleNone);
                        mma_f16<CG>(d + b * 128, al, bh, idesc, (h | ks) ? 1u : 0u);
                        mma_f16<CG>(d + b * 128, ah, bl, idesc, 1u);
                    }
                }
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    const uint64_t ah = smem_desc(sa + ks * a_step, a_lbo, a_sbo, kSwizzleNone);
#pragma unroll
                    for (int b = 0; b < C::kBBlocks; ++b) {
                        const uint32_t sb = sa + 32768 * (1 + b) + ks * b_step;
                        mma_f16<CG>(d + b * 128, ah,
                                    smem_desc(sb, b_lbo, b_sbo, kSwizzleNone), idesc, 1u);
                    }
                }
                if constexpr (CG == 1) {
                    mma_commit(&empty[stage]);
                } else {
                    mma_commit_cg2_mc(&empty[stage], static_cast<uint16_t>(3u << leader));
                }
                if (++stage == C::kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if constexpr (CG == 1) {
                mma_commit(&tfull[buf]);
            } else {
                mma_commit_cg2_mc(&tfull[buf], static_cast<uint16_t>(3u << leader));
            }
            if (++buf == 2) {
                buf = 0;
                tphase ^= 1u;
            }
        }
    }
}

// The largest of a value over the epilogue's threads, in a shared slot. Three sets of slots take
// turns: before a tile's barrier the next tile's set is cleared, which was last read before the
// barrier of the tile before.
__device__ __forceinline__ void x_max_into(uint32_t* red, uint32_t bits) {
    const uint32_t m = __reduce_max_sync(0xffffffffu, bits);
    if ((threadIdx.x & 31) == 0) atomicMax(red, m);
}

__device__ __forceinline__ void x_max_into(uint32_t* red, float amax) {
    x_max_into(red, __float_as_uint(amax));
}

// Thread (quarter q, half h, lane) owns row 32 q + lane of the CTA's 128 and, of every 128-column
// block of the tile, columns 64 h .. 64 h + 63: acc[64 b + j] is column 64 h + j of block b.
//
// SPL: the contraction is shared by g.splits CTAs (or pairs) of one cluster, one tile each. A CTA
// leaves its sums in its own shared memory (the stages are read by then) and takes over its share
// of each thread's eight groups of eight columns (at most four): it adds the cluster's sums of
// those, in rank order, through distributed shared memory, and finishes them. (Through L2, with one
// CTA adding and finishing everything, the exchange took 8 us of a 17 us product.)
template <int CG, int NB, int EPI, bool SPL>
__device__ __forceinline__ void x_epilogue(const XArgs& g, uint8_t* stages, uint8_t* epi_smem,
                                           uint32_t* red, uint32_t tmem, uint64_t* tfull,
                                           uint64_t* tempty, uint32_t rank, uint32_t leader,
                                           int first, int step) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int q = warp % 4, half = (warp - kXEpiWarp0) / 4;
    const int row = q * 32 + lane;
    const int et = threadIdx.x - kXEpiWarp0 * 32;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(q * 32) << 16);
    float* box = reinterpret_cast<float*>(epi_smem) + (warp - kXEpiWarp0) * kXBoxFloats;
    int buf = 0, parity = 0;
    uint32_t tphase = 0;
    bool alive = true;  // a wait that gave up: finish without waiting, so every barrier is met
    for (int u = first; u < g.units; u += step) {
        const XUnit w = x_unit<EPI>(g, u);
        if (x_skips<EPI>(g, w)) continue;
        const int i = w.tm * CG + static_cast<int>(rank);
        const bool third = x_third<EPI>(w.z);
        const int mb = third ? g.third.mb : g.mb, nb = third ? g.third.nb : g.nb;
        const int i_in = min(i, mb - 1);
        // this CTA's groups of eight columns: ng of them from ch0
        const int ch0 = SPL ? 8 * w.s / g.splits : 0;
        const int ng = SPL ? 8 * (w.s + 1) / g.splits - ch0 : 8;
        // What the epilogue reads comes eight columns (a turn) at a time through slots of the
        // warp's box, each lane copying what it reads itself: the backward's gate and up in two
        // slots, a split C in four. The first turns while the product is still computed (C read
        // when it was needed made the tail of a 1024 x 4096 product 6 us instead of 4).
        constexpr int kSlots = x_backward<EPI>() ? 2 : 4;
        const bool reads =
            x_backward<EPI>() || ((EPI == kXF32 || EPI == kXSplit) && g.beta != 0.0f);
        const int turns = reads && i < g.mb ? min(NB, g.nb - w.tn * NB) * ng : 0;
        auto fetch = [&](int turn) {
            if (turn < turns) {
                const int b = SPL ? turn / ng : turn >> 3, ch = turn - b * ng;
                const uint32_t dst = smem_u32(box) + (turn % kSlots) * (4096 / kSlots) + lane * 16;
                if constexpr (x_backward<EPI>()) {
                    const long long at =
                        ((static_cast<long long>(i * g.o[0].ldb + w.tn * NB + b) * 2 + half) * 64 +
                         (ch0 + ch) * 8) * kXBlk + row * 4;
                    cp_async_16(dst, g.gate + at);
                    cp_async_16(dst + 512, g.gate + at + 4 * kXBlk);
                    cp_async_16(dst + 1024, g.up + at);
                    cp_async_16(dst + 1536, g.up + at + 4 * kXBlk);
                } else {
                    const int blk = w.z * g.c.bstride + i * g.c.ldb + w.tn * NB + b;
                    const uint8_t* p = g.c.data + static_cast<long long>(blk) * kXBlockBytes +
                                       (half * 8 + ch0 + ch) * kXLineBytes + row * 16;
                    cp_async_16(dst, p);
                    cp_async_16(dst + 512, p + kXBlockBytes / 2);
                }
            }
            cp_async_commit();
        };
        if (reads) {
            __syncwarp();  // the box held the last tile's result
#pragma unroll
            for (int t = 0; t < kSlots; ++t) fetch(t);
        }
        if constexpr (x_backward<EPI>()) {
            for (int b = 0; b < NB; ++b) {
                const int jb = w.tn * NB + b;
                if (i < g.mb && jb < g.nb && w.s == 0) {
                    const long long at = static_cast<long long>(i * g.o[0].ldb + jb) * 16384;
                    for (int x = et * 32; x < 16384; x += kXEpiThreads * 32) {
                        prefetch_l2(g.gate + at + x);
                        prefetch_l2(g.up + at + x);
                    }
                }
            }
        }
        float acc[NB * 64];
#pragma unroll
        for (int j = 0; j < NB * 64; ++j) acc[j] = 0.0f;
        for (int c = w.c0; c < w.c1; ++c) {
            const int seg = x_third<EPI>(w.z) || (EPI == kXF32 && c >= g.kc0) ? 1 : 0;
            const int k = EPI == kXF32 && seg ? c - g.kc0 : c;
            const int a_blk = x_block(g.a[seg], w.z, i_in, k, x_flip(g.a[seg], w.tm * CG, k));
            const float ia = g.a[seg].by_row
                                 ? g.a[seg].inv[static_cast<long long>(a_blk) * kXBlk + row]
                                 : g.a[seg].inv[a_blk];
            float f1[NB], f2[NB];  // the two blocks' 1/s: multiplied together where that is safe
            bool safe = true;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const XOperand& ob = EPI == kXGated ? g.b[b] : g.b[seg];
                const int j0 = EPI == kXGated ? w.tn : w.tn * NB;
                const int j = EPI == kXGated ? w.tn : min(j0 + b, nb - 1);
                const float ib = ob.inv[x_block(ob, w.z, j, k, x_flip(ob, j0, k))];
                f1[b] = fminf(ia, ib);  // else the smaller first: no overflow on the way
                f2[b] = fmaxf(ia, ib);
                const float f = ia * ib;
                safe = safe && f > 1e-30f && f < 1e30f;
            }
            if (alive) alive = mbar_wait(&tfull[buf], tphase, 1u << 2);
            alive = __all_sync(0xffffffffu, alive);
            tc_fence_after();
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    float r[16];
                    tmem_ld_32x32b_x16(lanes + static_cast<uint32_t>(buf * NB * 128 + b * 128 +
                                                                     half * 64 + t * 16), r);
                    float* a = acc + b * 64 + t * 16;
                    if (safe) {
                        const float f = f1[b] * f2[b];
#pragma unroll
                        for (int j = 0; j < 16; j += 2) fma2(a[j], a[j + 1], r[j], r[j + 1], f);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) a[j] = fmaf(r[j] * f1[b], f2[b], a[j]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 1) {
                    mbar_arrive(&tempty[buf]);
                } else {
                    mbar_arrive_cluster(mapa_shared(&tempty[buf], leader));
                }
            }
            if (++buf == 2) {
                buf = 0;
                tphase ^= 1u;
            }
        }
        if constexpr (SPL) {  // (from here on at the front of acc)
            float4* mine = reinterpret_cast<float4*>(stages) + et;
#pragma unroll
            for (int j = 0; j < NB * 16; ++j)
                mine[j * kXEpiThreads] = make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2],
                                                     acc[4 * j + 3]);
            cluster_sync();
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int ch = 0; ch < 8; ++ch) {
                    float* v = acc + b * 64 + ch * 8;
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
                    if (ch < 4 && ch < ng) {
                        for (int r = 0; r < g.splits; ++r) {
                            const uint32_t at = mapa_shared(
                                mine + (b * 16 + (ch0 + ch) * 2) * kXEpiThreads,
                                r * CG + rank);
                            const float4 x = ld_cluster_v4(at);
                            const float4 y = ld_cluster_v4(at + kXEpiThreads * 16);
                            v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
                            v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
                        }
                    }
                }
            }
        }
        const bool row_block = i < mb;
        const int m = third ? g.third.m : g.m, n = third ? g.third.n : g.n;
        float* const out = third ? g.third.out : g.out + w.z * g.out_bs;
        const long long ld = third ? g.third.ld : g.ld;

        if constexpr (EPI == kXF32 || EPI == kXSplit) {
            if (reads) {  // alpha acc + beta C
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int jb = w.tn * NB + b;
                    if (row_block && jb < g.nb) {
                        const float f = g.c.inv[w.z * g.c.bstride + i * g.c.ldb + jb] * g.beta;
#pragma unroll
                        for (int ch = 0; ch < 8; ++ch) {
                            if (SPL && ch >= ng) break;
                            const int turn = b * ng + ch;
                            const uint32_t src =
                                smem_u32(box) + (turn % kSlots) * (4096 / kSlots) + lane * 16;
                            cp_async_wait<kSlots - 1>();
                            const float4 hq = ld_shared_v4(src), lq = ld_shared_v4(src + 512);
                            fetch(turn + kSlots);
                            const float hs[4] = {hq.x, hq.y, hq.z, hq.w};
                            const float ls[4] = {lq.x, lq.y, lq.z, lq.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 hf =
                                    __half22float2(*reinterpret_cast<const __half2*>(&hs[e]));
                                const float2 lf =
                                    __half22float2(*reinterpret_cast<const __half2*>(&ls[e]));
                                float* v = acc + b * 64 + ch * 8 + e * 2;
                                v[0] = fmaf(hf.x + lf.x, f, v[0] * g.alpha);
                                v[1] = fmaf(hf.y + lf.y, f, v[1] * g.alpha);
                            }
                        }
                    }
                }
                cp_async_wait<0>();
            } else if (EPI == kXSplit && g.alpha != 1.0f) {
#pragma unroll
                for (int j = 0; j < NB * 64; ++j) acc[j] *= g.alpha;
            }
        }

        if constexpr (x_fp32<EPI>() && SPL) {
            const int grow = i * kXBlk + row;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int ch = 0; ch < 4; ++ch) {
                    const int col = (w.tn * NB + b) * kXBlk + half * 64 + (ch0 + ch) * 8;
                    if (ch < ng && grow < m) {
                        float* dst = out + static_cast<long long>(grow) * ld + col;
                        const float* v = acc + b * 64 + ch * 8;
                        if (col + 8 <= n && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
                            *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
                            *reinterpret_cast<float4*>(dst + 4) =
                                make_float4(v[4], v[5], v[6], v[7]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (col + e < n) dst[e] = v[e];
                        }
                    }
                }
            }
        } else if constexpr (x_fp32<EPI>()) {
            // through a 32 x 32 box (16-byte column group c of row r at c ^ (r % 8): no bank
            // conflicts either way), so that eight lanes write 128 bytes of a row
            const bool wide = ((reinterpret_cast<uintptr_t>(out) & 15u) == 0) && (ld & 3) == 0;
            const uint32_t box0 = smem_u32(box);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const float* v = acc + b * 64 + t * 32 + c * 4;
                        st_shared_v4(box0 + lane * 128 + ((c ^ (lane & 7)) << 4), v[0], v[1], v[2],
                                     v[3]);
                    }
                    __syncwarp();
                    const int col = (w.tn * NB + b) * kXBlk + half * 64 + t * 32 + (lane & 7) * 4;
                    const int row0 = i * kXBlk + q * 32 + (lane >> 3);
                    if (row_block && col < n) {
                        float* dst = out + static_cast<long long>(row0) * ld + col;
                        const long long step = 4 * ld;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int r = e * 4 + (lane >> 3);
                            const float4 v =
                                ld_shared_v4(box0 + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
                            if (row0 + e * 4 < m) {
                                if (wide && col + 4 <= n) {
                                    *reinterpret_cast<float4*>(dst) = v;
                                } else {
                                    dst[0] = v.x;
                                    if (col + 1 < n) dst[1] = v.y;
                                    if (col + 2 < n) dst[2] = v.z;
                                    if (col + 3 < n) dst[3] = v.w;
                                }
                            }
                            dst += step;
                        }
                    }
                }
            }
        }

        if constexpr (EPI == kXSplit) {
            uint32_t* slot = red + parity * 8;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                x_max_into(slot + b, largest<64>(acc + b * 64));
            }
            parity = parity == 2 ? 0 : parity + 1;
            if (et < 8) red[parity * 8 + et] = 0u;
            epi_bar();
            uint32_t top_of[3] = {slot[0], slot[1], slot[2]};
            if constexpr (SPL) {
                cluster_sync();
                for (int r = 0; r < g.splits; ++r) {
                    const uint32_t at = mapa_shared(slot, r * CG + rank);
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        top_of[e] = max(top_of[e], ld_cluster_u32(at + e * 4));
                }
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int jb = w.tn * NB + b;
                if (row_block && jb < g.nb) {
                    float s, inv;
                    const int blk = w.z * g.o[0].bstride + i * g.o[0].ldb + jb;
                    split_scale(__uint_as_float(top_of[b]), s, inv);
                    if (et == 0 && w.s == 0) g.o[0].inv[blk] = inv;
                    uint8_t* dst = g.o[0].data + static_cast<long long>(blk) * kXBlockBytes;
#pragma unroll
                    for (int ch = 0; ch < 8; ++ch)
                        if (ch < ng)
                            store_split8(dst, half * 8 + ch0 + ch, row, acc + b * 64 + ch * 8, s);
                }
            }
        }

        if constexpr (EPI == kXGated) {
            // acc: 64 gate columns, then the same 64 up columns. Row maxima of h, gate and up go
            // through the (otherwise idle) boxes: two sets of [3][2 halves][128] take turns.
            float* rowmax = reinterpret_cast<float*>(epi_smem) + (parity & 1) * (6 * kXBlk);
            ++parity;
            const int blk = i_in * g.o[0].ldb + w.tn;
            if (g.gate != nullptr) {
                rowmax[(2 + half) * kXBlk + row] = largest<64>(acc);
                rowmax[(4 + half) * kXBlk + row] = largest<64>(acc + 64);
            }
            const long long at =
                ((static_cast<long long>(blk) * 2 + half) * 64 + ch0 * 8) * kXBlk + row * 4;
            const bool save = g.gate != nullptr && row_block;
            // the stores of the pre-activations go out between the activations' arithmetic
            with_act(g.store_h ? g.act : kXActNone, [&](auto kind) {
#pragma unroll
                for (int j = 0; j < 64; j += 4) {
                    if (SPL && j >= ng * 8) break;
                    if (save) {
                        *reinterpret_cast<float4*>(g.gate + at + j * kXBlk) =
                            make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
                        *reinterpret_cast<float4*>(g.up + at + j * kXBlk) = make_float4(
                            acc[64 + j], acc[64 + j + 1], acc[64 + j + 2], acc[64 + j + 3]);
                    }
#pragma unroll
                    for (int e = j; e < j + 4; e += 2) {
                        float2 ac, sl;
                        act_slope2<decltype(kind)::value>(make_float2(acc[e], acc[e + 1]), ac, sl);
                        const float2 h = mul2(ac, make_float2(acc[64 + e], acc[64 + e + 1]));
                        acc[e] = h.x, acc[e + 1] = h.y;
                    }
                }
            });
            if (g.store_h) rowmax[half * kXBlk + row] = largest<64>(acc);
            epi_bar();
            float hm = fmaxf(rowmax[row], rowmax[kXBlk + row]);
            float gm = rowmax[(2 + half) * kXBlk + row], um = rowmax[(4 + half) * kXBlk + row];
            if constexpr (SPL) {
                cluster_sync();
                for (int r = 0; r < g.splits; ++r) {
                    const uint32_t from = mapa_shared(rowmax + row, r * CG + rank);
                    hm = fmaxf(hm, fmaxf(ld_cluster_f32(from), ld_cluster_f32(from + kXBlk * 4)));
                    gm = fmaxf(gm, ld_cluster_f32(from + (2 + half) * kXBlk * 4));
                    um = fmaxf(um, ld_cluster_f32(from + (4 + half) * kXBlk * 4));
                }
            }
            if (row_block) {
                if (g.gate != nullptr && w.s == 0) {
                    float* to = g.gmax + static_cast<long long>(blk) * 4 * kXBlk + half * kXBlk +
                                row;
                    to[0] = gm;
                    to[2 * kXBlk] = um;
                }
                if (g.store_h) {
                    float s, inv;
                    split_scale(hm, s, inv);
                    if (half == 0 && w.s == 0)
                        g.o[0].inv[static_cast<long long>(blk) * kXBlk + row] = inv;
                    uint8_t* dst = g.o[0].data + static_cast<long long>(blk) * kXBlockBytes;
#pragma unroll
                    for (int ch = 0; ch < 8; ++ch)
                        if (ch < ng) store_split8(dst, half * 8 + ch0 + ch, row, acc + ch * 8, s);
                }
            }
        }

        if constexpr (x_backward<EPI>()) {
            // acc: the gradient of h. The three outputs are stored under scales from bounds, the
            // largest over a block's rows of
            // |dgate| <= 1.13 max|dh| max|up|, |dup| <= max|dh| max|gate|, |h| <= max|gate| max|up|
            // (the maxima over the row's 64 columns), and the largest |hi| is kept. On ordinary
            // rows a bound is up to three powers of two too large, which leaves an entry its 22
            // bits down to 2^-14 of the largest. Where gates are saturated, act and act' are tiny
            // and it can be any number too large (2^25 for SiLU at -20): such blocks are computed
            // once more by the next launch (kXGatedAgain), which looks for their largest values
            // first. (8192 x 4096 x 11008: 1800 us with bounds alone, 1835 so, and 5 for a next
            // launch that finds nothing to do; 2070 in one launch that stores loose blocks twice,
            // because a pair's 128 sums a thread stay alive for that.)
            // A row without a gradient has no part in any sum over rows, whatever is in it: its
            // dgate, dup and h are zeros (as computed they would be 0 times gate and up, which need
            // not be finite there), and its size does not count.
            uint32_t* slot = red + parity * 8;
            const int grow = i * kXBlk + row;
            const bool live = grow < g.m && g.live[grow] != 0;
            auto gathered = [&]() {
                parity = parity == 2 ? 0 : parity + 1;
                if (et < 8) red[parity * 8 + et] = 0u;
                epi_bar();
            };
            uint32_t top_of[NB * 3] = {};
            if constexpr (EPI == kXGatedBwd) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int jb = w.tn * NB + b;
                    if (row_block && jb < g.nb) {
                        const float* from =
                            g.gmax + static_cast<long long>(i * g.o[0].ldb + jb) * 4 * kXBlk +
                            half * kXBlk + row;
                        const float gm = live ? from[0] : 0.0f, um = live ? from[2 * kXBlk] : 0.0f;
                        const float dm = largest<64>(acc + b * 64);
                        const float top = 3.402823466e38f;
                        x_max_into(slot + b * 3, fminf(dm * um * kXMaxSlope, top));
                        x_max_into(slot + b * 3 + 1, fminf(dm * gm, top));
                        x_max_into(slot + b * 3 + 2, fminf(gm * um, top));
                    }
                }
                gathered();
#pragma unroll
                for (int e = 0; e < NB * 3; ++e) top_of[e] = slot[e];
                if constexpr (SPL) {
                    cluster_sync();
                    for (int r = 0; r < g.splits; ++r) {
                        const uint32_t at = mapa_shared(slot, r * CG + rank);
#pragma unroll
                        for (int e = 0; e < NB * 3; ++e)
                            top_of[e] = max(top_of[e], ld_cluster_u32(at + e * 4));
                    }
                }
            }
            // kXGatedAgain takes the maxima in a pass of its own
#pragma unroll 1
            for (int pass = EPI == kXGatedAgain ? 0 : 1; pass < 2; ++pass) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int jb = w.tn * NB + b;
                    if (!row_block || jb >= g.nb) continue;
                    const int blk = i * g.o[0].ldb + jb;
                    const long long off = static_cast<long long>(blk) * kXBlockBytes;
                    float sc[3], most[3] = {};
                    __half2 hi[3] = {};
#pragma unroll
                    for (int e = 0; e < 3; ++e) {
                        const uint32_t top = top_of[b * 3 + e];
                        float inv;
                        split_scale(__uint_as_float(max(top, 1u)), sc[e], inv);
                        if (pass == 1 && et == 0 && w.s == 0)
                            g.o[e].inv[blk] = top != 0u ? inv : 1.0f;  // (a block of zeros)
                    }
                    with_act(g.act, [&](auto kind) {
#pragma unroll
                        for (int ch = 0; ch < 8; ++ch) {
                            if (SPL && ch >= ng) break;
                            float out3[3][8];   // dgate, dup, h
                            const int turn = b * ng + ch;
                            const uint32_t src =
                                smem_u32(box) + (turn % kSlots) * (4096 / kSlots) + lane * 16;
                            cp_async_wait<kSlots - 1>();
                            const float4 g0 = ld_shared_v4(src), g1 = ld_shared_v4(src + 512);
                            const float4 u0 = ld_shared_v4(src + 1024);
                            const float4 u1 = ld_shared_v4(src + 1536);
                            fetch(turn + kSlots);
                            const float gs[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
                            const float us[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
#pragma unroll
                            for (int x = 0; x < 8; x += 2) {
                                const float* v = acc + b * 64 + ch * 8 + x;
                                const float2 dh = make_float2(v[0], v[1]);
                                const float2 u = make_float2(us[x], us[x + 1]);
                                float2 ac, sl;
                                act_slope2<decltype(kind)::value>(make_float2(gs[x], gs[x + 1]), ac,
                                                                  sl);
                                const float2 p = mul2(mul2(dh, u), sl), q = mul2(dh, ac);
                                const float2 h = mul2(ac, u);
                                out3[0][x] = p.x, out3[0][x + 1] = p.y;
                                out3[1][x] = q.x, out3[1][x + 1] = q.y;
                                out3[2][x] = h.x, out3[2][x + 1] = h.y;
                            }
                            if (!live) {
#pragma unroll
                                for (int x = 0; x < 8; ++x)
                                    out3[0][x] = out3[1][x] = out3[2][x] = 0.0f;
                            }
#pragma unroll
                            for (int e = 0; e < 3; ++e) {
                                if (pass == 0)
                                    most[e] = fmaxf(most[e], largest<8>(out3[e]));
                                else
                                    store_split8(g.o[e].data + off, half * 8 + ch0 + ch, row,
                                                 out3[e], sc[e],
                                                 EPI == kXGatedBwd ? &hi[e] : nullptr);
                            }
                        }
                    });
#pragma unroll
                    for (int e = 0; e < 3; ++e) {
                        if (pass == 0) {
                            x_max_into(slot + e, most[e]);
                        } else if constexpr (EPI == kXGatedBwd) {
                            const __half t = __hmax(__low2half(hi[e]), __high2half(hi[e]));
                            x_max_into(g.tops + static_cast<long long>(blk) * 4 + e,
                                       sc[e] == kXMostScale
                                           ? kXTight  // zeros, or nothing better
                                           : static_cast<uint32_t>(__half_as_ushort(t)));
                        }
                    }
                }
                if constexpr (EPI == kXGatedAgain) {
                    if (pass == 0) {
                        gathered();
#pragma unroll
                        for (int e = 0; e < NB * 3; ++e) top_of[e] = slot[e];
                        cp_async_wait<0>();
#pragma unroll
                        for (int t = 0; t < kSlots; ++t) fetch(t);
                    }
                }
            }
        }
        if constexpr (x_backward<EPI>()) cp_async_wait<0>();
        if constexpr (SPL) cluster_sync();  // nobody leaves while its sums or maxima are read
    }
}

template <int CG, int NB, int EPI, bool SPL = false>
__global__ void __launch_bounds__(kXThreads, 1)
    split_mm_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mm,
                    const __grid_constant__ XArgs g) {
    using C = XConfig<CG, NB>;
    extern __shared__ __align__(1024) uint8_t x_smem_raw[];
    uint8_t* stages = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(x_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* epi_smem = stages + C::kStageArea;
    uint64_t* bars = reinterpret_cast<uint64_t*>(epi_smem + C::kEpiBytes);
    uint64_t* full = bars;
    uint64_t* empty = full + C::kStages;
    uint64_t* tfull = empty + C::kStages;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
    uint32_t* red = tmem_holder + 1;                       // three sets of eight block maxima
    // the cluster barriers that the epilogue warps of an SPL kernel meet at
    constexpr int kSplitSyncs = !SPL ? 0 : x_fp32<EPI>() ? 2 : 3;

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    // CTAs 2 p and 2 p + 1 of a cluster are a pair
    const uint32_t rank = CG == 1 ? 0u : cluster_ctarank() & 1u;
    const uint32_t leader = CG == 1 ? 0u : cluster_ctarank() & ~1u;
    const int first = static_cast<int>(blockIdx.x) / CG, step = static_cast<int>(gridDim.x) / CG;

    grid_dependents_go();
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&tfull[s], 1);
            mbar_init(&tempty[s], 8 * CG);
        }
        mbar_init(drain, 1);
        for (int s = 0; s < 24; ++s) red[s] = 0u;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&mk);
        tma_prefetch_desc(&mm);
    }
    if (warp == 1) {
        if constexpr (CG == 1) {
            tmem_alloc(tmem_holder, C::kTmemCols);
        } else {
            tmem_alloc_cg2(tmem_holder, C::kTmemCols);
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    grid_wait();  // before anything of the launch before is read or overwritten

    bool work = true;
    if constexpr (EPI == kXGatedAgain) {  // most often none of the tiles has to be done again
        bool any = false;
        for (int u = first + static_cast<int>(threadIdx.x) * step; u < g.units;
             u += kXThreads * step)
            any = any || !x_skips<EPI>(g, x_unit<EPI>(g, u));
        work = __syncthreads_or(any) != 0;
    }
    if (!work) {
        // straight to the end
    } else if (warp == 0) {
        if (lane == 0)
            x_producer<CG, NB, EPI>(g, &mk, &mm, stages, full, empty, rank, leader, first, step);
        __syncwarp();
#pragma unroll
        for (int s = 0; s < kSplitSyncs; ++s) cluster_sync();
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            x_mma<CG, NB, EPI>(g, tmem, stages, full, empty, tfull, tempty, leader, first, step);
            // every MMA issued above must finish before TMEM is released, also on an error exit
            if constexpr (CG == 1) {
                mma_commit(drain);
            } else {
                mma_commit_cg2(drain);
            }
            mbar_wait(drain, 0, 1u << 1);
        }
        __syncwarp();
#pragma unroll
        for (int s = 0; s < kSplitSyncs; ++s) cluster_sync();
    } else {
        x_epilogue<CG, NB, EPI, SPL>(g, stages, epi_smem, red, tmem, tfull, tempty, rank, leader,
                                     first, step);
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (CG == 1) {
            tmem_dealloc(tmem, C::kTmemCols);
        } else {
            tmem_dealloc_cg2(tmem, C::kTmemCols);
        }
    }
}

}  // namespace mfk
