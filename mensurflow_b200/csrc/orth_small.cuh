// The orthogonalised update of small matrices in one launch: the smaller side at most 128, the
// larger at most 1024.
//
// A matrix is k x n (k <= 128) or its transpose; a cluster of ceil(n / 128) CTAs has one 128 x 128
// block of x each, in fp32 registers and, as the fp16 (hi, lo) pair that split_mm.cuh describes, in
// shared memory. One step is three 128 x 128 x 128 products on tcgen05 with nothing of it in
// global memory:
//     g = x x^T: each CTA its block's part, the parts added through distributed shared memory in
//         rank order (every CTA adds all of them, so all hold the same g);
//     p = b g + c g g;
//     x = a x + p x.
// Sums between products stay in fp32 registers (a thread has one row and 32 columns); only the
// operands are split. Products are as wide and as deep as the matrix in steps of 16, and a thread
// whose columns lie outside does nothing. Bound by latency: a product is up to 24 MMAs of 64 cycles
// and longer again for the way TMEM -> registers -> shared memory; 48 matrices of 64 x 128, five
// steps: 41 us, against 115 us as seventeen launches of the general kernels (and 52 us with eight
// warps of 64 columns a thread).
#pragma once

#include "split_mm.cuh"

namespace mfk {

constexpr int kOrthWarps = 16;             // with the values, and one that issues the MMAs
constexpr int kOrthValues = kOrthWarps * 32;
constexpr int kOrthThreads = kOrthValues + 32;
constexpr int kOrthCols = 32;              // of a thread
constexpr int kOrthSmem = 3 * kXBlockBytes + 1024 + 512;
constexpr int kOrthMaxRanks = 8;

struct OrthSmallArgs {
    const float* u;
    long long rs, bs;
    float* out;
    long long ld, out_bs;
    int rows, cols;       // of a matrix
    int tall;             // rows > cols: blocks down the rows
    int steps;
    float a, b, c, eps;
};

__device__ __forceinline__ double ld_cluster_f64(uint32_t addr) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
    return v;
}

// D (128 x n) = A B over `depth`, both in steps of 16: the lo products first.
__device__ __forceinline__ void orth_mma(uint32_t d, uint32_t a, int a_flip, uint32_t b, int b_flip,
                                         int n, int depth) {
    // blocks with all 16 lines: K-major 2 KB apart along k, 128 B along rows; MN-major 128 B
    // along k, 2 KB along the other
    const uint32_t a_lbo = a_flip ? 128u : 2048u, a_sbo = a_flip ? 2048u : 128u;
    const uint32_t b_lbo = b_flip ? 128u : 2048u, b_sbo = b_flip ? 2048u : 128u;
    const uint32_t a_step = a_flip ? 256u : 4096u, b_step = b_flip ? 256u : 4096u;
    const uint32_t idesc = idesc_f16(128, (n + 15) / 16 * 16, a_flip != 0, b_flip != 0);
    const int ks_end = (depth + 15) / 16;
    for (int ks = 0; ks < ks_end; ++ks) {
        const uint32_t sa = a + ks * a_step, sb = b + ks * b_step;
        const uint64_t ah = smem_desc(sa, a_lbo, a_sbo, kSwizzleNone);
        const uint64_t al = smem_desc(sa + kXBlockBytes / 2, a_lbo, a_sbo, kSwizzleNone);
        const uint64_t bh = smem_desc(sb, b_lbo, b_sbo, kSwizzleNone);
        const uint64_t bl = smem_desc(sb + kXBlockBytes / 2, b_lbo, b_sbo, kSwizzleNone);
        mma_f16<1>(d, al, bh, idesc, ks ? 1u : 0u);
        mma_f16<1>(d, ah, bl, idesc, 1u);
    }
    for (int ks = 0; ks < ks_end; ++ks)
        mma_f16<1>(d, smem_desc(a + ks * a_step, a_lbo, a_sbo, kSwizzleNone),
                   smem_desc(b + ks * b_step, b_lbo, b_sbo, kSwizzleNone), idesc, 1u);
}

__device__ __forceinline__ void orth_bar() {
    asm volatile("bar.sync 1, %0;" ::"n"(kOrthValues) : "memory");
}

// The largest magnitude over all values. Two sets of slots take turns; a set is next
// written two calls later, behind the barriers in between.
__device__ __forceinline__ float orth_max(uint32_t* red, int& turn, float amax) {
    uint32_t* slot = red + turn * kOrthWarps;
    turn ^= 1;
    const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = m;
    orth_bar();
    return __uint_as_float(
        __reduce_max_sync(0xffffffffu, slot[threadIdx.x & (kOrthWarps - 1)]));
}

// v (one row, 32 columns a thread, the first `groups` x 16 of them in use) as a split block in
// shared memory; returns 1/s.
__device__ __forceinline__ float orth_split(uint8_t* block, const float* v, int part, int row,
                                            int groups, uint32_t* red, int& turn) {
    float s, inv, m = 0.0f;
    if (groups > 0) m = largest<kOrthCols>(v);
    split_scale(orth_max(red, turn, m), s, inv);
#pragma unroll
    for (int ch = 0; ch < kOrthCols / 8; ++ch)
        if (ch < groups * 2) store_split8(block, part * (kOrthCols / 8) + ch, row, v + ch * 8, s);
    fence_proxy_async_smem();
    return inv;
}

__global__ void __launch_bounds__(kOrthThreads, 1)
    orth_small_kernel(const __grid_constant__ OrthSmallArgs g) {
    extern __shared__ __align__(1024) uint8_t orth_smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(orth_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* sx = base;                          // x
    uint8_t* sg = base + kXBlockBytes;           // g
    uint8_t* sp = base + 2 * kXBlockBytes;       // p, and before it the parts of g in fp32
    uint64_t* done = reinterpret_cast<uint64_t*>(base + 3 * kXBlockBytes);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done + 1);
    uint32_t* red = tmem_holder + 2;             // two sets of slots
    double* sums = reinterpret_cast<double*>(red + 2 * kOrthWarps);  // the warps', then the CTA's
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int ranks = static_cast<int>(cluster_nctarank());
    const int rank = static_cast<int>(cluster_ctarank());
    const long long z = blockIdx.x / ranks;
    const int k = g.tall ? g.cols : g.rows;

    if (threadIdx.x == 0) {
        mbar_init(done, 1);
        fence_barrier_init();
    }
    if (warp == kOrthWarps) tmem_alloc(tmem_holder, 128);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;

    if (warp == kOrthWarps) {
        // One lane issues; the three barriers a step are the other warps' word that the operands
        // of the next product lie in shared memory.
        const uint32_t ax = smem_u32(sx), ag = smem_u32(sg), ap = smem_u32(sp);
        const int own = min(128, (g.tall ? g.rows : g.cols) - rank * 128);
        cluster_sync();   // with the norm
        for (int step = 0; step < g.steps; ++step) {
#pragma unroll 1
            for (int i = 0; i < 3; ++i) {
                __syncthreads();
                if (lane == 0) {
                    tc_fence_after();
                    if (i == 0) {
                        orth_mma(tmem, ax, g.tall, ax, g.tall, k, own);
                    } else if (i == 1) {
                        orth_mma(tmem, ag, 0, ag, 0, k, k);
                    } else if (g.tall) {
                        orth_mma(tmem, ax, 0, ap, 0, k, k);
                    } else {
                        orth_mma(tmem, ap, 0, ax, 1, own, k);
                    }
                    mma_commit(done);
                }
                __syncwarp();
                if (i == 0 && ranks > 1) {
                    cluster_sync();
                    cluster_sync();
                }
            }
        }
    } else {
        const int q = warp % 4, part = warp / 4;   // TMEM lanes, columns 32 part ..
        const int row = q * 32 + lane;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(q * 32) << 16) + part * kOrthCols;
        const int r0 = g.tall ? rank * 128 : 0, c0 = g.tall ? 0 : rank * 128;
        // this thread's sixteens of columns in use: of the k x k matrices, and of x
        const int gk = max(0, min(2, (k - part * kOrthCols + 15) / 16));
        const int own = g.tall ? k : min(128, g.cols - rank * 128);
        const int gx = max(0, min(2, (own - part * kOrthCols + 15) / 16));
        int turn = 0;
        uint32_t phase = 0;
        float x[kOrthCols], acc[kOrthCols];
        // the block through shared memory, so that global rows are read along
        float* stage = reinterpret_cast<float*>(sg);     // [128][129], in g and p
        {
            const float* u = g.u + z * g.bs;
#pragma unroll 8
            for (int i = threadIdx.x; i < 128 * 128; i += kOrthValues) {
                const int r = i >> 7, c = i & 127;
                const bool in = r0 + r < g.rows && c0 + c < g.cols;
                stage[r * 129 + c] =
                    in ? u[static_cast<long long>(r0 + r) * g.rs + c0 + c] : 0.0f;
            }
            orth_bar();
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < kOrthCols; ++j) {
                x[j] = stage[row * 129 + part * kOrthCols + j];
                sum += static_cast<double>(x[j]) * static_cast<double>(x[j]);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) sums[warp] = sum;
            orth_bar();
            if (threadIdx.x == 0) {
                double t = 0.0;
                for (int w = 0; w < kOrthWarps; ++w) t += sums[w];
                sums[kOrthWarps] = t;
            }
            cluster_sync();
            double total = 0.0;
            for (int r = 0; r < ranks; ++r)
                total += ld_cluster_f64(mapa_shared(sums + kOrthWarps, r));
            // in two factors, a power of two and the rest: alone it leaves fp32's normal range
            // where the norm is above 2^126
            const double f = 1.0 / (sqrt(total) + static_cast<double>(g.eps));
            const int e = static_cast<int>((__double_as_longlong(f) >> 52) & 0x7ff) - 1023;
            const int half = max(-100, min(100, e / 2));
            const float f1 = __int_as_float((127 + half) << 23);
            const float f2 = static_cast<float>(
                f * __longlong_as_double(static_cast<long long>(1023 - half) << 52));
#pragma unroll
            for (int j = 0; j < kOrthCols; ++j) x[j] = (x[j] * f1) * f2;
        }
        bool alive = true;  // a wait that gave up: finish without waiting, every barrier is met
        auto product_done = [&]() {
            if (alive) alive = mbar_wait(done, phase, 1u << 2);
            alive = __all_sync(0xffffffffu, alive);
            phase ^= 1u;
            tc_fence_after();
        };
        for (int step = 0; step < g.steps; ++step) {
            const float xi = orth_split(sx, x, part, row, gx, red, turn);
            tc_fence_before();
            __syncthreads();
            product_done();
            // g; its rows from k on come from columns of x that no thread has written (x on its
            // side), and would set the scale
#pragma unroll
            for (int t = 0; t < kOrthCols / 16; ++t) {
                float r[16];
                if (t < gk) tmem_ld_32x32b_x16(lanes + t * 16, r);
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    acc[t * 16 + j] = t < gk && row < k ? (r[j] * xi) * xi : 0.0f;
            }
            if (ranks > 1) {
                float4* mine = reinterpret_cast<float4*>(sp) + threadIdx.x;
#pragma unroll
                for (int j = 0; j < kOrthCols / 4; ++j)
                    if (j < gk * 4)
                        mine[j * kOrthValues] = make_float4(acc[4 * j], acc[4 * j + 1],
                                                            acc[4 * j + 2], acc[4 * j + 3]);
                cluster_sync();
#pragma unroll
                for (int j = 0; j < kOrthCols; ++j) acc[j] = 0.0f;
                for (int r = 0; r < ranks; ++r) {
                    const uint32_t at = mapa_shared(mine, r);
#pragma unroll
                    for (int j = 0; j < kOrthCols / 4; ++j) {
                        if (j < gk * 4) {
                            const float4 v = ld_cluster_v4(at + j * kOrthValues * 16);
                            acc[4 * j] += v.x;
                            acc[4 * j + 1] += v.y;
                            acc[4 * j + 2] += v.z;
                            acc[4 * j + 3] += v.w;
                        }
                    }
                }
                cluster_sync();
            }
            const float gi = orth_split(sg, acc, part, row, gk, red, turn);
            tc_fence_before();
            __syncthreads();
            product_done();
            // p = b g + c g g
#pragma unroll
            for (int t = 0; t < kOrthCols / 16; ++t) {
                float r[16];
                if (t >= gk) break;
                tmem_ld_32x32b_x16(lanes + t * 16, r);
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    acc[t * 16 + j] = fmaf(g.b, acc[t * 16 + j], ((r[j] * gi) * gi) * g.c);
            }
            const float pi = orth_split(sp, acc, part, row, gk, red, turn);
            tc_fence_before();
            __syncthreads();
            product_done();
            // x = a x + p x
#pragma unroll
            for (int t = 0; t < kOrthCols / 16; ++t) {
                float r[16];
                if (t >= gx) break;
                tmem_ld_32x32b_x16(lanes + t * 16, r);
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    x[t * 16 + j] = fmaf(g.a, x[t * 16 + j], (r[j] * pi) * xi);
            }
            tc_fence_before();
        }
        // out, along the rows again
#pragma unroll
        for (int j = 0; j < kOrthCols; ++j) stage[row * 129 + part * kOrthCols + j] = x[j];
        orth_bar();
        float* out = g.out + z * g.out_bs;
#pragma unroll 8
        for (int i = threadIdx.x; i < 128 * 128; i += kOrthValues) {
            const int r = i >> 7, c = i & 127;
            if (r0 + r < g.rows && c0 + c < g.cols)
                out[static_cast<long long>(r0 + r) * g.ld + c0 + c] = stage[r * 129 + c];
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kOrthWarps) {
        tc_fence_after();
        tmem_dealloc(tmem, 128);
    }
}

}  // namespace mfk
