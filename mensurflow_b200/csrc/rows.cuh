// The gated feed-forward block for a few rows (decoding): y = (act(x Wg) * (x Wu)) Wd for up to
// 16 rows, fp32 FMAs on the weights as they lie.
//
// Bound by HBM: each weight is read once and used for every row; at 16 rows that is 32 flops per
// 4 bytes, still below the FMA units' rate. (The tensor-core path would first write the weights'
// split form: three times the bytes.) Two launches: gate, up and the activation into h, then the
// down projection. Of the output columns each cluster owns a tile; its CTAs share the depth and
// add their sums through distributed shared memory in rank order, so no partial sum goes through
// HBM and the result does not depend on timing. The second launch starts while the first still
// runs (programmatic dependent launch) and has its first weights on the way before it waits for h.
//
// Two forms, by how the weights lie: rows_n (output columns contiguous) gives each lane VEC
// columns, and the warps of a CTA alternate rows of the weights; rows_k (depth contiguous, the
// [outputs, inputs] layout) gives each warp two outputs, and its lanes the depth. The rows' values
// come from shared memory, transposed for rows_n so that one broadcast load serves four rows.
#pragma once

#include "split_mm.cuh"

namespace mfk {

constexpr int kRowsMax = 16;
constexpr int kRowsXBytes = 32768;      // of x staged at a time
constexpr int kRowsRedBytes = 32768;    // sums of four warps

struct RowsArgs {
    const float* x;          // element (r, k) at x[r*x_rs + k*x_cs]
    long long x_rs, x_cs;
    const float* w0;         // the weights (gate), row stride ld0
    const float* w1;         // up
    long long ld0, ld1;
    int rows, depth, cols;   // of the product
    float* out;              // rows x cols, row stride ldo
    long long ldo;
    int act;
    int wait;                // x comes from the launch before
};

__device__ __forceinline__ void grid_dependents_go() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ void grid_wait() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ uint32_t cluster_nctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

template <int VEC>
struct RowsVec {
    float v[VEC];
};

template <int VEC>
__device__ __forceinline__ RowsVec<VEC> rows_load(const float* p) {
    RowsVec<VEC> r;
    if constexpr (VEC == 4) {
        const float4 q = __ldcs(reinterpret_cast<const float4*>(p));
        r.v[0] = q.x, r.v[1] = q.y, r.v[2] = q.z, r.v[3] = q.w;
    } else if constexpr (VEC == 2) {
        const float2 q = __ldcs(reinterpret_cast<const float2*>(p));
        r.v[0] = q.x, r.v[1] = q.y;
    } else {
        r.v[0] = __ldcs(p);
    }
    return r;
}

// The cluster's sums of `tile` columns (res[(r * tile + c) * W + i], W = 2 with gate and up) in
// rank order, the activation, and the store.
template <int W>
__device__ __forceinline__ void rows_finish(const RowsArgs& g, float* res, int tile, int col0) {
    const uint32_t ranks = cluster_nctarank(), rank = cluster_ctarank();
    __syncthreads();
    cluster_sync();
    for (int i = static_cast<int>(rank) * 256 + threadIdx.x; i < g.rows * tile;
         i += static_cast<int>(ranks) * 256) {
        float s[W];
#pragma unroll
        for (int e = 0; e < W; ++e) s[e] = 0.0f;
        for (uint32_t q = 0; q < ranks; ++q) {
            const uint32_t at = mapa_shared(res + i * W, q);
#pragma unroll
            for (int e = 0; e < W; ++e) s[e] += ld_cluster_f32(at + e * 4);
        }
        const int r = i / tile, c = col0 + i - r * tile;
        if (c < g.cols) {
            float v = s[0];
            if constexpr (W == 2)
                with_act(g.act, [&](auto kind) {
                    v = act_slope<decltype(kind)::value>(s[0]).x * s[1];
                });
            g.out[r * g.ldo + c] = v;
        }
    }
    cluster_sync();  // no CTA leaves while another reads its sums
}

// MT rows (a power of two >= rows), VEC columns a lane, W = 2: gate and up.
template <int MT, int VEC, int W>
__global__ void __launch_bounds__(256) rows_n_kernel(RowsArgs g) {
    constexpr int kTile = 32 * VEC;
    constexpr int kAhead = MT * VEC * W >= 64 ? 4 : 8;   // weight rows in flight per warp
    constexpr int kXTile = kRowsXBytes / 4 / MT;         // depth staged at a time
    extern __shared__ __align__(16) float rows_smem[];
    float* xs = rows_smem;                               // [depth][MT]
    float* red = rows_smem + kRowsXBytes / 4;
    if (!g.wait) grid_dependents_go();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ranks = static_cast<int>(cluster_nctarank());
    const int rank = static_cast<int>(cluster_ctarank());
    const int col0 = (static_cast<int>(blockIdx.x) / ranks) * kTile;
    const int col = col0 + lane * VEC;
    const bool in = col < g.cols;   // VEC > 1 only where it divides cols
    const int k_begin = static_cast<int>(static_cast<long long>(g.depth) * rank / ranks);
    const int k_end = static_cast<int>(static_cast<long long>(g.depth) * (rank + 1) / ranks);
    const float* p0 = g.w0 + (in ? col : 0);
    const float* p1 = W == 2 ? g.w1 + (in ? col : 0) : nullptr;

    float acc[W][MT][VEC];
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
        for (int r = 0; r < MT; ++r)
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[i][r][e] = 0.0f;

    bool waited = g.wait == 0;
    for (int k0 = k_begin; k0 < k_end; k0 += kXTile) {
        const int depth = min(kXTile, k_end - k0);
        RowsVec<VEC> a[kAhead], b[kAhead];
        auto load = [&](int k) {
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const long long row = k0 + min(k + j, depth - 1);
                a[j] = rows_load<VEC>(p0 + row * g.ld0);
                if constexpr (W == 2) b[j] = rows_load<VEC>(p1 + row * g.ld1);
            }
        };
        const int first = warp * kAhead;
        if (first < depth) load(first);          // on the way while x is staged
        if (!waited) {
            grid_wait();
            waited = true;
        }
        if (k0 > k_begin) __syncthreads();
        for (int i = threadIdx.x; i < depth * MT; i += 256) {
            const int r = i / depth, k = i - r * depth;
            xs[k * MT + r] = r < g.rows ? g.x[r * g.x_rs + (k0 + k) * g.x_cs] : 0.0f;
        }
        __syncthreads();
        for (int k = first; k < depth; k += 8 * kAhead) {
            if (k != first) load(k);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (k + j < depth) {
                    const float* xr = xs + (k + j) * MT;
#pragma unroll
                    for (int r = 0; r < MT; ++r) {
                        const float xv = xr[r];
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            acc[0][r][e] = fmaf(xv, a[j].v[e], acc[0][r][e]);
                            if constexpr (W == 2) acc[1][r][e] = fmaf(xv, b[j].v[e], acc[1][r][e]);
                        }
                    }
                }
            }
        }
    }
    if (!waited) grid_wait();  // a CTA without depth still leaves after the launch before

    // the eight warps' sums by halves: fixed order
    constexpr int kVals = W * MT * VEC;
    __syncthreads();
#pragma unroll
    for (int half = 4; half > 0; half >>= 1) {
        if (warp >= half && warp < 2 * half) {
#pragma unroll
            for (int v = 0; v < kVals; ++v)
                red[((warp - half) * kVals + v) * 32 + lane] = (&acc[0][0][0])[v];
        }
        __syncthreads();
        if (warp < half) {
#pragma unroll
            for (int v = 0; v < kVals; ++v)
                (&acc[0][0][0])[v] += red[(warp * kVals + v) * 32 + lane];
        }
        __syncthreads();
    }
    if (warp == 0) {
#pragma unroll
        for (int r = 0; r < MT; ++r)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
#pragma unroll
                for (int i = 0; i < W; ++i)
                    red[(r * kTile + lane * VEC + e) * W + i] = acc[i][r][e];
    }
    rows_finish<W>(g, red, kTile, col0);
}

// Depth contiguous: a warp has two outputs (of each matrix), its lanes VEC values of the depth.
template <int MT, int VEC, int W>
__global__ void __launch_bounds__(256) rows_k_kernel(RowsArgs g) {
    constexpr int kTile = 16;                            // outputs per CTA
    constexpr int kXTile = kRowsXBytes / 4 / MT;
    constexpr int kStep = 32 * VEC;
    extern __shared__ __align__(16) float rows_smem[];
    float* xs = rows_smem;                               // [MT][kXTile]
    float* red = rows_smem + kRowsXBytes / 4;
    if (!g.wait) grid_dependents_go();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ranks = static_cast<int>(cluster_nctarank());
    const int rank = static_cast<int>(cluster_ctarank());
    const int col0 = (static_cast<int>(blockIdx.x) / ranks) * kTile;
    // shares of the depth in whole multiples of VEC, so that loads stay aligned
    const long long units = (g.depth + VEC - 1) / VEC;
    const int k_begin = static_cast<int>(units * rank / ranks) * VEC;
    const int k_end = min(g.depth, static_cast<int>(units * (rank + 1) / ranks) * VEC);
    const float* p[W][2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const long long c = min(col0 + warp * 2 + n, g.cols - 1);
        p[0][n] = g.w0 + c * g.ld0;
        if constexpr (W == 2) p[1][n] = g.w1 + c * g.ld1;
    }
    float acc[W][2][MT];
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int r = 0; r < MT; ++r) acc[i][n][r] = 0.0f;

    bool waited = g.wait == 0;
    for (int k0 = k_begin; k0 < k_end; k0 += kXTile) {
        const int depth = min(kXTile, k_end - k0);   // VEC > 1 only where it divides the depth
        constexpr int kAhead = 2;
        RowsVec<VEC> w[kAhead][W][2];
        auto load = [&](int k) {
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int at = k + j * kStep < depth ? k0 + k + j * kStep : k0;
#pragma unroll
                for (int i = 0; i < W; ++i)
#pragma unroll
                    for (int n = 0; n < 2; ++n) w[j][i][n] = rows_load<VEC>(p[i][n] + at);
            }
        };
        load(lane * VEC);
        if (!waited) {
            grid_wait();
            waited = true;
        }
        if (k0 > k_begin) __syncthreads();
        for (int i = threadIdx.x; i < depth * MT; i += 256) {
            const int r = i / depth, k = i - r * depth;
            xs[r * kXTile + k] = r < g.rows ? g.x[r * g.x_rs + (k0 + k) * g.x_cs] : 0.0f;
        }
        __syncthreads();
        for (int k = lane * VEC; k < depth; k += kAhead * kStep) {
            if (k != lane * VEC) load(k);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int at = k + j * kStep;
                if (at < depth) {
#pragma unroll
                    for (int r = 0; r < MT; ++r) {
                        float xv[VEC];
                        const float* xp = xs + r * kXTile + at;
                        if constexpr (VEC == 4) {
                            const float4 q = *reinterpret_cast<const float4*>(xp);
                            xv[0] = q.x, xv[1] = q.y, xv[2] = q.z, xv[3] = q.w;
                        } else {
                            xv[0] = *xp;
                        }
#pragma unroll
                        for (int i = 0; i < W; ++i)
#pragma unroll
                            for (int n = 0; n < 2; ++n)
#pragma unroll
                                for (int e = 0; e < VEC; ++e)
                                    acc[i][n][r] = fmaf(xv[e], w[j][i][n].v[e], acc[i][n][r]);
                    }
                }
            }
        }
    }
    if (!waited) grid_wait();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int r = 0; r < MT; ++r) {
                float s = acc[i][n][r];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                if (lane == 0) red[(r * kTile + warp * 2 + n) * W + i] = s;
            }
    rows_finish<W>(g, red, kTile, col0);
}

}  // namespace mfk
