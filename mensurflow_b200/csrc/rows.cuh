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
constexpr int kRowsXBytes = 40960;      // of x staged at a time
constexpr int kRowsRingBytes = 65536;   // weights on their way: 8 KB per warp; later the sums
constexpr int kRowsSmem = kRowsXBytes + kRowsRingBytes;

struct RowsArgs {
    const float* x;          // element (r, k) at x[r*x_rs + k]
    long long x_rs;
    const float* w0;         // the weights (gate), row stride ld0
    const float* w1;         // up
    long long ld0, ld1;
    int rows, depth, cols;   // of the product
    float* out;              // rows x cols, row stride ldo
    long long ldo;
    int act;
    int wait;                // x comes from the launch before
};

// 4, 8 or 16 bytes, global -> shared, in the thread's own copy groups.
template <int BYTES>
__device__ __forceinline__ void rows_copy(float* dst, const float* src) {
    if constexpr (BYTES == 16) {
        cp_async_16(smem_u32(dst), src);
    } else {
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src),
                     "n"(BYTES)
                     : "memory");
    }
}

template <int VEC>
__device__ __forceinline__ void rows_read(const float* p, float (&v)[VEC]) {
    if constexpr (VEC == 4) {
        const float4 q = *reinterpret_cast<const float4*>(p);
        v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
    } else if constexpr (VEC == 2) {
        const float2 q = *reinterpret_cast<const float2*>(p);
        v[0] = q.x, v[1] = q.y;
    } else {
        v[0] = *p;
    }
}

// x of rows [0, MT) and depth [k0, k0 + depth) into shared memory at xs[r * rs + k * ks].
// DUP: each value twice in a row.
template <int MT, int DUP>
__device__ __forceinline__ void rows_stage_x(const RowsArgs& g, float* xs, int k0, int depth,
                                             int rs, int ks) {
#pragma unroll 4
    for (int i = threadIdx.x; i < depth * MT; i += 256) {
        const int r = i % MT, k = i / MT;
        const float v = r < g.rows ? g.x[r * g.x_rs + (k0 + k)] : 0.0f;
        if constexpr (DUP == 2) {
            *reinterpret_cast<float2*>(xs + r * rs + k * ks) = make_float2(v, v);
        } else {
            xs[r * rs + k * ks] = v;
        }
    }
}

// a0 += r0 f0, a1 += r1 f1 with (f0, f1) already a register pair.
__device__ __forceinline__ void fma2_pair(float& a0, float& a1, float r0, float r1,
                                          unsigned long long f) {
    asm("{\n\t.reg .b64 a, r;\n\t"
        "mov.b64 a, {%0, %1};\n\t"
        "mov.b64 r, {%2, %3};\n\t"
        "fma.rn.f32x2 a, r, %4, a;\n\t"
        "mov.b64 {%0, %1}, a;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "f"(r0), "f"(r1), "l"(f));
}

constexpr int kRowsRanks = 8;   // largest cluster

// The cluster's sums of `tile` columns (res[(r * tile + c) * W + i], W = 2 with gate and up) in
// rank order, the activation, and the store.
template <int W, int TILE>
__device__ __forceinline__ void rows_finish(const RowsArgs& g, float* res, int col0) {
    const uint32_t ranks = cluster_nctarank(), rank = cluster_ctarank();
    __syncthreads();
    cluster_sync();
    for (int i = static_cast<int>(rank) * 256 + threadIdx.x; i < g.rows * TILE;
         i += static_cast<int>(ranks) * 256) {
        float v[kRowsRanks][W];
#pragma unroll
        for (uint32_t q = 0; q < kRowsRanks; ++q) {
            const uint32_t at = mapa_shared(res + i * W, q < ranks ? q : rank);
#pragma unroll
            for (int e = 0; e < W; ++e) v[q][e] = ld_cluster_f32(at + e * 4);
        }
        float s[W];
#pragma unroll
        for (int e = 0; e < W; ++e) s[e] = v[0][e];
#pragma unroll
        for (uint32_t q = 1; q < kRowsRanks; ++q)
#pragma unroll
            for (int e = 0; e < W; ++e) s[e] += q < ranks ? v[q][e] : 0.0f;
        const int r = i / TILE, c = col0 + i % TILE;
        if (c < g.cols) {
            float y = s[0];
            if constexpr (W == 2)
                with_act(g.act, [&](auto kind) {
                    y = act_slope<decltype(kind)::value>(s[0]).x * s[1];
                });
            g.out[r * g.ldo + c] = y;
        }
    }
    cluster_sync();  // no CTA leaves while another reads its sums
}

// MT rows (a power of two >= rows), VEC columns a lane, W = 2: gate and up. Every warp keeps a
// ring of eight stages of 1 KB in flight through asynchronous copies that each lane makes and
// reads itself (no barrier in the loop); a stage is R rows of the weights. x lies in shared memory
// with each value twice, ready for the packed FMA (a copy per value otherwise).
template <int MT, int VEC, int W>
__global__ void __launch_bounds__(256, 2) rows_n_kernel(RowsArgs g) {
    constexpr int kTile = 32 * VEC;
    constexpr int kR = 8 / (VEC * W);
    constexpr int kStages = 8;
    constexpr int kDup = VEC == 1 ? 1 : 2;
    constexpr int kTurn = 8 * kR;                        // depth of a turn of the eight warps
    constexpr int kXTurns = kRowsXBytes / 4 / kDup / MT / kTurn / kStages * kStages;
    static_assert(kXTurns > 0, "the ring turns within the staged x");
    extern __shared__ __align__(16) float rows_smem[];
    float* xs = rows_smem;                               // [depth][MT][kDup]
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
    const int depth = k_end - k_begin;
    const int turns = (depth + kTurn - 1) / kTurn;
    const float* p0 = g.w0 + (in ? col : 0);
    const float* p1 = W == 2 ? g.w1 + (in ? col : 0) : nullptr;
    float* ring = red + warp * 2048 + lane * VEC;        // [stage][row][matrix][lane][VEC]

    float acc[W][MT][VEC];
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
        for (int r = 0; r < MT; ++r)
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[i][r][e] = 0.0f;

    // the next turn's rows: running pointers, this warp's first row of the turn
    const float* q0 = p0 + static_cast<long long>(k_begin + warp * kR) * g.ld0;
    const float* q1 = W == 2 ? p1 + static_cast<long long>(k_begin + warp * kR) * g.ld1 : nullptr;
    const long long step0 = g.ld0 * kTurn, step1 = W == 2 ? g.ld1 * kTurn : 0;
    int next = warp * kR;
    auto issue = [&](int stage) {
#pragma unroll
        for (int j = 0; j < kR; ++j) {
            if (next + j < depth) {
                float* dst = ring + stage * 256 + j * W * kTile;
                rows_copy<VEC * 4>(dst, q0 + j * g.ld0);
                if constexpr (W == 2) rows_copy<VEC * 4>(dst + kTile, q1 + j * g.ld1);
            }
        }
        q0 += step0;
        if constexpr (W == 2) q1 += step1;
        next += kTurn;
        cp_async_commit();
    };
    for (int t = 0; t < kStages; ++t) issue(t);   // on the way while x is staged
    if (g.wait) grid_wait();
    for (int t0 = 0; t0 < turns; t0 += kXTurns) {
        const int x0 = t0 * kTurn;
        if (t0 > 0) __syncthreads();
        rows_stage_x<MT, kDup>(g, xs, k_begin + x0, min(kXTurns * kTurn, depth - x0), kDup,
                               MT * kDup);
        __syncthreads();
        const int t1 = min(turns, t0 + kXTurns);
        const float* xr = xs + warp * kR * (MT * kDup);
        int left = depth - x0 - warp * kR;               // rows of the depth from this warp's first
        for (int t = t0; t < t1; t += kStages) {
#pragma unroll
            for (int u = 0; u < kStages; ++u) {
                if (t + u < t1) {
                    cp_async_wait<kStages - 1>();
#pragma unroll
                    for (int j = 0; j < kR; ++j) {
                        if (j < left) {
                            float w[W][VEC];
                            const float* src = ring + u * 256 + j * W * kTile;
#pragma unroll
                            for (int i = 0; i < W; ++i) rows_read<VEC>(src + i * kTile, w[i]);
                            const float* xj = xr + j * (MT * kDup);
                            if constexpr (VEC == 1) {
#pragma unroll
                                for (int r = 0; r < MT; ++r)
#pragma unroll
                                    for (int i = 0; i < W; ++i)
                                        acc[i][r][0] = fmaf(xj[r], w[i][0], acc[i][r][0]);
                            } else {
#pragma unroll
                                for (int r = 0; r < MT; ++r) {
                                    const unsigned long long xv =
                                        reinterpret_cast<const unsigned long long*>(xj)[r];
#pragma unroll
                                    for (int i = 0; i < W; ++i)
#pragma unroll
                                        for (int e = 0; e < VEC; e += 2)
                                            fma2_pair(acc[i][r][e], acc[i][r][e + 1], w[i][e],
                                                      w[i][e + 1], xv);
                                }
                            }
                        }
                    }
                    issue(u);
                    xr += kTurn * MT * kDup;
                    left -= kTurn;
                }
            }
        }
    }
    cp_async_wait<0>();

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
    rows_finish<W, kTile>(g, red, col0);
}

// Depth contiguous: a warp has two outputs (of each matrix), its lanes the depth, 4 / VEC values
// of VEC each a stage and row; a ring as above.
template <int MT, int VEC, int W>
__global__ void __launch_bounds__(256, 2) rows_k_kernel(RowsArgs g) {
    constexpr int kTile = 16;                            // outputs per CTA
    constexpr int kXTile = kRowsXBytes / 4 / MT / 128 * 128;
    constexpr int kJ = 4 / VEC;
    constexpr int kStages = 8 / W;                       // of 128 values of 2 W rows
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
    float* ring = red + warp * 2048 + lane * VEC;        // [stage][matrix][output][kJ][lane][VEC]
    float acc[W][2][MT];
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int r = 0; r < MT; ++r) acc[i][n][r] = 0.0f;

    const int depth = k_end - k_begin;               // VEC > 1 only where it divides the depth
    const int turns = (depth + 127) / 128;
    auto issue = [&](int turn) {
        if (turn < turns) {
            float* dst = ring + (turn % kStages) * (256 * W);
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
                const int k = turn * 128 + (j * 32 + lane) * VEC;
                const int at = k_begin + (k < depth ? k : 0);   // past the end: not used
#pragma unroll
                for (int i = 0; i < W; ++i)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
                        rows_copy<VEC * 4>(dst + (i * 2 + n) * 128 + j * 32 * VEC, p[i][n] + at);
            }
        }
        cp_async_commit();
    };
    for (int t = 0; t < kStages; ++t) issue(t);
    if (g.wait) grid_wait();
    constexpr int kXTurns = kXTile / 128;
    for (int t0 = 0; t0 < turns; t0 += kXTurns) {
        const int x0 = t0 * 128;
        if (t0 > 0) __syncthreads();
        rows_stage_x<MT, 1>(g, xs, k_begin + x0, min(kXTile, depth - x0), kXTile, 1);
        __syncthreads();
        const int t1 = min(turns, t0 + kXTurns);
        for (int t = t0; t < t1; ++t) {
            cp_async_wait<kStages - 1>();
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
                const int k = t * 128 + (j * 32 + lane) * VEC;
                if (k < depth) {
                    float w[W][2][VEC];
                    const float* src = ring + (t % kStages) * (256 * W) + j * 32 * VEC;
#pragma unroll
                    for (int i = 0; i < W; ++i)
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            rows_read<VEC>(src + (i * 2 + n) * 128, w[i][n]);
#pragma unroll
                    for (int r = 0; r < MT; ++r) {
                        float xv[VEC];
                        rows_read<VEC>(xs + r * kXTile + k - x0, xv);
#pragma unroll
                        for (int i = 0; i < W; ++i)
#pragma unroll
                            for (int n = 0; n < 2; ++n)
#pragma unroll
                                for (int e = 0; e < VEC; ++e)
                                    acc[i][n][r] = fmaf(xv[e], w[i][n][e], acc[i][n][r]);
                    }
                }
            }
            issue(t + kStages);
        }
    }
    cp_async_wait<0>();
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
    rows_finish<W, kTile>(g, red, col0);
}

}  // namespace mfk
