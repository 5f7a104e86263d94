// The embedding lookup and its table's gradient, fp32.
//
// out[i] = scale * table[ids[i]]: one pass, bound by HBM (each token's row read and written).
//
// d_table[v] = scale * sum over i with ids[i] == v of grad[i], for every row v of a dense table.
// The sums are taken in the tokens' order whatever the launch does, so the same inputs give the
// same bits: the tokens are sorted by id with a stable radix sort (id and position, 8 bits a
// pass), the sorted list is cut into windows, and one block adds a window's rows in order; runs
// of one id that cross windows leave partial rows, which a last kernel adds window by window.
// Rows that no token names are filled with zeros, each written once. Bound by HBM: grad read
// once, the table written once.
#pragma once

#include "split_mm.cuh"

namespace mfk {

// Set when a kernel met an id outside the table; reported by mfk_device_status. Kept apart from
// g_device_error, which ends the waits of kernels in flight.
__device__ unsigned int g_index_error = 0u;

constexpr int kEmbedPiece = 1024;      // columns a block of 256 threads takes, four a thread
constexpr int kSortTile = 2048;        // items per block of the radix passes
constexpr int kSortItems = 8;          // per thread

template <typename ID>
__global__ void __launch_bounds__(256)
    embedding_kernel(const float* __restrict__ table, long long rows, int d, long long ld,
                     const ID* __restrict__ ids, long long n, float scale, float* __restrict__ out,
                     long long ld_out, int vec) {
    // one warp per token and piece of 512 columns, 16 values in flight per lane
    const int lane = threadIdx.x & 31;
    const int pieces = (d + 511) / 512;
    const long long total = n * pieces;
    for (long long w = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 5; w < total;
         w += static_cast<long long>(gridDim.x) * 8) {
        const long long i = w / pieces;
        const int c0 = static_cast<int>(w - i * pieces) * 512;
        const long long id = static_cast<long long>(ids[i]);
        const bool ok = id >= 0 && id < rows;
        if (!ok && lane == 0) atomicOr(&g_index_error, 1u);
        const float* src = table + (ok ? id : 0) * ld + c0;
        float* dst = out + i * ld_out + c0;
        const int width = min(512, d - c0);
        const float f = ok ? scale : 0.0f;
        if (vec) {
            float4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = (j * 32 + lane) * 4;
                if (c < width) v[j] = ok ? __ldg(reinterpret_cast<const float4*>(src + c))
                                         : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = (j * 32 + lane) * 4;
                if (c < width)
                    *reinterpret_cast<float4*>(dst + c) =
                        make_float4(v[j].x * f, v[j].y * f, v[j].z * f, v[j].w * f);
            }
        } else {
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int c = j * 32 + lane;
                if (c < width) v[j] = ok ? __ldg(src + c) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int c = j * 32 + lane;
                if (c < width) dst[c] = v[j] * f;
            }
        }
    }
}

// The same for rows of up to 128 columns, VEC of them a load: as many lanes as the row needs (a
// power of two), four tokens in flight a lane. A warp per token leaves lanes idle and has one chain
// of id and row on its way: 65536 tokens of 65536 x 32 take 29.8 us so and 5 us here.
template <typename ID, int VEC>
__global__ void __launch_bounds__(256)
    embedding_narrow_kernel(const float* __restrict__ table, long long rows, int d, long long ld,
                            const ID* __restrict__ ids, long long n, float scale,
                            float* __restrict__ out, long long ld_out, int lanes) {
    constexpr int kTokens = 4, kLoads = VEC == 4 ? 1 : 4;
    const int lane = threadIdx.x & 31;
    const int per = 32 / lanes;              // tokens of a warp at once
    const int c = (lane % lanes) * VEC;
    const long long first = ((static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 5) *
                                (kTokens * per) + lane / lanes;
    const float* src[kTokens];
    bool ok[kTokens];
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
        const long long i = first + t * per;
        const long long id = i < n ? static_cast<long long>(ids[i]) : 0;
        ok[t] = i < n && id >= 0 && id < rows;
        if (i < n && !ok[t] && c == 0) atomicOr(&g_index_error, 1u);
        src[t] = table + (ok[t] ? id : 0) * ld + c;
    }
    float v[kTokens][kLoads][VEC];
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            if constexpr (VEC == 4) {
                const float4 q = ok[t] && c < d ? __ldg(reinterpret_cast<const float4*>(src[t]))
                                                : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                v[t][k][0] = q.x, v[t][k][1] = q.y, v[t][k][2] = q.z, v[t][k][3] = q.w;
            } else {
                v[t][k][0] = ok[t] && c + k * 32 < d ? __ldg(src[t] + k * 32) : 0.0f;
            }
        }
    }
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
        const long long i = first + t * per;
        if (i >= n) continue;
        const float f = ok[t] ? scale : 0.0f;
        float* dst = out + i * ld_out + c;
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            if constexpr (VEC == 4) {
                if (c < d)
                    *reinterpret_cast<float4*>(dst) = make_float4(
                        v[t][k][0] * f, v[t][k][1] * f, v[t][k][2] * f, v[t][k][3] * f);
            } else {
                if (c + k * 32 < d) dst[k * 32] = v[t][k][0] * f;
            }
        }
    }
}

// ---- the sort --------------------------------------------------------------------------------

// Keys of the first pass: the id, or `rows` for a token that takes no part (padding, or outside
// the table). Marks the ids that are present and counts the first digit per tile.
template <typename ID>
__global__ void __launch_bounds__(256)
    embed_keys_kernel(const ID* __restrict__ ids, long long n, long long rows, long long padding,
                      uint32_t* __restrict__ keys, uint32_t* __restrict__ present,
                      uint32_t* __restrict__ counts, int tiles) {
    __shared__ uint32_t bins[256];
    bins[threadIdx.x] = 0u;
    __syncthreads();
    const long long base = static_cast<long long>(blockIdx.x) * kSortTile;
    for (int r = 0; r < kSortItems; ++r) {
        const long long i = base + r * 256 + threadIdx.x;
        if (i >= n) break;
        const long long id = static_cast<long long>(ids[i]);
        const bool inside = id >= 0 && id < rows;
        if (!inside && (padding < 0 || id != padding)) atomicOr(&g_index_error, 1u);
        const uint32_t key = static_cast<uint32_t>(inside && id != padding ? id : rows);
        keys[i] = key;
        if (key < rows) {
            uint32_t* word = present + (key >> 5);
            const uint32_t bit = 1u << (key & 31u);
            if ((*reinterpret_cast<volatile uint32_t*>(word) & bit) == 0u) atomicOr(word, bit);
        }
        atomicAdd(&bins[key & 255u], 1u);
    }
    __syncthreads();
    counts[static_cast<long long>(threadIdx.x) * tiles + blockIdx.x] = bins[threadIdx.x];
}

__global__ void __launch_bounds__(256)
    sort_count_kernel(const uint32_t* __restrict__ keys, long long n, int shift,
                      uint32_t* __restrict__ counts, int tiles) {
    __shared__ uint32_t bins[256];
    bins[threadIdx.x] = 0u;
    __syncthreads();
    const long long base = static_cast<long long>(blockIdx.x) * kSortTile;
    for (int r = 0; r < kSortItems; ++r) {
        const long long i = base + r * 256 + threadIdx.x;
        if (i < n) atomicAdd(&bins[(keys[i] >> shift) & 255u], 1u);
    }
    __syncthreads();
    counts[static_cast<long long>(threadIdx.x) * tiles + blockIdx.x] = bins[threadIdx.x];
}

// Exclusive sums of `n` counts in place, one block.
__global__ void __launch_bounds__(1024) sort_scan_kernel(uint32_t* __restrict__ counts,
                                                         long long n) {
    __shared__ uint32_t sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t carry = 0;
    for (long long base = 0; base < n; base += 4096) {
        const long long i = base + threadIdx.x * 4;
        uint32_t v[4], t = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = i + j < n ? counts[i + j] : 0u;
            t += v[j];
        }
        uint32_t s = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += up;
        }
        if (lane == 31) sums[warp] = s;
        __syncthreads();
        uint32_t before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < 32; ++w) {
            const uint32_t x = sums[w];
            before += w < warp ? x : 0u;
            all += x;
        }
        uint32_t at = carry + before + s - t;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i + j < n) counts[i + j] = at;
            at += v[j];
        }
        carry += all;
        __syncthreads();
    }
}

// One stable pass: a warp takes 256 consecutive items in rounds of 32, ranks equal digits by
// lane within a round and by the rounds before it; warps and tiles follow in order.
__global__ void __launch_bounds__(256)
    sort_scatter_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                        long long n, int shift, const uint32_t* __restrict__ offsets, int tiles,
                        uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out) {
    __shared__ uint32_t counts[8][257];
    grid_dependents_go();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < 8 * 257; i += 256) (&counts[0][0])[i] = 0u;
    __syncthreads();
    const long long base = static_cast<long long>(blockIdx.x) * kSortTile + warp * 256;
    uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        const long long i = base + r * 32 + lane;
        key[r] = i < n ? keys[i] : 0u;
        const uint32_t digit = i < n ? (key[r] >> shift) & 255u : 256u;
        const uint32_t same = __match_any_sync(0xffffffffu, digit);
        const uint32_t before = counts[warp][digit];
        rank[r] = before + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if ((same >> lane) == 1u) counts[warp][digit] = before + __popc(same);  // the last one
        __syncwarp();
    }
    __syncthreads();
    {   // counts -> first output index of (warp, digit)
        uint32_t at = offsets[static_cast<long long>(threadIdx.x) * tiles + blockIdx.x];
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            const uint32_t c = counts[w][threadIdx.x];
            counts[w][threadIdx.x] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortItems; ++r) {
        const long long i = base + r * 32 + lane;
        if (i < n) {
            const uint32_t to = counts[warp][(key[r] >> shift) & 255u] + rank[r];
            keys_out[to] = key[r];
            pos_out[to] = pos != nullptr ? pos[i] : static_cast<uint32_t>(i);
        }
    }
}

// ---- the sort in one launch ------------------------------------------------------------------

constexpr int kClusterSortRanks = 8;
constexpr int kClusterSortMax = kClusterSortRanks * 8192;   // tokens

__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// Up to 65536 tokens in one cluster of up to 8 CTAs: each holds `chunk` of the list in shared
// memory and a pass scatters straight into the others'. Ranks within a warp's items as in
// sort_scatter_kernel, then over the CTA's warps, then over the CTAs. Also clears the marks and
// sets those of the ids that are present. IT: rounds of 32 items per warp.
template <typename ID, int IT>
__global__ void __launch_bounds__(1024, 1)
    embed_sort_kernel(const ID* __restrict__ ids, int n, int chunk, long long rows,
                      long long padding, int passes, uint32_t* __restrict__ present,
                      uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out) {
    extern __shared__ __align__(16) uint32_t sort_smem[];
    uint32_t* buffers = sort_smem;                         // keys, positions; twice
    uint32_t* counts = sort_smem + 4 * chunk;              // [32 warps][256]
    uint32_t* total = counts + 32 * 256;                   // [256] this CTA's
    uint32_t* base = total + 256;                          // [256]
    uint32_t* scan = base + 256;                           // [8]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ranks = static_cast<int>(gridDim.x);         // one cluster
    const int rank = static_cast<int>(cluster_ctarank());
    const int first = rank * chunk;
    const int count = max(0, min(chunk, n - first));

    grid_dependents_go();
    const long long words = (rows + 31) / 32;
    for (long long i = rank * 1024 + static_cast<int>(threadIdx.x); i < words; i += ranks * 1024)
        present[i] = 0u;
    __threadfence();
    cluster_sync();

    const int mine = warp * IT * 32 + lane;                // first item of this lane
    uint32_t key[IT], pos[IT];
#pragma unroll
    for (int r = 0; r < IT; ++r) {
        const int i = mine + r * 32;
        key[r] = 0u;
        pos[r] = static_cast<uint32_t>(first + i);
        if (i < count) {
            const long long id = static_cast<long long>(ids[first + i]);
            const bool inside = id >= 0 && id < rows;
            if (!inside && (padding < 0 || id != padding)) atomicOr(&g_index_error, 1u);
            key[r] = static_cast<uint32_t>(inside && id != padding ? id : rows);
            if (key[r] < rows) {
                uint32_t* word = present + (key[r] >> 5);
                const uint32_t bit = 1u << (key[r] & 31u);
                if ((*reinterpret_cast<volatile uint32_t*>(word) & bit) == 0u) atomicOr(word, bit);
            }
        }
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * 8;
        uint32_t* out = buffers + (pass & 1) * 2 * chunk;
        if (pass > 0) {
            const uint32_t* in = buffers + ((pass - 1) & 1) * 2 * chunk;
#pragma unroll
            for (int r = 0; r < IT; ++r) {
                const int i = mine + r * 32;
                if (i < count) {
                    key[r] = in[i];
                    pos[r] = in[chunk + i];
                }
            }
        }
        for (int i = threadIdx.x; i < 32 * 256; i += 1024) counts[i] = 0u;
        __syncthreads();
        uint32_t at[IT];
#pragma unroll
        for (int r = 0; r < IT; ++r) {
            const bool in = mine + r * 32 < count;
            const uint32_t digit = in ? (key[r] >> shift) & 255u : 256u;
            const uint32_t same = __match_any_sync(0xffffffffu, digit);
            const uint32_t before = in ? counts[warp * 256 + digit] : 0u;
            at[r] = before + __popc(same & ((1u << lane) - 1u));
            __syncwarp();
            if (in && (same >> lane) == 1u) counts[warp * 256 + digit] = before + __popc(same);
            __syncwarp();
        }
        __syncthreads();
        if (threadIdx.x < 256) {                           // over this CTA's warps
            uint32_t sum = 0;
#pragma unroll 8
            for (int w = 0; w < 32; ++w) {
                const uint32_t c = counts[w * 256 + threadIdx.x];
                counts[w * 256 + threadIdx.x] = sum;
                sum += c;
            }
            total[threadIdx.x] = sum;
        }
        __syncthreads();
        cluster_sync();
        if (threadIdx.x < 256) {                           // over the CTAs, then over the digits
            uint32_t before = 0, all = 0;
            for (int q = 0; q < ranks; ++q) {
                const uint32_t c = ld_cluster_u32(mapa_shared(total + threadIdx.x, q));
                before += q < rank ? c : 0u;
                all += c;
            }
            uint32_t s = all;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += up;
            }
            if (lane == 31) scan[warp] = s;
            base[threadIdx.x] = s - all + before;
        }
        __syncthreads();
        if (threadIdx.x < 256) {
            uint32_t lower = 0;
            for (int w = 0; w < warp; ++w) lower += scan[w];
            base[threadIdx.x] += lower;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < IT; ++r) {
            if (mine + r * 32 < count) {
                const uint32_t digit = (key[r] >> shift) & 255u;
                const uint32_t to = base[digit] + counts[warp * 256 + digit] + at[r];
                if (pass + 1 == passes) {
                    keys_out[to] = key[r];
                    pos_out[to] = pos[r];
                } else {
                    const uint32_t q = to / static_cast<uint32_t>(chunk);
                    const uint32_t local = mapa_shared(out + (to - q * chunk), q);
                    st_cluster_u32(local, key[r]);
                    st_cluster_u32(local + 4u * chunk, pos[r]);
                }
            }
        }
        cluster_sync();  // the list is complete, and nobody leaves or reuses what others read
    }
}

// ---- the sums --------------------------------------------------------------------------------

// A thread's four columns of a piece: neighbours where every row can be read 16 bytes at a time
// (`vec`), else 256 apart, so that a warp still covers whole lines.
__device__ __forceinline__ float4 embed_load(const float* p, int c0, int d, int vec) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (vec) {
        const int c = c0 + static_cast<int>(threadIdx.x) * 4;
        if (c < d) v = __ldg(reinterpret_cast<const float4*>(p + c));
    } else {
        const int c = c0 + static_cast<int>(threadIdx.x);
        if (c < d) v.x = __ldg(p + c);
        if (c + 256 < d) v.y = __ldg(p + c + 256);
        if (c + 512 < d) v.z = __ldg(p + c + 512);
        if (c + 768 < d) v.w = __ldg(p + c + 768);
    }
    return v;
}

__device__ __forceinline__ void embed_store(float* p, int c0, int d, int vec, float4 v) {
    if (vec) {
        const int c = c0 + static_cast<int>(threadIdx.x) * 4;
        if (c < d) *reinterpret_cast<float4*>(p + c) = v;
    } else {
        const int c = c0 + static_cast<int>(threadIdx.x);
        if (c < d) p[c] = v.x;
        if (c + 256 < d) p[c + 256] = v.y;
        if (c + 512 < d) p[c + 512] = v.z;
        if (c + 768 < d) p[c + 768] = v.w;
    }
}

constexpr int kEmbedMaxWindow = 256;

// The first `sum_blocks` blocks: one per window of `window` sorted tokens and piece of 1024
// columns. A run of one id that lies inside the window is written out; the part of a run that came
// in from the window before goes to part[2 w], the part of one that only goes on into the next to
// part[2 w + 1]. The blocks behind them write zeros into the rows that no token names, a warp per
// row: they fill the memory system while the sums wait for their rows.
__global__ void __launch_bounds__(256)
    embed_sum_kernel(const uint32_t* keys, const uint32_t* pos,
                     long long n, int window, uint32_t rows, const float* __restrict__ grad,
                     long long ld_grad, int d, float scale, float* __restrict__ out, long long ld,
                     float* part, int vec, int pieces, int sum_blocks,
                     const uint32_t* present) {
    grid_dependents_go();
    grid_wait();
    if (static_cast<int>(blockIdx.x) >= sum_blocks) {
        const int lane = threadIdx.x & 31;
        const int warps = (static_cast<int>(gridDim.x) - sum_blocks) * 8;
        const int mine = (static_cast<int>(blockIdx.x) - sum_blocks) * 8 +
                         static_cast<int>(threadIdx.x >> 5);
        for (long long v = mine; v < rows; v += warps) {
            if ((present[v >> 5] >> (v & 31)) & 1u) continue;
            float* p = out + v * ld;
            if (vec) {
                for (int c = lane * 4; c < d; c += 128)
                    *reinterpret_cast<float4*>(p + c) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            } else {
                for (int c = lane; c < d; c += 32) p[c] = 0.0f;
            }
        }
        return;
    }
    __shared__ uint32_t s_key[kEmbedMaxWindow + 1], s_pos[kEmbedMaxWindow];
    const long long w = static_cast<int>(blockIdx.x) / pieces;
    const int c0 = (static_cast<int>(blockIdx.x) - static_cast<int>(w) * pieces) * kEmbedPiece;
    const long long first = w * window;
    const int count = static_cast<int>(min(static_cast<long long>(window), n - first));
    for (int i = threadIdx.x; i < count; i += 256) {
        s_key[i] = keys[first + i];
        s_pos[i] = pos[first + i];
    }
    if (threadIdx.x == 0) s_key[count] = first + count < n ? keys[first + count] : 0xffffffffu;
    __syncthreads();
    const uint32_t previous = first > 0 ? keys[first - 1] : 0xffffffffu;
    bool from_before = s_key[0] == previous;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int kAhead = 8;
    for (int i0 = 0; i0 < count; i0 += kAhead) {
        float4 g[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            g[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i0 + j < count && s_key[i0 + j] < rows)
                g[j] = embed_load(grad + static_cast<long long>(s_pos[i0 + j]) * ld_grad, c0, d,
                                  vec);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = i0 + j;
            if (i < count && s_key[i] < rows) {
                acc.x += g[j].x;
                acc.y += g[j].y;
                acc.z += g[j].z;
                acc.w += g[j].w;
                const bool ends = s_key[i + 1] != s_key[i];
                if (ends || i + 1 == count) {
                    if (from_before) {
                        embed_store(part + (2 * w) * d, c0, d, vec, acc);
                    } else if (!ends) {
                        embed_store(part + (2 * w + 1) * d, c0, d, vec, acc);
                    } else {
                        const float4 v = make_float4(acc.x * scale, acc.y * scale, acc.z * scale,
                                                     acc.w * scale);
                        embed_store(out + static_cast<long long>(s_key[i]) * ld, c0, d, vec,
                                    v);
                    }
                    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    from_before = false;
                }
            }
        }
    }
}

// One block per window whose last run starts in it and goes on: the run's parts in order.
__global__ void __launch_bounds__(256)
    embed_join_kernel(const uint32_t* keys, long long n, int window, uint32_t rows,
                      int d, float scale, float* __restrict__ out, long long ld,
                      const float* part, int vec) {
    grid_wait();
    const long long w = blockIdx.x;
    const long long next = (w + 1) * window;   // first token of the next window
    if (next >= n) return;
    const uint32_t key = keys[next - 1];
    if (key >= rows || keys[next] != key) return;
    if (w > 0 && keys[w * window - 1] == key) return;  // it started earlier
    const int c0 = blockIdx.y * kEmbedPiece;
    // the run's end: the first token of another key (keys are sorted)
    long long lo = next, hi = n;
    while (lo < hi) {
        const long long mid = (lo + hi) / 2;
        if (keys[mid] > key) hi = mid; else lo = mid + 1;
    }
    const long long last = (lo - 1) / window;  // the window that holds the run's last token
    float4 acc = embed_load(part + (2 * w + 1) * d, c0, d, vec);
    constexpr int kAhead = 8;
    for (long long v = w + 1; v <= last; v += kAhead) {
        float4 g[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            g[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (v + j <= last) g[j] = embed_load(part + (2 * (v + j)) * d, c0, d, vec);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (v + j <= last) {
                acc.x += g[j].x;
                acc.y += g[j].y;
                acc.z += g[j].z;
                acc.w += g[j].w;
            }
        }
    }
    embed_store(out + static_cast<long long>(key) * ld, c0, d, vec,
                make_float4(acc.x * scale, acc.y * scale, acc.z * scale, acc.w * scale));
}

}  // namespace mfk
