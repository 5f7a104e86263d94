// Host side of the embedding kernels (embed.cuh). Part of the library's one translation unit.
#pragma once

namespace {

int check_embed(int64_t rows, int64_t d, int64_t n, int32_t id_bytes) {
    if (rows < 0 || d < 0 || n < 0 || (id_bytes != 4 && id_bytes != 8))
        return MFK_ERR_INVALID_ARGUMENT;
    if (rows > (int64_t(1) << 31) - 2 || n > (int64_t(1) << 31) - 4096 ||
        d > (int64_t(1) << 31) - 4096)
        return MFK_ERR_UNSUPPORTED;
    return MFK_OK;
}

template <typename ID>
int launch_embedding(const float* table, int64_t rows, int64_t d, int64_t ld, const ID* ids,
                     int64_t n, float scale, float* out, int64_t ld_out, const DeviceInfo* info,
                     cudaStream_t stream) {
    const int vec = d % 4 == 0 && ld % 4 == 0 && ld_out % 4 == 0 && aligned16(table) &&
                    aligned16(out);
    if (d <= 128) {
        int lanes = 1;
        while (lanes < 32 && lanes * (vec ? 4 : 1) < d) lanes *= 2;
        const int64_t per_block = 8 * 4 * (32 / lanes);
        auto kernel =
            vec ? mfk::embedding_narrow_kernel<ID, 4> : mfk::embedding_narrow_kernel<ID, 1>;
        kernel<<<static_cast<unsigned>((n + per_block - 1) / per_block), 256, 0, stream>>>(
            table, rows, static_cast<int>(d), ld, ids, n, scale, out, ld_out, lanes);
        g_launches.fetch_add(1);
        MFK_CUDA(cudaGetLastError());
        return MFK_OK;
    }
    const int64_t warps = n * ((d + 511) / 512);
    const int64_t blocks = std::min<int64_t>((warps + 7) / 8, int64_t(info->sm_count) * 64);
    mfk::embedding_kernel<ID><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(
        table, rows, static_cast<int>(d), ld, ids, n, scale, out, ld_out, vec);
    g_launches.fetch_add(1);
    MFK_CUDA(cudaGetLastError());
    return MFK_OK;
}

template <typename ID, int IT>
int launch_cluster_sort_it(const ID* ids, int64_t n, int ranks, int chunk, int64_t rows,
                           int64_t padding, int passes, uint32_t* marks, uint32_t* keys,
                           uint32_t* pos, int device, cudaStream_t stream) {
    auto kernel = mfk::embed_sort_kernel<ID, IT>;
    const int smem = (4 * chunk + 32 * 256 + 2 * 256 + 8) * 4;
    static std::atomic<uint64_t> ready{0};  // a bit per device
    if ((ready.load() >> device & 1u) == 0u) {
        MFK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (4 * IT * 1024 + 32 * 256 + 2 * 256 + 8) * 4));
        ready.fetch_or(uint64_t(1) << device);
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(static_cast<unsigned>(ranks), 1, 1);
    cfg.blockDim = dim3(1024, 1, 1);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    MFK_CUDA(cudaLaunchKernelEx(&cfg, kernel, ids, static_cast<int>(n), chunk,
                                static_cast<long long>(rows), static_cast<long long>(padding),
                                passes, marks, keys, pos));
    g_launches.fetch_add(1);
    return MFK_OK;
}

// A cluster of CTAs with 2048 tokens each, or up to 8192 where eight CTAs need that.
template <typename ID>
int launch_cluster_sort(const ID* ids, int64_t n, int64_t rows, int64_t padding, int passes,
                        uint32_t* marks, uint32_t* keys, uint32_t* pos, int device,
                        cudaStream_t stream) {
    const int ranks = static_cast<int>(
        std::min<int64_t>(mfk::kClusterSortRanks, (n + 2047) / 2048));
    const int chunk = static_cast<int>((n + ranks - 1) / ranks);
    if (chunk <= 2048)
        return launch_cluster_sort_it<ID, 2>(ids, n, ranks, chunk, rows, padding, passes, marks,
                                             keys, pos, device, stream);
    return launch_cluster_sort_it<ID, 8>(ids, n, ranks, chunk, rows, padding, passes, marks, keys,
                                         pos, device, stream);
}

int run_embedding_grad(const float* grad, int64_t n, int64_t d, int64_t ld_grad, const void* ids,
                       int32_t id_bytes, int64_t rows, float scale, int64_t padding, float* out,
                       int64_t ld, cudaStream_t stream) {
    int rc = check_embed(rows, d, n, id_bytes);
    if (rc != MFK_OK) return rc;
    if (rows == 0 || d == 0) return MFK_OK;
    if (out == nullptr || ld < d) return MFK_ERR_INVALID_ARGUMENT;
    if (n > 0 && (grad == nullptr || ids == nullptr || ld_grad < 0))
        return MFK_ERR_INVALID_ARGUMENT;
    int dev = 0;
    DeviceInfo* info = nullptr;
    rc = current_device(&dev, &info);
    if (rc != MFK_OK) return rc;
    if (n == 0) return x_zero(out, rows, d, ld, stream);

    const int vec = d % 4 == 0 && ld % 4 == 0 && ld_grad % 4 == 0 && aligned16(grad) &&
                    aligned16(out);
    const int pieces = static_cast<int>((d + mfk::kEmbedPiece - 1) / mfk::kEmbedPiece);
    // windows of 16 to 256 tokens: three blocks per SM or more, and short joins of long runs
    int window = 16;
    while (window < mfk::kEmbedMaxWindow && n * pieces / (window * 2) >= info->sm_count * 3)
        window *= 2;
    const int64_t windows = (n + window - 1) / window;
    const int tiles = static_cast<int>((n + mfk::kSortTile - 1) / mfk::kSortTile);
    if (windows * pieces > (int64_t(1) << 30) || pieces > 65535) return MFK_ERR_UNSUPPORTED;

    // one allocation: keys and positions twice, digit counts, the marks, the partial rows
    const size_t items = (static_cast<size_t>(n) + 63) / 64 * 64;
    const size_t counts = static_cast<size_t>(tiles) * 256;
    const size_t marks = (static_cast<size_t>(rows) + 31) / 32 + 64;
    const size_t part = static_cast<size_t>(windows) * 2 * static_cast<size_t>(d);
    uint8_t* base = nullptr;
    MFK_CUDA(cudaMallocAsync(reinterpret_cast<void**>(&base),
                             (part + 4 * items + counts + marks + 64) * 4, stream));
    struct Free {
        void* p;
        cudaStream_t s;
        ~Free() { cudaFreeAsync(p, s); }
    } release{base, stream};
    float* d_part = reinterpret_cast<float*>(base);
    uint32_t* words = reinterpret_cast<uint32_t*>(base) + (part + 63) / 64 * 64;
    uint32_t* keys[2] = {words, words + items};
    uint32_t* pos[2] = {words + 2 * items, words + 3 * items};
    uint32_t* d_counts = words + 4 * items;
    uint32_t* d_marks = d_counts + counts;
    int passes = 0;
    while (passes < 4 && (rows >> (passes * 8)) != 0) ++passes;
    int at = 0;
    if (n <= mfk::kClusterSortMax) {
        rc = id_bytes == 8 ? launch_cluster_sort(static_cast<const int64_t*>(ids), n, rows, padding,
                                                 passes, d_marks, keys[0], pos[0], dev, stream)
                           : launch_cluster_sort(static_cast<const int32_t*>(ids), n, rows, padding,
                                                 passes, d_marks, keys[0], pos[0], dev, stream);
        if (rc != MFK_OK) return rc;
    } else {
        MFK_CUDA(cudaMemsetAsync(d_marks, 0, marks * 4, stream));
        if (id_bytes == 8) {
            mfk::embed_keys_kernel<int64_t><<<tiles, 256, 0, stream>>>(
                static_cast<const int64_t*>(ids), n, rows, padding, keys[0], d_marks, d_counts,
                tiles);
        } else {
            mfk::embed_keys_kernel<int32_t><<<tiles, 256, 0, stream>>>(
                static_cast<const int32_t*>(ids), n, rows, padding, keys[0], d_marks, d_counts,
                tiles);
        }
        g_launches.fetch_add(1);
        for (int pass = 0; pass < passes; ++pass) {
            if (pass > 0) {
                mfk::sort_count_kernel<<<tiles, 256, 0, stream>>>(keys[at], n, pass * 8, d_counts,
                                                                  tiles);
                g_launches.fetch_add(1);
            }
            mfk::sort_scan_kernel<<<1, 1024, 0, stream>>>(d_counts, static_cast<int64_t>(counts));
            mfk::sort_scatter_kernel<<<tiles, 256, 0, stream>>>(
                keys[at], pass > 0 ? pos[at] : nullptr, n, pass * 8, d_counts, tiles, keys[at ^ 1],
                pos[at ^ 1]);
            g_launches.fetch_add(2);
            at ^= 1;
        }
    }
    const int sum_blocks = static_cast<int>(windows * pieces);
    const int64_t zero_blocks = std::min<int64_t>((rows + 7) / 8, int64_t(info->sm_count) * 64);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = stream;
    cfg.gridDim = dim3(static_cast<unsigned>(sum_blocks + zero_blocks), 1, 1);
    const uint32_t *sorted = keys[at], *order = pos[at], *present = d_marks;
    MFK_CUDA(cudaLaunchKernelEx(&cfg, mfk::embed_sum_kernel, sorted, order,
                                static_cast<long long>(n), window, static_cast<uint32_t>(rows),
                                grad, static_cast<long long>(ld_grad), static_cast<int>(d), scale,
                                out, static_cast<long long>(ld), d_part, vec, pieces, sum_blocks,
                                present));
    g_launches.fetch_add(1);
    if (windows > 1) {
        cfg.gridDim = dim3(static_cast<unsigned>(windows), static_cast<unsigned>(pieces), 1);
        MFK_CUDA(cudaLaunchKernelEx(&cfg, mfk::embed_join_kernel, sorted,
                                    static_cast<long long>(n), window,
                                    static_cast<uint32_t>(rows), static_cast<int>(d), scale, out,
                                    static_cast<long long>(ld), static_cast<const float*>(d_part),
                                    vec));
        g_launches.fetch_add(1);
    }
    MFK_CUDA(cudaGetLastError());
    return MFK_OK;
}

}  // namespace

extern "C" {

int mfk_embedding_f32(const float* table, int64_t rows, int64_t d, int64_t ld, const void* ids,
                      int32_t id_bytes, int64_t n, float scale, float* out, int64_t ld_out,
                      void* stream) {
    int rc = check_embed(rows, d, n, id_bytes);
    if (rc != MFK_OK) return rc;
    if (n == 0 || d == 0) return MFK_OK;
    if (rows == 0 || table == nullptr || ids == nullptr || out == nullptr || ld_out < d ||
        ld < 0)
        return MFK_ERR_INVALID_ARGUMENT;
    int dev = 0;
    DeviceInfo* info = nullptr;
    rc = current_device(&dev, &info);
    if (rc != MFK_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (id_bytes == 8)
        return launch_embedding(table, rows, d, ld, static_cast<const int64_t*>(ids), n, scale,
                                out, ld_out, info, s);
    return launch_embedding(table, rows, d, ld, static_cast<const int32_t*>(ids), n, scale, out,
                            ld_out, info, s);
}

int mfk_embedding_grad_f32(const float* grad, int64_t n, int64_t d, int64_t ld_grad,
                           const void* ids, int32_t id_bytes, int64_t rows, float scale,
                           int64_t padding, float* out, int64_t ld, void* stream) {
    return run_embedding_grad(grad, n, d, ld_grad, ids, id_bytes, rows, scale, padding, out, ld,
                              static_cast<cudaStream_t>(stream));
}

}  // extern "C"
