// Host side of the operators between a layer's projections (adapters, heads, attention) against the HIP stand-in (hipstub.cpp, built
// with its hipLaunchKernel renamed to hipstub_launch): every form of every call from the smallest sizes to the largest
// that the header allows, from one thread and then from four at once.  Every launch is checked against what a launch may be;
// workspaces are asked for and given exactly.  "Device" addresses are made up: nothing on the host may touch them.
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <atomic>
#include <cstdio>
#include <cstdlib>
#include <thread>
#include <vector>

#include "../../include/sptmm.h"

extern "C" hipError_t hipstub_launch(const void *f, dim3 grid, dim3 block, void **args, size_t shmem, hipStream_t st);
static std::atomic<long> launches{0};

extern "C" hipError_t hipLaunchKernel(const void *f, dim3 grid, dim3 block, void **args, size_t shmem, hipStream_t st)
{
    ++launches;
    const unsigned long threads = (unsigned long)block.x * block.y * block.z;
    if (!grid.x || !grid.y || !grid.z || !threads || threads > 1024 || (unsigned long)grid.x * block.x >= 1ul << 32 || grid.y > 65535 || grid.z > 65535 || shmem > 64 << 10) {
        fprintf(stderr, "a launch of %u x %u x %u workgroups of %lu, %zu bytes\n", grid.x, grid.y, grid.z, threads, shmem);
        exit(1);
    }
    return hipstub_launch(f, grid, block, args, shmem, st);
}

#define IS(x, want)                                                                              \
    do {                                                                                         \
        const long rc_ = (long)(x);                                                              \
        if (rc_ != (long)(want)) {                                                               \
            fprintf(stderr, "%s -> %ld, not %ld: %s\n", #x, rc_, (long)(want), sptmm_last_error()); \
            exit(1);                                                                             \
        }                                                                                        \
    } while (0)
#define OK(x) IS(x, SPTMM_OK)

template <typename T> T *at(size_t i) { return (T *)(((size_t)1 << 40) + (i << 36)); }

static void adapters(int K, int N, int type, int slots, int max_rank)
{
    sptmm_adapters *a = nullptr;
    OK(sptmm_adapters_create(K, N, type, slots, max_rank, &a));
    for (int rank : {0, 1, (max_rank + 1) / 2, max_rank})
        for (int slot : {0, slots - 1}) OK(sptmm_adapters_set(a, slot, at<uint16_t>(1), at<uint16_t>(2), rank, 0.5f, nullptr));
    IS(sptmm_adapters_set(a, slots, at<uint16_t>(1), at<uint16_t>(2), 1, 0.5f, nullptr), SPTMM_ERR_INVALID);
    size_t before = 0;
    for (int M : {1, 2, 15, 16, 17, 48, 64, 127, 128, 129, 333, 1000, 3001, 4080, 4096, 20000, 1 << 20, 1 << 24}) {
        const size_t n = sptmm_adapters_workspace_bytes(a, M);
        if (n < before) IS(M, 0);  // (fewer rows never need more)
        before = n;
        const bool fits = (int64_t)((M + 15) / 16) * (((N + 31) / 32 + 3) / 4) < 1 << 24;
        for (const float *base : {(const float *)nullptr, (const float *)at<float>(4), (const float *)at<float>(5)})
            IS(sptmm_adapters_apply(a, at<uint16_t>(3), at<int32_t>(6), M, base, at<float>(5), n ? at<void>(7) : nullptr, n, nullptr), fits ? SPTMM_OK : SPTMM_ERR_UNSUPPORTED);
    }
    sptmm_adapters_free(a);
}

static void heads(int tokens, int q_heads, int kv_heads, int dim, int shift)
{
    std::vector<double> f(dim / 2, 0.25);
    for (int in : {1, 2, 3})
        for (int out : {1, 2})
            for (int pairs : {0, dim / 4, dim / 2})
                for (int inter : {0, 1}) {
                    sptmm_rotation r;
                    OK(sptmm_rotation_init(f.data(), pairs, inter, &r));
                    sptmm_heads_args a{};
                    const size_t isz = in == 3 ? 4 : 2;
                    a.q = at<char>(1) + shift * isz, a.k = at<char>(2) + shift * isz, a.v = at<char>(3) + shift * isz;
                    a.q_stride = a.q_out_stride = (int64_t)q_heads * dim + shift, a.k_stride = a.v_stride = a.k_out_stride = a.v_out_stride = (int64_t)kv_heads * dim + shift;
                    a.in_type = in, a.out_type = out, a.q_out = at<char>(4), a.k_out = at<char>(5), a.v_out = at<char>(6);
                    a.tokens = tokens, a.q_heads = q_heads, a.kv_heads = kv_heads, a.head_dim = dim;
                    a.positions = at<int32_t>(7), a.kv_rows = at<int32_t>(8), a.kv_capacity = 100, a.eps = 1e-5f, a.rotation = &r;
                    a.q_gain = pairs ? at<float>(9) : nullptr, a.k_gain = inter ? at<float>(10) : nullptr;
                    OK(sptmm_heads_norm_rotate(&a, nullptr));
                    a.v = nullptr;
                    OK(sptmm_heads_norm_rotate(&a, nullptr));
                }
}

static void attention(int batch, int total_q, int max_q, int max_kv, int q_heads, int kv_heads, int dim, int64_t kv_rows)
{
    for (int type : {SPTMM_X_F16, SPTMM_X_BF16}) {
        sptmm_attention_args a{};
        a.q = at<uint16_t>(1), a.k = at<uint16_t>(2), a.v = at<uint16_t>(3), a.out = at<uint16_t>(4);
        a.q_stride = a.out_stride = (int64_t)q_heads * dim, a.k_stride = a.v_stride = (int64_t)kv_heads * dim;
        a.kv_rows = kv_rows, a.q_start = at<int32_t>(5), a.kv_start = at<int32_t>(6), a.kv_len = at<int32_t>(7);
        a.batch = batch, a.total_q = total_q, a.max_q = max_q, a.max_kv = max_kv, a.q_heads = q_heads, a.kv_heads = kv_heads, a.head_dim = dim, a.type = type, a.scale = 0.125f;
        const size_t n = sptmm_attention_workspace_bytes(&a);
        OK(sptmm_attention(&a, n ? at<void>(8) : nullptr, n, nullptr));
        a.kv_start = a.kv_len = nullptr;
        OK(sptmm_attention(&a, n ? at<void>(8) : nullptr, n, nullptr));
        if (n) IS(sptmm_attention(&a, nullptr, n, nullptr), SPTMM_ERR_INVALID);
    }
}

static void all()
{
    for (int type : {SPTMM_X_F16, SPTMM_X_BF16}) {
        adapters(16, 16, type, 1, 1);
        adapters(2560, 3840, type, 8, 16);
        adapters(6912, 2560, type, 3, 64);
        adapters(2560, 13824, type, 2, 256);
        adapters(48, 1 << 14, type, 1, 200);
    }
    for (int tokens : {0, 1, 7, 1023, 1024, 20011, 1 << 30})
        for (int dim : {2, 34, 64, 128, 250, 256})
            for (int shift : {0, 1, 8}) heads(tokens, 20, 5, dim, shift), heads(tokens, 0, 3, dim, shift), heads(tokens, 65535, 0, dim, shift);
    for (int dim : {8, 64, 72, 128, 136, 256}) {
        for (int batch : {0, 1, 3, 32, 64, 100, 1000, 50000})
            for (int max_q : {0, 1, 8, 60, 500, 1 << 30})
                for (int max_kv : {0, 1, 129, 5000, 1 << 30}) {
                    const int total = batch * std::min(std::max(max_q, 1), 64);
                    attention(batch, total, max_q, max_kv, 20, 5, dim, 1 << 20);
                    attention(batch, total + 3, max_q, max_kv, 16, 16, dim, 1 << 30);
                    attention(batch, total, max_q, max_kv, 40, 1, dim, 0);
                }
        for (int max_q : {1, 1 << 30}) {  // the largest
            attention(1 << 22, 1 << 22, max_q, 1 << 30, 1, 1, dim, 1 << 30);
            const int most = std::min(65535, (1 << 22) / dim);  // (a row of keys is at most 2^22 elements)
            attention(64, 1 << 13, max_q, 1 << 30, most, most, dim, 1 << 30);
            attention(1, 1 << 29, max_q, 1 << 30, 1, 1, dim, 1 << 30);
            attention(1, 1 << 13, max_q, 1 << 30, 65535, 1, dim, 1 << 30);
        }
    }
}

int main()
{
    sptmm_devinfo info;
    OK(sptmm_device_init(0, &info));
    all();
    printf("one thread: %ld launches\n", launches.load());
    std::vector<std::thread> th;
    for (int t = 0; t < 4; ++t) th.emplace_back(all);
    for (auto &t : th) t.join();
    printf("four threads: %ld launches in all\n", launches.load());
    return 0;
}
