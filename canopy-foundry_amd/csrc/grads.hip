// The global norm of a list of gradients, and the gradients clipped by it:
//     S = sum over all tensors of g^2,  norm = sqrt(S),  coef = norm > max_norm ? max_norm / norm : 1,  out = T(g * coef).
// What bounds it: HBM; the gradients are read twice, but for up to 256 MB that stay in the last-level cache.  The sum of 3.9 GB in fp32 runs at 6.5 to 6.6 TB/s, both
// at 5.7 to 6.2, by the card (a copy of 4 GiB at 4.9).
// S is summed in 64 bits: the square of a large or a small fp32 gradient does not fit fp32, and a billion terms lose their last bits there.
// The sums' order follows from the list alone, so the same gradients give the same norm.
#include "common.hpp"

#include <cmath>

namespace cf {
namespace {

constexpr int kThreads = 256;
constexpr size_t kChunk = 16384;                // elements of one entry at most
// entries at the list's end that the sum leaves in the caches for the clipping, which begins there: 256 MB of fp32, 128 MB of bf16
constexpr unsigned kCached = 4096;
constexpr int kMaxParts = 2048;                 // workgroups that leave a partial sum

struct Entry {                                  // a run of one tensor's elements
    const void* src;
    void* dst;
    uint32_t count;
    uint32_t is_f32;
    uint64_t unused;
};
static_assert(sizeof(Entry) == 32);

__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// Sixteen bytes at any alignment an element has: one instruction all the same.  (Entries begin on 16 bytes but for a tensor's first: 1.9 GB of bf16
// tensors one element off 2254 us before that, 1874 since; aligned ones 1870.)
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// f(values, number) for each whole run of `per` elements (16 bytes) of an entry; a thread's runs lie kThreads apart and are loaded eight at a time.
// STREAM: past the caches.
template <bool STREAM, class F>
__device__ __forceinline__ void sweep(const Entry& e, F&& f) {
    const unsigned runs = e.count / (e.is_f32 ? 4 : 8);
    const u32x4_any* src = static_cast<const u32x4_any*>(e.src);
    auto load = [&](unsigned r) {
        if constexpr (STREAM) return __builtin_nontemporal_load(src + r);
        else return src[r];
    };
    unsigned r = threadIdx.x;
    u32x4_any v[8];
    for (; r + 7 * kThreads < runs; r += 8 * kThreads) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = load(r + k * kThreads);
#pragma unroll
        for (int k = 0; k < 8; ++k) f(v[k], r + k * kThreads);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (r + k * kThreads < runs) v[k] = load(r + k * kThreads);
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (r + k * kThreads < runs) f(v[k], r + k * kThreads);
}

__global__ __launch_bounds__(kThreads) void k_grad_sumsq(const Entry* __restrict__ list, unsigned chunks, double* __restrict__ parts) {
    __shared__ double sh[4];
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
        const Entry e = list[c];
        auto add = [&](int k, float g) { sum[k] = fma(static_cast<double>(g), static_cast<double>(g), sum[k]); };
        auto all = [&](auto f) {
            if (c + kCached < chunks) sweep<true>(e, f);
            else sweep<false>(e, f);
        };
        if (e.is_f32) {
            all([&](const u32x4_any& v, unsigned) {
#pragma unroll
                for (int k = 0; k < 4; ++k) add(k, __uint_as_float(v[k]));
            });
            for (unsigned i = (e.count & ~3u) + threadIdx.x; i < e.count; i += kThreads) add(0, static_cast<const float*>(e.src)[i]);
        } else {
            all([&](const u32x4_any& v, unsigned) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    add(k, bf16_lo(v[k]));
                    add(k, bf16_hi(v[k]));
                }
            });
            for (unsigned i = (e.count & ~7u) + threadIdx.x; i < e.count; i += kThreads) add(0, bf16_to_f32(static_cast<const uint16_t*>(e.src)[i]));
        }
    }
    const double all = block_sum((sum[0] + sum[1]) + (sum[2] + sum[3]), sh);
    if (threadIdx.x == 0) parts[blockIdx.x] = all;
}

// sqrt of the parts' sum, in every thread
__device__ __forceinline__ double norm_of(const double* __restrict__ parts, int n, double* sh) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) v += parts[i];
    return sqrt(block_sum(v, sh));
}

__global__ __launch_bounds__(kThreads) void k_grad_norm(const double* __restrict__ parts, int n, float* __restrict__ norm) {
    __shared__ double sh[4];
    const double v = norm_of(parts, n, sh);
    if (threadIdx.x == 0) *norm = static_cast<float>(v);
}

// parts null: the norm is given in *norm_in
__global__ __launch_bounds__(kThreads) void k_grad_clip(const Entry* __restrict__ list, unsigned chunks, const double* __restrict__ parts, int n,
                                                        const float* norm_in, float max_norm, float* norm_out, float* coef_out) {
    __shared__ double sh[4];
    // the norm as the caller sees it, so that one call and two (a norm summed over several GPUs between them) clip alike
    const float norm = parts ? static_cast<float>(norm_of(parts, n, sh)) : *norm_in;
    // a norm that is no finite number gives no direction to keep: the gradients stay as they are
    const float coef = norm > max_norm && norm < __builtin_inff() ? static_cast<float>(static_cast<double>(max_norm) / norm) : 1.0f;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        if (norm_out) *norm_out = norm;
        if (coef_out) *coef_out = coef;
    }
    // The entries that this workgroup, and with it this XCD, summed, the last ones first: those are what the sum left in the caches.  (32 tensors of
    // 3.1 million elements in all: 15.5 us with the list walked from its end by whichever workgroup, 12.4 so; 67 MB 37.4 and 36.2.)
    if (blockIdx.x >= chunks) return;
    for (unsigned turn = (chunks - 1 - blockIdx.x) / gridDim.x + 1; turn-- > 0;) {
        const unsigned c = blockIdx.x + turn * gridDim.x;
        const Entry e = list[c];
        auto all = [&](auto f) {
            if (c + kCached < chunks) sweep<true>(e, f);
            else sweep<false>(e, f);
        };
        if (coef == 1.0f && e.src == e.dst) continue;
        u32x4_any* dst = static_cast<u32x4_any*>(e.dst);
        if (e.is_f32) {
            all([&](u32x4_any v, unsigned r) {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * coef);
                __builtin_nontemporal_store(v, dst + r);
            });
            for (unsigned i = (e.count & ~3u) + threadIdx.x; i < e.count; i += kThreads)
                static_cast<float*>(e.dst)[i] = static_cast<const float*>(e.src)[i] * coef;
        } else {
            all([&](u32x4_any v, unsigned r) {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = pack_bf16x2_hw(bf16_lo(v[k]) * coef, bf16_hi(v[k]) * coef);
                __builtin_nontemporal_store(v, dst + r);
            });
            for (unsigned i = (e.count & ~7u) + threadIdx.x; i < e.count; i += kThreads)
                static_cast<uint16_t*>(e.dst)[i] = static_cast<uint16_t>(pack_bf16x2_hw(bf16_to_f32(static_cast<const uint16_t*>(e.src)[i]) * coef, 0.0f));
        }
    }
}

bool misaligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

// the number of entries of a list, or an error below zero.  The kernels step beyond the last one in 32 bits.
long long entries_of(const void* d_list, size_t list_bytes) {
    if (list_bytes % sizeof(Entry) != 0 || list_bytes / sizeof(Entry) > 0x7fffffffull) return CF_ERR_INVALID_ARG;
    if (list_bytes && (!d_list || misaligned(d_list, 16))) return CF_ERR_INVALID_ARG;
    return static_cast<long long>(list_bytes / sizeof(Entry));
}
// Workgroups: 2048 over a long list (3.9 GB: 1884 us, 1024 of them 1946 on the same card; 2064 on another), 1024 over a short one, whose partial sums are the longer part (3000 tensors
// of 300: 15.0 us and 12.0).
unsigned grid_of(long long entries) {
    const long long most = entries >= 8192 ? kMaxParts : kMaxParts / 2;
    return static_cast<unsigned>(entries < 1 ? 1 : entries < most ? entries : most);
}
bool bad_workspace(const void* d_workspace, size_t bytes) { return !d_workspace || misaligned(d_workspace, 16) || bytes < kMaxParts * sizeof(double); }

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" {

int cf_grad_list_bytes(const size_t* counts, int num_tensors, size_t* bytes) {
    if (num_tensors < 0 || !bytes || (num_tensors > 0 && !counts)) return CF_ERR_INVALID_ARG;
    size_t entries = 0;
    for (int i = 0; i < num_tensors; ++i) {
        if (counts[i] >> 48) return CF_ERR_INVALID_ARG;
        if (counts[i]) entries += (counts[i] + 7 + kChunk - 1) / kChunk;        // the first may be cut short by up to seven elements
    }
    *bytes = entries * sizeof(Entry);
    return CF_OK;
}

int cf_grad_list_fill(void* const* d_tensors, void* const* d_out, const size_t* counts, const int* types, int num_tensors, void* list,
                      size_t list_bytes) {
    size_t need = 0;
    if (const int rc = cf_grad_list_bytes(counts, num_tensors, &need)) return rc;
    if (list_bytes < need || (list_bytes && !list) || (need && (!d_tensors || !types))) return CF_ERR_INVALID_ARG;
    for (int i = 0; i < num_tensors; ++i) {
        if (counts[i] == 0) continue;
        const unsigned el = types[i] == CF_GRAD_F32 ? 4 : 2;
        if (types[i] != CF_GRAD_F32 && types[i] != CF_GRAD_BF16) return CF_ERR_INVALID_ARG;
        if (!d_tensors[i] || misaligned(d_tensors[i], el) || (d_out && (!d_out[i] || misaligned(d_out[i], el)))) return CF_ERR_INVALID_ARG;
    }
    char* at = static_cast<char*>(list);
    auto put = [&](const Entry& e) {
        __builtin_memcpy(at, &e, sizeof(e));
        at += sizeof(e);
    };
    for (int i = 0; i < num_tensors; ++i) {
        const size_t el = types[i] == CF_GRAD_F32 ? 4 : 2;
        // a tensor's first entry is cut short so that the others begin on 16 bytes
        size_t most = kChunk - (reinterpret_cast<uintptr_t>(d_tensors[i]) & 15u) / el;
        for (size_t first = 0, n; first < counts[i]; first += n, most = kChunk) {
            n = counts[i] - first < most ? counts[i] - first : most;
            Entry e{};
            e.src = static_cast<const char*>(d_tensors[i]) + first * el;
            e.dst = static_cast<char*>(d_out ? d_out[i] : d_tensors[i]) + first * el;
            e.count = static_cast<uint32_t>(n);
            e.is_f32 = types[i] == CF_GRAD_F32;
            put(e);
        }
    }
    for (const char* end = static_cast<char*>(list) + list_bytes; end - at >= static_cast<ptrdiff_t>(sizeof(Entry));) put(Entry{});      // not needed
    return CF_OK;
}

int cf_grad_norm_workspace_bytes(size_t* bytes) {
    if (!bytes) return CF_ERR_INVALID_ARG;
    *bytes = kMaxParts * sizeof(double);
    return CF_OK;
}

int cf_grad_norm(const void* d_list, size_t list_bytes, float* d_norm, void* d_workspace, size_t workspace_bytes, cf_stream_t stream) {
    const long long entries = entries_of(d_list, list_bytes);
    if (entries < 0) return static_cast<int>(entries);
    if (!d_norm || misaligned(d_norm, 4) || bad_workspace(d_workspace, workspace_bytes)) return CF_ERR_INVALID_ARG;
    hipStream_t st = as_stream(stream);
    const unsigned grid = grid_of(entries);
    double* parts = static_cast<double*>(d_workspace);
    k_grad_sumsq<<<grid, kThreads, 0, st>>>(static_cast<const Entry*>(d_list), static_cast<unsigned>(entries), parts);
    k_grad_norm<<<1, kThreads, 0, st>>>(parts, grid, d_norm);
    return launch_status();
}

int cf_grad_clip(const void* d_list, size_t list_bytes, float max_norm, const float* d_norm, float* d_coef, cf_stream_t stream) {
    const long long entries = entries_of(d_list, list_bytes);
    if (entries < 0) return static_cast<int>(entries);
    if (!(max_norm >= 0.0f) || !d_norm || misaligned(d_norm, 4) || misaligned(d_coef, 4) || d_coef == d_norm) return CF_ERR_INVALID_ARG;
    hipStream_t st = as_stream(stream);
    k_grad_clip<<<grid_of(entries), kThreads, 0, st>>>(static_cast<const Entry*>(d_list), static_cast<unsigned>(entries), nullptr, 0, d_norm,
                                                       max_norm, nullptr, d_coef);
    return launch_status();
}

int cf_grad_norm_clip(const void* d_list, size_t list_bytes, float max_norm, float* d_norm, float* d_coef, void* d_workspace,
                      size_t workspace_bytes, cf_stream_t stream) {
    const long long entries = entries_of(d_list, list_bytes);
    if (entries < 0) return static_cast<int>(entries);
    if (!(max_norm >= 0.0f) || !d_norm || misaligned(d_norm, 4) || misaligned(d_coef, 4) || d_coef == d_norm ||
        bad_workspace(d_workspace, workspace_bytes))
        return CF_ERR_INVALID_ARG;
    hipStream_t st = as_stream(stream);
    const unsigned grid = grid_of(entries);
    double* parts = static_cast<double*>(d_workspace);
    k_grad_sumsq<<<grid, kThreads, 0, st>>>(static_cast<const Entry*>(d_list), static_cast<unsigned>(entries), parts);
    k_grad_clip<<<grid, kThreads, 0, st>>>(static_cast<const Entry*>(d_list), static_cast<unsigned>(entries), parts, grid, nullptr, max_norm,
                                           d_norm, d_coef);
    return launch_status();
}

}  // extern "C"
