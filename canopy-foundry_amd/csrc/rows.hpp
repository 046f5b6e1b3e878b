// What the kernels that hold a row in registers share: eight elements a chunk at any alignment, reductions over a row's threads, recording a maximum from
// every row.
#pragma once
#include "common.hpp"
#include "row_threads.hpp"

namespace cf {

static_assert(kRowWave == kWave);
constexpr int kMaxH = 16384;

enum { Q_ROWS = 0, Q_BLOCK = 1, Q_RECORD = 2 };

// Eight elements at any alignment that one element has: gfx950 moves them in one instruction all the same.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// Eight elements as they lie in memory; converted where they are used, so that a load on its way is not waited for.
template <bool F32>
struct Raw8 {
    u32x4_any v[F32 ? 2 : 1];
    __device__ __forceinline__ float at(int i) const {
        if constexpr (F32) return __uint_as_float(v[i >> 2][i & 3]);
        else return (i & 1) ? bf16_hi(v[0][i >> 1]) : bf16_lo(v[0][i >> 1]);
    }
};
// A row's last chunk, n < 8 elements (TAIL), is loaded whole where enough follows, and cut when it is used: element by element the loads of the
// last lane kept a row waiting for eight of them in turn (8192 x 4095: 88 us, now 55; 4096 43).  `whole`: the eight elements lie in the tensor.
template <bool F32, bool TAIL>
__device__ __forceinline__ void load8(const void* p, size_t at, int n, bool whole, Raw8<F32>& r) {
    if (!TAIL || n >= 8 || whole) {
        const u32x4_any* q = F32 ? reinterpret_cast<const u32x4_any*>(static_cast<const float*>(p) + at)
                                 : reinterpret_cast<const u32x4_any*>(static_cast<const uint16_t*>(p) + at);
        r.v[0] = q[0];
        if constexpr (F32) r.v[1] = q[1];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) {
                if constexpr (F32) r.v[i >> 2][i & 3] = static_cast<const uint32_t*>(p)[at + i];
                else r.v[0][i >> 1] |= static_cast<uint32_t>(static_cast<const uint16_t*>(p)[at + i]) << (16 * (i & 1));
            }
    }
}
template <bool F32>
__device__ __forceinline__ void clear8(Raw8<F32>& r) {
    r.v[0] = u32x4_any{0, 0, 0, 0};
    if constexpr (F32) r.v[1] = u32x4_any{0, 0, 0, 0};
}
template <bool F32, bool TAIL>
__device__ __forceinline__ float value8(const Raw8<F32>& r, int i, int n) {
    return !TAIL || i < n ? r.at(i) : 0.0f;
}
// Eight weights as bf16 pairs.  A last chunk is the end of the eight elements that the weight ends with, moved down.
template <bool TAIL>
__device__ __forceinline__ u32x4_any load_weight(const uint16_t* w, int at, int n, int H) {
    if (!TAIL || n >= 8) return *reinterpret_cast<const u32x4_any*>(w + at);
    u32x4_any v = {0, 0, 0, 0};
    if (H >= 8) {
        v = *reinterpret_cast<const u32x4_any*>(w + H - 8);
        const int down = 8 - n;
        if (down & 4) v = u32x4_any{v[2], v[3], 0, 0};
        if (down & 2) v = u32x4_any{v[1], v[2], v[3], 0};
        if (down & 1) v = u32x4_any{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) v[i >> 1] |= static_cast<uint32_t>(w[at + i]) << (16 * (i & 1));
    }
    return v;
}
// Streaming stores, which leave through the L2 (plain ones: 8192 x 4096 45.4 us instead of 42.9, 16384 x 1024 25.3 instead of 21.6).  A last chunk
// goes in pieces of four, two and one elements.
template <bool TAIL>
__device__ __forceinline__ void store8_bf16(uint16_t* p, size_t at, int n, const float (&v)[8]) {
    u32x4_any o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2_hw(v[2 * i], v[2 * i + 1]);
    if (!TAIL || n >= 8) {
        __builtin_nontemporal_store(o, reinterpret_cast<u32x4_any*>(p + at));
    } else {
        typedef uint32_t u32_any __attribute__((aligned(2)));
        uint16_t* q = p + at;
        if (n & 4) {
            reinterpret_cast<u32_any*>(q)[0] = o[0];
            reinterpret_cast<u32_any*>(q)[1] = o[1];
        }
        if (n & 2) *reinterpret_cast<u32_any*>(q + (n & 4)) = (n & 4) ? o[2] : o[0];
        if (n & 1) q[n - 1] = static_cast<uint16_t>(n == 1 ? o[0] : n == 3 ? o[1] : n == 5 ? o[2] : o[3]);
    }
}
// An fp32 chunk goes in two halves, so that a line is written by two instructions.  PAST_L2 lets them leave at once (forward: 2000 rows of 7168 28.3 us, 33.8 without); the gradient's lines are gathered in the L2 (8192 x 4096 90.1 -> 87.9 us).
template <bool F32, bool TAIL, bool PAST_L2>
__device__ __forceinline__ void store8_stream(void* p, size_t at, int n, const float (&v)[8]) {
    if constexpr (!F32) {
        store8_bf16<TAIL>(static_cast<uint16_t*>(p), at, n, v);
    } else {
        f32x4_any* q = reinterpret_cast<f32x4_any*>(static_cast<float*>(p) + at);
        const f32x4_any a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
        if (!TAIL || n >= 4) {
            if constexpr (PAST_L2) __builtin_nontemporal_store(a, q);
            else *q = a;
        }
        if (!TAIL || n >= 8) {
            if constexpr (PAST_L2) __builtin_nontemporal_store(b, q + 1);
            else q[1] = b;
        } else {
            float* r = static_cast<float*>(p) + at;
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (i >= (n & 4) && i < n) r[i] = v[i];
        }
    }
}
// Eight values as bytes by the conversion alone: what is not above the format's largest value by more than roundings, or, after saturate_fp8(), anything
// finite.  A NaN is a NaN; an infinity is one in E4M3 and an infinity in E5M2.
template <bool E5M2>
__device__ __forceinline__ u32x2_any convert8_fp8(const float (&v)[8]) {
    u32x2_any o;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int r = 0;
        if constexpr (E5M2) {
            r = __builtin_amdgcn_cvt_pk_bf8_f32(v[4 * i], v[4 * i + 1], r, false);
            r = __builtin_amdgcn_cvt_pk_bf8_f32(v[4 * i + 2], v[4 * i + 3], r, true);
        } else {
            r = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], r, false);
            r = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], r, true);
        }
        o[i] = static_cast<uint32_t>(r);
    }
    return o;
}
// From here on the wavefront's conversions to 8 bits give the largest finite value for finite ones beyond it (MODE.FP16_OVFL, which holds for fp16 and bf16 as well), so
// that no clamp is needed.  What is converted has to be a product with `factor`, by which the compiler cannot move it up past the change.
__device__ __forceinline__ void saturate_fp8(float& factor) {
    asm volatile("s_setreg_imm32_b32 hwreg(HW_REG_MODE, 23, 1), 1\n\ts_nop 1" : "+v"(factor));
}
// Eight values as bytes; finite: there is no NaN among them.
__device__ __forceinline__ u32x2_any pack8_fp8(bool e5m2, bool finite, const float (&v)[8]) {
    u32x2_any o;
    if (finite) {
        o.x = e5m2 ? cvt4_fp8_finite<true>(v[0], v[1], v[2], v[3]) : cvt4_fp8_finite<false>(v[0], v[1], v[2], v[3]);
        o.y = e5m2 ? cvt4_fp8_finite<true>(v[4], v[5], v[6], v[7]) : cvt4_fp8_finite<false>(v[4], v[5], v[6], v[7]);
    } else {
        o.x = e5m2 ? cvt4_fp8<true>(v[0], v[1], v[2], v[3]) : cvt4_fp8<false>(v[0], v[1], v[2], v[3]);
        o.y = e5m2 ? cvt4_fp8<true>(v[4], v[5], v[6], v[7]) : cvt4_fp8<false>(v[4], v[5], v[6], v[7]);
    }
    return o;
}
template <bool TAIL, bool PAST_L2 = true>
__device__ __forceinline__ void store8_bytes(uint8_t* p, size_t at, int n, u32x2_any o) {
    if (!TAIL || n >= 8) {
        if constexpr (PAST_L2) __builtin_nontemporal_store(o, reinterpret_cast<u32x2_any*>(p + at));
        else *reinterpret_cast<u32x2_any*>(p + at) = o;
    } else {
        typedef uint32_t u32_byte __attribute__((aligned(1)));
        typedef uint16_t u16_byte __attribute__((aligned(1)));
        uint8_t* q = p + at;
        uint32_t rest = o.x;
        if (n & 4) {
            *reinterpret_cast<u32_byte*>(q) = o.x;
            rest = o.y;
            q += 4;
        }
        if (n & 2) {
            *reinterpret_cast<u16_byte*>(q) = static_cast<uint16_t>(rest);
            rest >>= 16;
            q += 2;
        }
        if (n & 1) *q = static_cast<uint8_t>(rest);
    }
}
template <bool TAIL>
__device__ __forceinline__ void store8_fp8(uint8_t* p, size_t at, int n, bool e5m2, bool finite, const float (&v)[8]) {
    store8_bytes<TAIL>(p, at, n, pack8_fp8(e5m2, finite, v));
}
// Eight E4M3 bytes as the values they stand for times `scale`.
__device__ __forceinline__ void unpack8_e4m3(const u32x2_any& v, float scale, float (&o)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(v[i]), false);
        const f32x2_t b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(v[i]), true);
        o[4 * i] = a.x * scale;
        o[4 * i + 1] = a.y * scale;
        o[4 * i + 2] = b.x * scale;
        o[4 * i + 3] = b.y * scale;
    }
}
// Eight bytes, n of them where neither that many follow nor the chunk is whole.
template <bool TAIL>
__device__ __forceinline__ u32x2_any load8_bytes(const uint8_t* p, size_t at, int n, bool whole) {
    if (!TAIL || n >= 8 || whole) return *reinterpret_cast<const u32x2_any*>(p + at);
    u32x2_any v = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) v[i >> 2] |= static_cast<uint32_t>(p[at + i]) << (8 * (i & 3));
    return v;
}

// What a value is after the lanes of a group of 16 have exchanged it, by DPP: quad, half row, row.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true); }
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, dpp<0xb1>(v));           // lane ^ 1
    v = max(v, dpp<0x4e>(v));           // lane ^ 2
    v = max(v, dpp<0x141>(v));          // the other quad of the half row
    return max(v, dpp<0x140>(v));       // the other half of the row
}
__device__ __forceinline__ float add16(float v) {
    v += __uint_as_float(dpp<0xb1>(__float_as_uint(v)));
    v += __uint_as_float(dpp<0x4e>(__float_as_uint(v)));
    v += __uint_as_float(dpp<0x141>(__float_as_uint(v)));
    return v + __uint_as_float(dpp<0x140>(__float_as_uint(v)));
}
// Over a row's threads, the same in each.  A row of more than one wavefront is a workgroup's only one; `sh` holds a word for each of its
// wavefronts, at most 16, and is not used again.
template <bool ONE_WAVE>
__device__ __forceinline__ float row_sum(float v, float* sh) {
    v = add16(v);
    v += __shfl_xor(v, 16, kWave);
    v += __shfl_xor(v, 32, kWave);
    if constexpr (!ONE_WAVE) {
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
        __syncthreads();
        const int w = threadIdx.x & 15;
        v = add16(w < static_cast<int>(blockDim.x >> 6) ? sh[w] : 0.0f);
    }
    return v;
}
template <bool ONE_WAVE>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* sh) {
    v = max16(v);
    v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16, kWave)));
    v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 32, kWave)));
    if constexpr (!ONE_WAVE) {
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
        __syncthreads();
        const int w = threadIdx.x & 15;
        v = max16(w < static_cast<int>(blockDim.x >> 6) ? sh[w] : 0u);
    }
    return v;
}

constexpr uint32_t kInf = 0x7f800000u;
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Over a row's threads in 64 bits, as row_sum().
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = dpp<CTRL>(static_cast<uint32_t>(b)), hi = dpp<CTRL>(static_cast<uint32_t>(b >> 32));
    return __builtin_bit_cast(double, hi << 32 | lo);
}
__device__ __forceinline__ double add16(double v) {
    v += dpp64<0xb1>(v);
    v += dpp64<0x4e>(v);
    v += dpp64<0x141>(v);
    return v + dpp64<0x140>(v);
}
template <bool ONE_WAVE>
__device__ __forceinline__ double row_sum(double v, double* sh) {
    v = add16(v);
    v += __shfl_xor(v, 16, kWave);
    v += __shfl_xor(v, 32, kWave);
    if constexpr (!ONE_WAVE) {
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
        __syncthreads();
        const int w = threadIdx.x & 15;
        v = add16(w < static_cast<int>(blockDim.x >> 6) ? sh[w] : 0.0);
    }
    return v;
}

// The root mean square of a row that its threads hold in chunks of eight, V each: sqrt(mean(h^2) + eps) = 2^e times what is returned, with the row scaled by
// 2^-e, which h / rms does not see.  e is 0 but where squares leave fp32 (|h| of 1e19 and more, or of 1e-15 and less under as small an eps): then the sum is taken once
// more of the scaled row.  A row that holds infinities or NaNs stays as it is.  SUM: the type of the sum; the mean, eps's addition and the root are one rounding to fp32 each.  `sh`: two sums, `sh_max`: one maximum, as row_sum() and row_max() ask.
template <bool ONE_WAVE, int V, typename SUM>
__device__ __forceinline__ float row_rms(float (&h)[V][8], int H, float eps, SUM (*sh)[16], uint32_t* sh_max, int& e) {
    auto mean_square = [&](SUM* s) {
        SUM ss = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            SUM part = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const SUM v = h[j][i];
                if constexpr (sizeof(SUM) == 8) part = __builtin_fma(v, v, part);
                else part = __builtin_fmaf(v, v, part);
            }
            ss += part;
        }
        return static_cast<float>(row_sum<ONE_WAVE>(ss, s) / static_cast<SUM>(H));
    };
    float mean = mean_square(sh[0]) + eps;
    e = 0;
    if (!(mean >= 1e-30f && mean < __builtin_inff())) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, abs_bits(h[j][i]));
        m = row_max<ONE_WAVE>(m, sh_max);
        const float most = fmaxf(__uint_as_float(m), sqrtf(eps));
        if (m < kInf && most > 0.0f) {
            e = __builtin_amdgcn_frexp_expf(most);
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) h[j][i] = ldexpf(h[j][i], -e);
            mean = mean_square(sh[1]) + ldexpf(eps, -2 * e);
        }
    }
    return sqrtf(mean);
}

// Raising one maximum from every row.  Atomics on one address take turns, and the rows that run first all find the value they start from: with an
// atomic from each row that finds its own the larger, 1000 rows of 4096 took 15.8 us, 7.8 with a scale a row; 8192 (fp32) 94 and 78, 32768 x 1024 86 and 51.  So one
// row in 128 raises it as soon as it knows its own; the others look again behind their stores and a microsecond and a half: 10.8, 84 and 61 us.
// Up to 128 rows have an atomic each at once: with the amax's clearing 16 rows 5.6 us, 7.4 the other way; 128 6.9 and 8.1.
__device__ __forceinline__ bool raises_at_once(unsigned row, int rows) { return rows <= 128 || row % 128 == 0; }
__device__ __forceinline__ void raise_first(float* amax, uint32_t m, unsigned row, int rows, float& before) {
    before = atomic_load_agent(amax);
    if (raises_at_once(row, rows) && __uint_as_float(m) > before) atomicMax(reinterpret_cast<int*>(amax), static_cast<int>(m));
}
// Before it comes back to memory it looks at the copy in its own L2: brought there by the first who looked behind the pause, a value that the maximum has had and so a bound that most are
// under, for which nobody waits in turn (8192 x 4096 70.1 -> 66.0 us, 16384 x 2048 75.4 -> 70.5).
__device__ __forceinline__ bool above_l2_copy(const float* amax, uint32_t m) {
    return __uint_as_float(m) > __hip_atomic_load(amax, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}
__device__ __forceinline__ void raise_last(float* amax, uint32_t m, unsigned row, int rows, float before) {
    if (raises_at_once(row, rows) || __uint_as_float(m) <= before) return;
    __builtin_amdgcn_s_sleep(48);           // 48 x 64 cycles
    if (!above_l2_copy(amax, m)) return;
    if (__uint_as_float(m) > atomic_load_agent(amax)) atomicMax(reinterpret_cast<int*>(amax), static_cast<int>(m));
}

// 0: run, 1: nothing to do, < 0: error
inline int check_shape(int rows, int H) {
    if (rows < 0 || H < 0) return CF_ERR_INVALID_ARG;
    if (rows == 0 || H == 0) return 1;
    return H > kMaxH ? CF_ERR_UNSUPPORTED : 0;
}
inline bool misaligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

constexpr unsigned kLaunchRows = 1u << 21;             // a launch has fewer than 2^32 threads

}  // namespace cf
