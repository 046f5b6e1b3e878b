// SwiGLU with the 8-bit operand of the product behind it and with gate and up kept in 8 bits, and its gradient from those bytes.
//
// Forward, per element:  a = g * s * u,  s = 1 / (1 + e^-g);  per 128 elements of a row:  e4m3(g * 448 / max|g|), e4m3(u * 448 / max|u|);  q = f8(a * scale).
// Backward, with g and u from their bytes:  dg = dO * u * s * (1 + g * (1 - s)),  du = dO * g * s.
#include "rows.hpp"

namespace cf {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRow = 32768;              // of the form that holds a whole row

// sigmoid(g).  The exponent g * log2(e) is carried in two terms, so that the result keeps its relative error of a few 2^-24 where g is far below zero (one term:
// |g| * 2^-24).  Below -87, where it is under 2^-125, it is taken as 0.
__device__ __forceinline__ float sigmoid(float g) {
    const float x = __builtin_amdgcn_fmed3f(g, -87.0f, 87.0f), t = x * -1.44269502f;        // log2(e) to 24 bits, and what that leaves
    const float rest = __builtin_fmaf(x, -1.92596299e-8f, __builtin_fmaf(x, -1.44269502f, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_fmaf(e, rest * 0.693147181f, e));
    return g < -87.0f ? 0.0f : s;
}

struct SwigluKeepArgs {
    const uint16_t *gate, *up;
    size_t ld;
    uint8_t *gate8, *up8, *q;       // [rows, I]
    float *gate_descale, *up_descale;
    float *scale, *descale;         // Q_ROWS: [rows]; Q_BLOCK: [rows, ceil(I / 128)]
    const float* qscale;            // Q_RECORD
    float* amax;
    int rows, I;
    unsigned row0, row_end;         // the launch's rows
    int e5m2;
};

// a last chunk's elements behind the row as zeros
template <bool TAIL>
__device__ __forceinline__ void cut(Raw8<false>& r, int n) {
    if constexpr (TAIL) {
#pragma unroll
        for (int k = 0; k < 4; ++k) r.v[0][k] &= 2 * k + 1 < n ? 0xffffffffu : 2 * k < n ? 0xffffu : 0u;
    }
}

// The maximum of |v| over the 16 lanes of a group, as bits and without NaNs; finite: there is neither an infinity nor a NaN.
__device__ __forceinline__ uint32_t group_max(const Raw8<false>& r, bool& finite) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) m = pk_absmax(m, r.v[0][k]);
    m = max16(max(m << 16, m & 0xffff0000u));
    finite = __all(m < kInf);
    if (!finite) {
        float f = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f = fmaxf(f, fabsf(r.at(i)));
        m = max16(__float_as_uint(f));
    }
    return m;
}
// A chunk of a checkpoint, and by its group's first lane the descale.
template <bool TAIL>
__device__ __forceinline__ void keep(const Raw8<false>& r, uint8_t* to, size_t at, int n, float* descale) {
    bool finite;
    const float a = fmaxf(__uint_as_float(group_max(r, finite)), 1e-12f), s = 448.0f / a;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = r.at(i) * s;
    if (n > 0) {
        store8_fp8<TAIL>(to, at, n, false, finite, v);
        if ((threadIdx.x & 15) == 0) *descale = a / 448.0f;
    }
}
__device__ __forceinline__ void activate(const Raw8<false>& g, const Raw8<false>& u, float (&a)[8], uint32_t& top) {
    top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = g.at(i);
        a[i] = v * sigmoid(v) * u.at(i);
        top = max(top, abs_bits(a[i]));
    }
}
__device__ __forceinline__ uint32_t number(const float (&a)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(a[i]));
    return __float_as_uint(m);
}
template <bool TAIL>
__device__ __forceinline__ void load_pair(const SwigluKeepArgs& p, unsigned row, int at, int n, Raw8<false>& g, Raw8<false>& u) {
    clear8(g);
    clear8(u);
    if (n > 0) {
        const size_t from = row * p.ld + at;
        const bool whole = static_cast<size_t>(static_cast<unsigned>(p.rows) - 1 - row) * p.ld + n >= 8;       // eight elements from here on in the tensor
        load8<false, TAIL>(p.gate, from, n, whole, g);
        load8<false, TAIL>(p.up, from, n, whole, u);
        cut<TAIL>(g, n);
        cut<TAIL>(u, n);
    }
}

// 16 lanes a group of 128 elements, workgroups that walk over all groups.
template <int QMODE, bool TAIL>
__global__ __launch_bounds__(kThreads) void k_swiglu_keep(const SwigluKeepArgs p) {
    __shared__ uint32_t sh[16];
    const unsigned groups = (static_cast<unsigned>(p.I) + 127) / 128, total = (p.row_end - p.row0) * groups;
    const int lane = threadIdx.x & 15;
    const float F = QMODE == Q_RECORD && p.e5m2 ? 57344.0f : 448.0f;
    const float qs = QMODE == Q_RECORD ? *p.qscale : 0.0f;
    uint32_t most = 0;
    for (unsigned i = blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4); i < total; i += gridDim.x * (kThreads / 16)) {
        const unsigned row = p.row0 + i / groups, group = i % groups;
        const int at = group * 128 + lane * 8, n = p.I - at;
        const size_t to = static_cast<size_t>(row) * p.I + at, slot = static_cast<size_t>(row) * groups + group;
        Raw8<false> g, u;
        load_pair<TAIL>(p, row, at, n, g, u);
        keep<TAIL>(g, p.gate8, to, n, p.gate_descale + slot);
        keep<TAIL>(u, p.up8, to, n, p.up_descale + slot);
        float a[8];
        uint32_t m;
        activate(g, u, a, m);
        float s = qs;
        bool finite;
        if constexpr (QMODE == Q_BLOCK) {
            m = max16(m);
            finite = __all(m < kInf);
            if (!finite) m = max16(number(a));
            const float top = fmaxf(__uint_as_float(m), 1e-12f);
            s = F / top;
            if (lane == 0) {
                p.scale[slot] = s;
                p.descale[slot] = top / F;
            }
        } else {
            finite = __all(m < kInf) && abs_bits(s) < kInf;
            most = max(most, m < kInf ? m : number(a));
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) a[k] *= s;
        if (n > 0) store8_fp8<TAIL>(p.q, to, n, QMODE == Q_RECORD && p.e5m2, finite, a);
    }
    if constexpr (QMODE == Q_RECORD) {
        most = row_max<false>(most, sh);
        if (threadIdx.x == 0) atomic_max_nonneg(p.amax, __uint_as_float(most));
    }
}

// A row in the registers of its threads, V chunks of eight elements each, for a scale that is the whole row's.
template <bool TAIL, bool ONE_WAVE, int V>
__global__ __launch_bounds__(ONE_WAVE ? 256 : 1024) void k_swiglu_keep_rows(const SwigluKeepArgs p) {
    __shared__ uint32_t sh[2][16];
    const int T = ONE_WAVE ? kWave : blockDim.x;
    unsigned row = p.row0 + blockIdx.x;
    int t = threadIdx.x;
    if constexpr (ONE_WAVE) {
        row = __builtin_amdgcn_readfirstlane(p.row0 + blockIdx.x * 4 + (threadIdx.x >> 6));
        t &= 63;
        if (row >= p.row_end) return;
    }
    const unsigned groups = (static_cast<unsigned>(p.I) + 127) / 128;
    const size_t base = static_cast<size_t>(row) * p.I;
    Raw8<false> g[V], u[V];
#pragma unroll
    for (int j = 0; j < V; ++j) load_pair<TAIL>(p, row, (t + j * T) * 8, p.I - (t + j * T) * 8, g[j], u[j]);
    float a[V][8];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = t + j * T, n = p.I - c * 8;
        const size_t slot = static_cast<size_t>(row) * groups + (c >> 4);
        keep<TAIL>(g[j], p.gate8, base + c * 8, n, p.gate_descale + slot);
        keep<TAIL>(u[j], p.up8, base + c * 8, n, p.up_descale + slot);
        uint32_t top;
        activate(g[j], u[j], a[j], top);
        m = max(m, top);
    }
    m = row_max<ONE_WAVE>(m, sh[0]);
    const bool finite = m < kInf;
    if (!finite) {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) top = max(top, number(a[j]));
        m = row_max<ONE_WAVE>(top, sh[1]);
    }
    const float F = p.e5m2 ? 57344.0f : 448.0f, most = fmaxf(__uint_as_float(m), 1e-12f), s = F / most;
    if (t == 0) {
        p.scale[row] = s;
        p.descale[row] = most / F;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int n = p.I - (t + j * T) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[j][i] *= s;
        if (n > 0) store8_fp8<TAIL>(p.q, base + (t + j * T) * 8, n, p.e5m2, finite, a[j]);
    }
}

struct SwigluGradArgs {
    const uint16_t* grad;           // [rows, I] bf16
    const uint8_t *gate8, *up8;     // [rows, I] E4M3
    const float *gate_descale, *up_descale;
    uint16_t *grad_gate, *grad_up;  // bf16, rows ld apart
    size_t ld;
    uint16_t* act;                  // [rows, I] bf16 or null
    uint8_t *grad8, *grad8_t;       // [rows, 2 I], [2 I, rows] E5M2
    uint8_t* act8_t;                // [I, rows] E4M3
    const float *qscale, *act_qscale;
    float* amax;
    int rows, I;
    unsigned row0, row_end;
};

// what eight elements give: dg, du and the activation
struct Grads8 {
    float dg[8], du[8], a[8];
};
template <bool TAIL>
__device__ __forceinline__ void grads8(const Raw8<false>& d, const u32x2_any& g8, const u32x2_any& u8, float gs, float us, int n, Grads8& o) {
    float g[8], u[8];
    unpack8_e4m3(g8, gs, g);
    unpack8_e4m3(u8, us, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float dv = value8<false, TAIL>(d, i, n), s = sigmoid(g[i]), silu = g[i] * s;
        o.dg[i] = dv * u[i] * (s * __builtin_fmaf(g[i], 1.0f - s, 1.0f));
        o.du[i] = dv * silu;
        o.a[i] = silu * u[i];
    }
}

// bf16 outputs: 16 lanes a group of 128 elements, as k_swiglu_keep.
template <bool TAIL>
__global__ __launch_bounds__(kThreads) void k_swiglu_grad(const SwigluGradArgs p) {
    const unsigned groups = (static_cast<unsigned>(p.I) + 127) / 128, total = (p.row_end - p.row0) * groups;
    for (unsigned i = blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4); i < total; i += gridDim.x * (kThreads / 16)) {
        const unsigned row = p.row0 + i / groups, group = i % groups;
        const int at = group * 128 + (threadIdx.x & 15) * 8, n = p.I - at;
        if (n <= 0) continue;
        const size_t from = static_cast<size_t>(row) * p.I + at, slot = static_cast<size_t>(row) * groups + group;
        const bool whole = static_cast<size_t>(static_cast<unsigned>(p.rows) - 1 - row) * p.I + n >= 8;
        Raw8<false> d;
        clear8(d);
        load8<false, TAIL>(p.grad, from, n, whole, d);
        const u32x2_any g8 = load8_bytes<TAIL>(p.gate8, from, n, whole), u8 = load8_bytes<TAIL>(p.up8, from, n, whole);
        Grads8 o;
        grads8<TAIL>(d, g8, u8, p.gate_descale[slot], p.up_descale[slot], n, o);
        store8_bf16<TAIL>(p.grad_gate, row * p.ld + at, n, o.dg);
        store8_bf16<TAIL>(p.grad_up, row * p.ld + at, n, o.du);
        if (p.act) store8_bf16<TAIL>(p.act, from, n, o.a);
    }
}

// rows r0..r3 hold bytes n0..n3; returns columns: c[j] = {r0.bj, r1.bj, r2.bj, r3.bj}
__device__ __forceinline__ void transpose4x4(uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3, uint32_t (&c)[4]) {
    const uint32_t t0 = __builtin_amdgcn_perm(r1, r0, 0x05010400u);
    const uint32_t t1 = __builtin_amdgcn_perm(r1, r0, 0x07030602u);
    const uint32_t u0 = __builtin_amdgcn_perm(r3, r2, 0x05010400u);
    const uint32_t u1 = __builtin_amdgcn_perm(r3, r2, 0x07030602u);
    c[0] = __builtin_amdgcn_perm(u0, t0, 0x05040100u);
    c[1] = __builtin_amdgcn_perm(u0, t0, 0x07060302u);
    c[2] = __builtin_amdgcn_perm(u1, t1, 0x05040100u);
    c[3] = __builtin_amdgcn_perm(u1, t1, 0x07060302u);
}

typedef uint32_t u32x4_byte __attribute__((ext_vector_type(4), aligned(1)));

// 8-bit outputs: a workgroup has 128 x 128 elements, a thread 8 x 8 of them, whose bytes it writes along the rows and, through LDS, along the columns.
constexpr int kTile = 128;
template <bool TAIL>
__global__ __launch_bounds__(kThreads) void k_swiglu_grad8(const SwigluGradArgs p) {
    __shared__ __attribute__((aligned(16))) uint8_t tile[kTile * kTile];      // [column][row]
    __shared__ uint32_t sh[16];
    const unsigned across = (static_cast<unsigned>(p.I) + kTile - 1) / kTile;
    const unsigned r0 = blockIdx.x / across * kTile;
    const int c0 = static_cast<int>(blockIdx.x % across) * kTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int at = c0 + tx * 8, n = p.I - at;
    const unsigned rows = p.rows;
    const float s = *p.qscale, as = p.act8_t ? *p.act_qscale : 0.0f;
    const bool s_finite = abs_bits(s) < kInf, as_finite = abs_bits(as) < kInf;
    u32x2_any bytes[3][8];
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned row = r0 + ty * 8 + i;
        bytes[0][i] = bytes[1][i] = bytes[2][i] = u32x2_any{0, 0};
        if (row >= rows || n <= 0) continue;
        const size_t from = static_cast<size_t>(row) * p.I + at, slot = static_cast<size_t>(row) * across + blockIdx.x % across;
        const bool whole = static_cast<size_t>(rows - 1 - row) * p.I + n >= 8;
        Raw8<false> d;
        clear8(d);
        load8<false, TAIL>(p.grad, from, n, whole, d);
        const u32x2_any g8 = load8_bytes<TAIL>(p.gate8, from, n, whole), u8 = load8_bytes<TAIL>(p.up8, from, n, whole);
        Grads8 o;
        grads8<TAIL>(d, g8, u8, p.gate_descale[slot], p.up_descale[slot], n, o);
        uint32_t top = 0, act_top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (!TAIL || k < n) most = fmaxf(most, fmaxf(fabsf(o.dg[k]), fabsf(o.du[k])));
            top = max(top, max(abs_bits(o.dg[k]), abs_bits(o.du[k])));
            act_top = max(act_top, abs_bits(o.a[k]));
        }
        const bool finite = __all(top < kInf) && s_finite, act_finite = __all(act_top < kInf) && as_finite;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            o.dg[k] *= s;
            o.du[k] *= s;
            o.a[k] *= as;
        }
        bytes[0][i] = pack8_fp8(true, finite, o.dg);
        bytes[1][i] = pack8_fp8(true, finite, o.du);
        bytes[2][i] = pack8_fp8(false, act_finite, o.a);
        store8_bytes<TAIL>(p.grad8, static_cast<size_t>(row) * 2 * p.I + at, n, bytes[0][i]);
        store8_bytes<TAIL>(p.grad8, static_cast<size_t>(row) * 2 * p.I + p.I + at, n, bytes[1][i]);
    }
#pragma unroll
    for (int part = 0; part < 3; ++part) {
        uint8_t* out = part == 2 ? p.act8_t : p.grad8_t ? p.grad8_t + (part == 1 ? static_cast<size_t>(p.I) * rows : 0) : nullptr;
        if (!out) continue;             // the same in every thread
        __syncthreads();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t lo[4], hi[4];
            transpose4x4(bytes[part][0][half], bytes[part][1][half], bytes[part][2][half], bytes[part][3][half], lo);
            transpose4x4(bytes[part][4][half], bytes[part][5][half], bytes[part][6][half], bytes[part][7][half], hi);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *reinterpret_cast<uint2*>(&tile[(tx * 8 + half * 4 + k) * kTile + ty * 8]) = make_uint2(lo[k], hi[k]);
        }
        __syncthreads();
        const int chunk = threadIdx.x & 7, rr = threadIdx.x >> 3;       // 8 lanes cover one 128-byte output row
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = i * 32 + rr;
            const unsigned row = r0 + chunk * 16;
            if (c0 + c >= p.I || row >= rows) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(&tile[c * kTile + chunk * 16]);
            uint8_t* to = out + static_cast<size_t>(c0 + c) * rows + row;
            if (!TAIL || row + 16 <= rows) {
                __builtin_nontemporal_store(u32x4_byte{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4_byte*>(to));
            } else {
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (row + k < rows) to[k] = static_cast<uint8_t>(w[k >> 2] >> (8 * (k & 3)));
            }
        }
    }
    __syncthreads();
    const uint32_t m = row_max<false>(__float_as_uint(most), sh);
    if (threadIdx.x == 0) atomic_max_nonneg(p.amax, __uint_as_float(m));
}

// the groups of a launch and, at 16 a workgroup, its workgroups: a few for each CU, which walk over the rest
constexpr unsigned kWalkers = 2048;
unsigned rows_of_launch(int I) { return (1u << 30) / (static_cast<unsigned>(I + 127) / 128); }
unsigned walkers(unsigned rows, int I) {
    const size_t groups = static_cast<size_t>(rows) * ((I + 127) / 128);
    const unsigned blocks = ceil_div(groups, kThreads / 16);
    return blocks < kWalkers ? blocks : kWalkers;
}

template <int QMODE, bool TAIL>
int launch_keep(SwigluKeepArgs p, hipStream_t st) {
    const unsigned rows = p.rows, most = QMODE == Q_ROWS ? kLaunchRows : rows_of_launch(p.I);
    for (p.row0 = 0; p.row0 < rows; p.row0 += most) {
        const unsigned n = rows - p.row0 < most ? rows - p.row0 : most;
        p.row_end = p.row0 + n;
        if constexpr (QMODE == Q_ROWS) {
            if (p.I <= kOneWaveH) k_swiglu_keep_rows<TAIL, true, 1><<<(n + 3) / 4, 4 * kWave, 0, st>>>(p);
            else if (p.I <= kOneChunkH) k_swiglu_keep_rows<TAIL, false, 1><<<n, row_threads(p.I, 1), 0, st>>>(p);
            else if (p.I <= 2 * kOneChunkH) k_swiglu_keep_rows<TAIL, false, 2><<<n, row_threads(p.I, 2), 0, st>>>(p);
            else k_swiglu_keep_rows<TAIL, false, 4><<<n, row_threads(p.I, 4), 0, st>>>(p);
        } else {
            k_swiglu_keep<QMODE, TAIL><<<walkers(n, p.I), kThreads, 0, st>>>(p);
        }
    }
    return launch_status();
}

// 0: run, 1: nothing to do, < 0: error
int check_rows(int rows, int I, int ld) {
    if (rows < 0 || I < 0 || ld < I) return CF_ERR_INVALID_ARG;
    if (I >= 1 << 30) return CF_ERR_UNSUPPORTED;
    return rows == 0 || I == 0 ? 1 : 0;
}

template <int QMODE>
int swiglu_keep(const uint16_t* d_gate, const uint16_t* d_up, int ld, int rows, int I, int is_e5m2, void* d_gate8, float* d_gate8_descale, void* d_up8,
                float* d_up8_descale, void* d_q, float* d_scale, float* d_descale, const float* d_qscale, float* d_amax, cf_stream_t stream) {
    const int chk = check_rows(rows, I, ld);
    if (chk != 0) return chk < 0 ? chk : CF_OK;
    if (QMODE == Q_ROWS && I > kMaxRow) return CF_ERR_UNSUPPORTED;
    if (!d_gate || !d_up || !d_gate8 || !d_gate8_descale || !d_up8 || !d_up8_descale || !d_q) return CF_ERR_INVALID_ARG;
    if (QMODE == Q_RECORD ? !d_qscale || !d_amax : !d_scale || !d_descale) return CF_ERR_INVALID_ARG;
    if (misaligned(d_gate, 2) || misaligned(d_up, 2) || misaligned(d_gate8_descale, 4) || misaligned(d_up8_descale, 4) || misaligned(d_scale, 4) ||
        misaligned(d_descale, 4) || misaligned(d_qscale, 4) || misaligned(d_amax, 4))
        return CF_ERR_INVALID_ARG;
    SwigluKeepArgs p{};
    p.gate = d_gate; p.up = d_up; p.ld = static_cast<size_t>(ld); p.rows = rows; p.I = I; p.e5m2 = is_e5m2 != 0;
    p.gate8 = static_cast<uint8_t*>(d_gate8); p.gate_descale = d_gate8_descale; p.up8 = static_cast<uint8_t*>(d_up8); p.up_descale = d_up8_descale;
    p.q = static_cast<uint8_t*>(d_q); p.scale = d_scale; p.descale = d_descale; p.qscale = d_qscale; p.amax = d_amax;
    hipStream_t st = as_stream(stream);
    return I % 8 != 0 ? launch_keep<QMODE, true>(p, st) : launch_keep<QMODE, false>(p, st);
}

// what both backward entry points ask of the arguments they share, the sizes checked
int check_backward(const SwigluGradArgs& p) {
    if (!p.grad || !p.gate8 || !p.up8 || !p.gate_descale || !p.up_descale) return CF_ERR_INVALID_ARG;
    if (misaligned(p.grad, 2) || misaligned(p.gate_descale, 4) || misaligned(p.up_descale, 4)) return CF_ERR_INVALID_ARG;
    return CF_OK;
}
SwigluGradArgs backward_args(const uint16_t* d_grad_out, const void* d_gate8, const float* d_gate8_descale, const void* d_up8, const float* d_up8_descale,
                             int rows, int I) {
    SwigluGradArgs p{};
    p.grad = d_grad_out; p.gate8 = static_cast<const uint8_t*>(d_gate8); p.up8 = static_cast<const uint8_t*>(d_up8); p.gate_descale = d_gate8_descale;
    p.up_descale = d_up8_descale; p.rows = rows; p.I = I;
    return p;
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" {

int cf_swiglu_ckpt8_quantize_rows(const uint16_t* d_gate, const uint16_t* d_up, int ld, int rows, int I, int is_e5m2, void* d_gate8,
                                  float* d_gate8_descale, void* d_up8, float* d_up8_descale, void* d_q, float* d_row_scale, float* d_row_descale,
                                  cf_stream_t stream) {
    return swiglu_keep<Q_ROWS>(d_gate, d_up, ld, rows, I, is_e5m2, d_gate8, d_gate8_descale, d_up8, d_up8_descale, d_q, d_row_scale, d_row_descale,
                               nullptr, nullptr, stream);
}

int cf_swiglu_ckpt8_quantize_block_1x128(const uint16_t* d_gate, const uint16_t* d_up, int ld, int rows, int I, void* d_gate8,
                                         float* d_gate8_descale, void* d_up8, float* d_up8_descale, void* d_q, float* d_group_scale,
                                         float* d_group_descale, cf_stream_t stream) {
    return swiglu_keep<Q_BLOCK>(d_gate, d_up, ld, rows, I, 0, d_gate8, d_gate8_descale, d_up8, d_up8_descale, d_q, d_group_scale, d_group_descale,
                                nullptr, nullptr, stream);
}

int cf_swiglu_ckpt8_quantize_record(const uint16_t* d_gate, const uint16_t* d_up, int ld, int rows, int I, int is_e5m2, void* d_gate8,
                                    float* d_gate8_descale, void* d_up8, float* d_up8_descale, void* d_q, const float* d_qscale, float* d_amax,
                                    cf_stream_t stream) {
    return swiglu_keep<Q_RECORD>(d_gate, d_up, ld, rows, I, is_e5m2, d_gate8, d_gate8_descale, d_up8, d_up8_descale, d_q, nullptr, nullptr, d_qscale,
                                 d_amax, stream);
}

int cf_swiglu_ckpt8_backward(const uint16_t* d_grad_out, const void* d_gate8, const float* d_gate8_descale, const void* d_up8,
                             const float* d_up8_descale, int rows, int I, uint16_t* d_grad_gate, uint16_t* d_grad_up, int ld, uint16_t* d_act,
                             cf_stream_t stream) {
    const int chk = check_rows(rows, I, ld);
    if (chk != 0) return chk < 0 ? chk : CF_OK;
    SwigluGradArgs p = backward_args(d_grad_out, d_gate8, d_gate8_descale, d_up8, d_up8_descale, rows, I);
    if (const int rc = check_backward(p)) return rc;
    if (!d_grad_gate || !d_grad_up || misaligned(d_grad_gate, 2) || misaligned(d_grad_up, 2) || misaligned(d_act, 2)) return CF_ERR_INVALID_ARG;
    p.grad_gate = d_grad_gate; p.grad_up = d_grad_up; p.ld = static_cast<size_t>(ld); p.act = d_act;
    hipStream_t st = as_stream(stream);
    const unsigned most = rows_of_launch(I), all = rows;
    for (p.row0 = 0; p.row0 < all; p.row0 += most) {
        const unsigned n = all - p.row0 < most ? all - p.row0 : most;
        p.row_end = p.row0 + n;
        if (I % 8 != 0) k_swiglu_grad<true><<<walkers(n, I), kThreads, 0, st>>>(p);
        else k_swiglu_grad<false><<<walkers(n, I), kThreads, 0, st>>>(p);
    }
    return launch_status();
}

int cf_swiglu_ckpt8_backward_quant_e5m2(const uint16_t* d_grad_out, const void* d_gate8, const float* d_gate8_descale, const void* d_up8,
                                        const float* d_up8_descale, int rows, int I, void* d_grad8, void* d_grad8_t, const float* d_qscale,
                                        float* d_amax, void* d_act8_t, const float* d_act_qscale, cf_stream_t stream) {
    const int chk = check_rows(rows, I, I);
    if (chk != 0) return chk < 0 ? chk : CF_OK;
    SwigluGradArgs p = backward_args(d_grad_out, d_gate8, d_gate8_descale, d_up8, d_up8_descale, rows, I);
    if (const int rc = check_backward(p)) return rc;
    if (!d_grad8 || !d_qscale || !d_amax || (d_act8_t && !d_act_qscale) || misaligned(d_qscale, 4) || misaligned(d_amax, 4) || misaligned(d_act_qscale, 4))
        return CF_ERR_INVALID_ARG;
    p.grad8 = static_cast<uint8_t*>(d_grad8); p.grad8_t = static_cast<uint8_t*>(d_grad8_t); p.act8_t = static_cast<uint8_t*>(d_act8_t);
    p.qscale = d_qscale; p.amax = d_amax; p.act_qscale = d_act_qscale;
    const size_t tiles = static_cast<size_t>(ceil_div(rows, kTile)) * ceil_div(I, kTile);
    if (tiles * kThreads >= (static_cast<size_t>(1) << 32)) return CF_ERR_UNSUPPORTED;         // a terabyte of gradients
    if (rows % 16 != 0 || I % 8 != 0) k_swiglu_grad8<true><<<static_cast<unsigned>(tiles), kThreads, 0, as_stream(stream)>>>(p);
    else k_swiglu_grad8<false><<<static_cast<unsigned>(tiles), kThreads, 0, as_stream(stream)>>>(p);
    return launch_status();
}

}  // extern "C"
