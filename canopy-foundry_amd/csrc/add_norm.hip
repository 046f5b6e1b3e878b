// Residual addition, RMS norm and the 8-bit output with its scales in one pass, and the gradient of it.
//
// Forward, per row:  h = T(r + x),  rms = sqrt(mean(h^2) + eps),  y = h / rms * w,  q = sat_rne(y * F / max|y| of the scale group).
// T is the type the residual stream is kept in (bf16 or fp32).  The norm reads h as it is stored: the backward pass, which has only
// h, then differentiates the function that was computed.  y stays in fp32 up to the 8-bit rounding, the only one it takes on that way.
//
// Backward, per row:  xh = h / rms,  g = dy * w,  c = mean(g * xh),  dr = dh + (g - xh * c) / rms;  over the rows:  dw = sum(dy * xh).
#include "rows.hpp"

#include <type_traits>

namespace cf {
namespace {

struct AddNormArgs {
    const void* residual;     // [rows, H] bf16 or fp32
    const uint16_t* x;        // [rows, H] bf16 or null
    const uint16_t* weight;   // [H] bf16
    void* sum;                // [rows, H] like residual, or null
    uint16_t* normed;         // [rows, H] bf16 or null
    float* rms;               // [rows] or null
    uint8_t* q;               // [rows, H]
    float* scale;             // Q_ROWS: [rows]; Q_BLOCK: [rows, ceil(H / 128)]
    float* descale;
    const float* qscale;      // Q_RECORD
    float* amax;
    int rows, H;
    unsigned row0;            // the launch's first row
    float eps;
    int e5m2;
};

// A row is held in registers, V chunks of eight elements a thread, chunk c by thread c % T: one read and one write of everything.  Sixteen
// threads next to each other hold a scale group of 128.  TAIL: H is no multiple of 8, the last chunk is a part.
// What bounds it: HBM, and for few rows the chain load - sum - maximum - store.  Both want a row on as many threads as it has chunks.  Threads a row x
// chunks a thread, one row a workgroup (64: four rows), several sets of buffers in turn (one over and over, a part of which stays in the last-level cache:
// 8192 x 4096 36 us), us:
//     rows x H                        512 x 1   256 x 2   128 x 4    64 x 8   1024 x 1
//     1 x 4096, bf16                    3.4       3.8       5.0       7.0       3.6
//     512 x 4096                        4.6       4.8       6.2       8.7       5.4
//     8192 x 4096                      42.0      44.0      46.4      56.8      57.0
//     4000 x 7168, 1x128 scales           (512 x 2: 39.1)            100.0     38.4
//     8192 x 4096, fp32, bf16 rows     79.6      82.4      90.8     107.5      74.8
// So V = 1 up to H = 8192 and 2 beyond, with as many wavefronts as that takes; below 512 elements four rows share a workgroup.
// Maxima are taken of the bits of |y|: they order like the values, with NaN above infinity, so one maximum also says whether
// anything needs the slow conversion, which keeps NaN codes.
template <bool F32, int QMODE, bool TAIL, bool ONE_WAVE, int V>
__global__ __launch_bounds__(ONE_WAVE ? 256 : 1024) void k_add_norm(const AddNormArgs p) {
    __shared__ float sh_sum[2][16];
    __shared__ uint32_t sh_max[3][16];
    const int H = p.H, T = ONE_WAVE ? kWave : blockDim.x;
    unsigned row = p.row0 + blockIdx.x;
    int t = threadIdx.x;
    if constexpr (ONE_WAVE) {
        row = __builtin_amdgcn_readfirstlane(p.row0 + blockIdx.x * 4 + (threadIdx.x >> 6));
        t &= 63;
        if (row >= static_cast<unsigned>(p.rows)) return;
    }
    const int chunks = TAIL ? (H + 7) / 8 : H / 8;
    const size_t base = static_cast<size_t>(row) * H;
    auto left = [&](int j) { return TAIL ? H - (t + j * T) * 8 : 8; };      // elements from chunk j of this thread on
    auto has = [&](int j) { return t + j * T < chunks; };
    const bool follows = static_cast<size_t>(p.rows - 1 - row) * H >= 7;         // elements behind this row, as many as a last chunk lacks

    float h[V][8];
    u32x4_any w[V];
    {
        Raw8<F32> r[V];
        Raw8<false> x[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            clear8(r[j]);
            clear8(x[j]);
            w[j] = u32x4_any{0, 0, 0, 0};
            if (has(j)) {
                load8<F32, TAIL>(p.residual, base + (t + j * T) * 8, left(j), follows, r[j]);
                if (p.x) load8<false, TAIL>(p.x, base + (t + j * T) * 8, left(j), follows, x[j]);
                w[j] = load_weight<TAIL>(p.weight, (t + j * T) * 8, left(j), H);
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[j][i] = value8<F32, TAIL>(r[j], i, left(j));
                if (p.x) {
                    h[j][i] += value8<false, TAIL>(x[j], i, left(j));
                    if constexpr (!F32) h[j][i] = round_bf16_hw(h[j][i]);
                }
            }
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (p.sum && has(j)) store8_stream<F32, TAIL, true>(p.sum, base + (t + j * T) * 8, left(j), h[j]);
    int e;
    const float rms = row_rms<ONE_WAVE, V>(h, H, p.eps, sh_sum, sh_max[2], e);
    if (t == 0 && p.rms) p.rms[row] = ldexpf(rms, e);
    const float inv = 1.0f / rms;

    const float F = p.e5m2 ? 57344.0f : 448.0f;
    uint32_t top[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        top[j] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            h[j][i] = h[j][i] * inv * ((i & 1) ? bf16_hi(w[j][i >> 1]) : bf16_lo(w[j][i >> 1]));        // y from here on
            top[j] = max(top[j], abs_bits(h[j][i]));
        }
        if (p.normed && has(j)) store8_bf16<TAIL>(p.normed, base + (t + j * T) * 8, left(j), h[j]);
    }
    // the largest |y| of a chunk without its NaNs
    auto number = [&](int j) {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(h[j][i]));
        return __float_as_uint(m);
    };
    auto quantize = [&](int j, float s, bool finite) {
        if (!has(j)) return;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = h[j][i] * s;
        store8_fp8<TAIL>(p.q, base + (t + j * T) * 8, left(j), p.e5m2, finite, v);
    };
    if constexpr (QMODE == Q_BLOCK) {
        const int groups = (H + 127) >> 7;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            uint32_t m = max16(top[j]);
            const bool finite = __all(m < kInf);
            if (!finite) m = max16(number(j));
            const float a = fmaxf(__uint_as_float(m), 1e-12f), s = F / a;
            const int c = t + j * T;
            if ((c & 15) == 0 && has(j)) {
                p.scale[static_cast<size_t>(row) * groups + (c >> 4)] = s;
                p.descale[static_cast<size_t>(row) * groups + (c >> 4)] = a / F;
            }
            quantize(j, s, finite);
        }
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) m = max(m, top[j]);
        m = row_max<ONE_WAVE>(m, sh_max[0]);
        bool finite = m < kInf;
        if (!finite) {
            uint32_t n = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) n = max(n, number(j));
            m = row_max<ONE_WAVE>(n, sh_max[1]);
        }
        float s, before = 0.0f;
        if constexpr (QMODE == Q_ROWS) {
            const float a = fmaxf(__uint_as_float(m), 1e-12f);
            s = F / a;
            if (t == 0) { p.scale[row] = s; p.descale[row] = a / F; }
        } else {
            s = *p.qscale;
            if (t == 0) raise_first(p.amax, m, row, p.rows, before);
            finite = finite && abs_bits(s) < kInf;         // 0 times infinity
        }
#pragma unroll
        for (int j = 0; j < V; ++j) quantize(j, s, finite);
        if constexpr (QMODE == Q_RECORD) {
            if (t == 0) raise_last(p.amax, m, row, p.rows, before);
        }
    }
}

struct AddNormGradArgs {
    const uint16_t* dy;       // [rows, H] bf16: the gradient of y
    const void* sum;          // [rows, H] h as the forward pass stored it
    const uint16_t* weight;
    const float* rms;         // [rows]
    const void* dh;           // [rows, H] the residual stream's gradient, or null
    void* dr;                 // [rows, H]
    float* partial;           // [parts, H]
    float* part_amax;         // [parts]
    uint8_t* q;               // [rows, H] E5M2, or null
    const float* qscale;
    float* amax;
    int rows, H;
};

// Workgroup b takes rows b, b + parts, ... as k_add_norm holds one, loads the next row's operands before it works on one, and leaves its share of
// dw in partial[b].  ONE_WAVE: four rows at a time, one a wavefront, whose shares are added in LDS.
// dw is summed in 64 bits, in which thousands of rows lose nothing (in fp32 its error was three times that of a 64-bit sum), and each share is rounded to
// fp32 once on its way through memory: relative error 6.1e-8, 5.2e-8 and 5.9e-8 for 333 x 2048, 2000 x 7168 and 8192 x 4096, where the result's own rounding
// gives 5e-8 to 6e-8.  64-bit shares are twice the bytes: 333 x 2048 8.4 us instead of 7.2, 2000 x 7168 49.9 and 46.8, 8192 x 4096 58.1 and 56.3.
template <bool F32, bool QUANT, bool TAIL, bool ONE_WAVE, int V>
__global__ __launch_bounds__(ONE_WAVE ? 256 : 1024) void k_add_norm_grad(const AddNormGradArgs p) {
    __shared__ float sh[2][16];
    __shared__ double sh_dw[ONE_WAVE ? 4 : 1][ONE_WAVE ? 512 : 1];
    const int H = p.H, T = ONE_WAVE ? kWave : blockDim.x;
    const int t = ONE_WAVE ? threadIdx.x & 63 : threadIdx.x;
    const unsigned first = ONE_WAVE ? __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)) : blockIdx.x;
    const unsigned step = ONE_WAVE ? gridDim.x * 4 : gridDim.x, rows = p.rows;
    const int chunks = TAIL ? (H + 7) / 8 : H / 8;
    auto left = [&](int j) { return TAIL ? H - (t + j * T) * 8 : 8; };
    auto has = [&](int j) { return t + j * T < chunks; };

    struct Row {
        Raw8<false> dy[V];
        Raw8<F32> h[V], dh[V];
        float rms;
    };
    auto load = [&](Row& r, unsigned row) {
        const size_t base = static_cast<size_t>(row) * H;
        const bool follows = static_cast<size_t>(rows - 1 - row) * H >= 7;
        r.rms = p.rms[row];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            clear8(r.dy[j]);
            clear8(r.h[j]);
            clear8(r.dh[j]);
            if (has(j)) {
                load8<false, TAIL>(p.dy, base + (t + j * T) * 8, left(j), follows, r.dy[j]);
                load8<F32, TAIL>(p.sum, base + (t + j * T) * 8, left(j), follows, r.h[j]);
                if (p.dh) load8<F32, TAIL>(p.dh, base + (t + j * T) * 8, left(j), follows, r.dh[j]);
            }
        }
    };
    u32x4_any w[V];
    double dw[V][8];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        w[j] = u32x4_any{0, 0, 0, 0};
        if (has(j)) w[j] = load_weight<TAIL>(p.weight, (t + j * T) * 8, left(j), H);
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[j][i] = 0.0;
    }
    const float s = QUANT ? *p.qscale : 0.0f;
    const bool s_finite = abs_bits(s) < kInf;
    float amax = 0.0f;
    constexpr bool AHEAD = V == 1;          // 1024 threads have 128 registers each, too few for two rows of two chunks
    Row r, next;
    if (AHEAD && first < rows) load(next, first);
    int turn = 0;
    for (unsigned row = first; row < rows; row += step, turn ^= 1) {
        if constexpr (AHEAD) {
            r = next;
            if (row + step < rows) load(next, row + step);
        } else {
            load(r, row);
        }
        const size_t base = static_cast<size_t>(row) * H;
        const float inv = 1.0f / r.rms;
        auto dy_at = [&](int j, int i) { return value8<false, TAIL>(r.dy[j], i, left(j)); };
        auto xh_at = [&](int j, int i) { return value8<F32, TAIL>(r.h[j], i, left(j)) * inv; };
        auto g_at = [&](int j, int i) { return dy_at(j, i) * ((i & 1) ? bf16_hi(w[j][i >> 1]) : bf16_lo(w[j][i >> 1])); };
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dw[j][i] += static_cast<double>(dy_at(j, i) * xh_at(j, i));
                if constexpr (V > 1) asm volatile("" : "+v"(dw[j][i]));       // added here, not at the row's end, to which its terms would be kept
                dot = __builtin_fmaf(g_at(j, i), xh_at(j, i), dot);
            }
        const float c = row_sum<ONE_WAVE>(dot, sh[turn]) / static_cast<float>(H);
#pragma unroll
        for (int j = 0; j < V; ++j)
            if constexpr (V > 1) asm volatile("" : "+v"(w[j]));         // kept as pairs, not as fp32 from row to row
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float d[8];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                d[i] = __builtin_fmaf(__builtin_fmaf(-xh_at(j, i), c, g_at(j, i)), inv, value8<F32, TAIL>(r.dh[j], i, left(j)));
                if constexpr (QUANT) {
                    amax = fmaxf(amax, fabsf(d[i]));
                    top = max(top, abs_bits(d[i]));
                }
            }
            if (has(j)) store8_stream<F32, TAIL, false>(p.dr, base + (t + j * T) * 8, left(j), d);
            if constexpr (QUANT) {
                const bool finite = __all(top < kInf) && s_finite;
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] *= s;
                if (has(j)) store8_fp8<TAIL>(p.q, base + (t + j * T) * 8, left(j), true, finite, d);
            }
        }
    }
    float* part = p.partial + static_cast<size_t>(blockIdx.x) * H;
    if constexpr (ONE_WAVE) {
        static_assert(V == 1);
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int i = 0; i < 8; ++i) sh_dw[wave][t * 8 + i] = dw[0][i];
        __syncthreads();
        for (int i = threadIdx.x; i < H; i += 256) part[i] = static_cast<float>((sh_dw[0][i] + sh_dw[1][i]) + (sh_dw[2][i] + sh_dw[3][i]));
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (has(j)) {
                const int at = (t + j * T) * 8;
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(dw[j][i]);
                if (!TAIL || left(j) >= 8) {
                    reinterpret_cast<f32x4_any*>(part + at)[0] = f32x4_any{v[0], v[1], v[2], v[3]};
                    reinterpret_cast<f32x4_any*>(part + at)[1] = f32x4_any{v[4], v[5], v[6], v[7]};
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i < left(j)) part[at + i] = v[i];
                }
            }
    }
    if constexpr (QUANT) {
        __syncthreads();
        const uint32_t m = row_max<false>(__float_as_uint(amax), reinterpret_cast<uint32_t*>(sh[0]));
        if (threadIdx.x == 0) p.part_amax[blockIdx.x] = __uint_as_float(m);
    }
}

// dw[i] = (dw[i] +) the parts' shares, in 64 bits: 32 columns a workgroup, 32 threads to a column that take every 32nd part and are added in order.
// The workgroup behind them raises *amax to the parts' maxima.
constexpr int kSumColumns = 32, kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void k_sum_parts(const float* __restrict__ partial, float* __restrict__ dw, int H, int parts, int accumulate,
                                                           const float* __restrict__ part_amax, float* __restrict__ amax) {
    constexpr int kGroups = kSumThreads / kSumColumns;
    __shared__ double sh[kSumThreads];
    const int t = threadIdx.x;
    if (static_cast<int>(blockIdx.x) * kSumColumns >= H) {
        uint32_t m = 0;
        for (int b = t; b < parts; b += kSumThreads) m = max(m, __float_as_uint(part_amax[b]));
        m = row_max<false>(m, reinterpret_cast<uint32_t*>(sh));
        if (t == 0) atomic_max_nonneg(amax, __uint_as_float(m));
        return;
    }
    const int column = blockIdx.x * kSumColumns + t % kSumColumns, group = t / kSumColumns;
    double v = 0.0;
    if (column < H) {
#pragma unroll 8
        for (int b = group; b < parts; b += kGroups) v += partial[static_cast<size_t>(b) * H + column];
    }
    sh[t] = v;
    __syncthreads();
    if (group == 0 && column < H) {
        v = accumulate ? static_cast<double>(dw[column]) : 0.0;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) v += sh[g * kSumColumns + t];
        dw[column] = static_cast<float>(v);
    }
}

template <bool F32, int QMODE, bool TAIL>
int launch_add_norm(AddNormArgs p, hipStream_t st) {
    for (; p.row0 < static_cast<unsigned>(p.rows); p.row0 += kLaunchRows) {
        const unsigned left = static_cast<unsigned>(p.rows) - p.row0, n = left < kLaunchRows ? left : kLaunchRows;
        if (p.H <= kOneWaveH) k_add_norm<F32, QMODE, TAIL, true, 1><<<(n + 3) / 4, 4 * kWave, 0, st>>>(p);
        else if (p.H <= kOneChunkH) k_add_norm<F32, QMODE, TAIL, false, 1><<<n, row_threads(p.H, 1), 0, st>>>(p);
        else k_add_norm<F32, QMODE, TAIL, false, 2><<<n, row_threads(p.H, 2), 0, st>>>(p);
    }
    return launch_status();
}

template <int QMODE>
int add_norm(AddNormArgs p, bool f32, bool e5m2, int rows, cf_stream_t stream) {
    hipStream_t st = as_stream(stream);
    p.rows = rows;
    p.e5m2 = e5m2;
    if (p.H % 8 != 0) return f32 ? launch_add_norm<true, QMODE, true>(p, st) : launch_add_norm<false, QMODE, true>(p, st);
    return f32 ? launch_add_norm<true, QMODE, false>(p, st) : launch_add_norm<false, QMODE, false>(p, st);
}

// what the three forward entry points ask of the arguments they share
int check_forward(const void* d_residual, const uint16_t* d_x, int stream_is_f32, const uint16_t* d_scale, const void* d_sum,
                  const uint16_t* d_normed, const float* d_rms, const void* d_q) {
    if (!d_residual || !d_scale || !d_q) return CF_ERR_INVALID_ARG;
    const unsigned el = stream_is_f32 ? 4 : 2;
    if (misaligned(d_residual, el) || misaligned(d_sum, el) || misaligned(d_x, 2) || misaligned(d_scale, 2) || misaligned(d_normed, 2) ||
        misaligned(d_rms, 4))
        return CF_ERR_INVALID_ARG;
    return CF_OK;
}

AddNormArgs forward_args(const void* d_residual, const uint16_t* d_x, const uint16_t* d_scale, int H, float eps, void* d_sum,
                         uint16_t* d_normed, float* d_rms, void* d_q) {
    AddNormArgs p{};
    p.residual = d_residual; p.x = d_x; p.weight = d_scale; p.sum = d_sum; p.normed = d_normed; p.rms = d_rms;
    p.q = static_cast<uint8_t*>(d_q); p.H = H; p.eps = eps;
    return p;
}

// Workgroups of the backward pass, each with a share of dw that is written and read once more: eight wavefronts a CU, which keep HBM busy with
// the next row's operands on their way, and a workgroup on each of 256 CUs at least.  8192 x 4096 bf16, 8 wavefronts a workgroup: 256 57.9 us, 512 62.5, 1024 66.0;
// 32768 x 1024, 2 of them: 256 101, 512 67.6, 1024 58.0, 2048 66.5; 65536 x 512, 4 rows a workgroup: 256 70.4, 512 58.2, 1024 64.2.
// But four turns each, or the shares cost more than the rows: 1000 x 1000 with a workgroup a row 14.3, with 256 8.8.
int grad_parts(int rows, int H) {
    const int waves = H <= kOneWaveH ? 4 : row_threads(H, H <= kOneChunkH ? 1 : 2) / kWave;
    const int turns = H <= kOneWaveH ? (rows - 1) / 4 + 1 : rows;
    int parts = waves < 8 ? 2048 / waves : 256;
    parts = parts < turns / 4 ? parts : turns / 4;
    parts = parts > 256 ? parts : 256;
    return parts < turns ? parts : turns;
}
size_t grad_workspace(int rows, int H) { return static_cast<size_t>(grad_parts(rows, H)) * (static_cast<size_t>(H) + 1) * 4; }

template <bool F32, bool QUANT, bool TAIL>
void launch_grad(const AddNormGradArgs& p, int parts, hipStream_t st) {
    if (p.H <= kOneWaveH) k_add_norm_grad<F32, QUANT, TAIL, true, 1><<<parts, 4 * kWave, 0, st>>>(p);
    else if (p.H <= kOneChunkH) k_add_norm_grad<F32, QUANT, TAIL, false, 1><<<parts, row_threads(p.H, 1), 0, st>>>(p);
    else k_add_norm_grad<F32, QUANT, TAIL, false, 2><<<parts, row_threads(p.H, 2), 0, st>>>(p);
}

int add_norm_grad(AddNormGradArgs p, int f32, float* d_grad_scale, int accumulate, void* d_workspace, size_t workspace_bytes,
                  cf_stream_t stream) {
    if (p.H == 0) return CF_OK;
    if (!d_grad_scale || misaligned(d_grad_scale, 4)) return CF_ERR_INVALID_ARG;
    if (p.rows == 0) {              // no rows: their sum is zero
        if (accumulate) return CF_OK;
        k_sum_parts<<<ceil_div(p.H, kSumColumns), kSumThreads, 0, as_stream(stream)>>>(nullptr, d_grad_scale, p.H, 0, 0, nullptr, nullptr);
        return launch_status();
    }
    if (!p.dy || !p.sum || !p.weight || !p.rms || !p.dr || !d_workspace) return CF_ERR_INVALID_ARG;
    const unsigned el = f32 ? 4 : 2;
    if (misaligned(p.dy, 2) || misaligned(p.sum, el) || misaligned(p.weight, 2) || misaligned(p.rms, 4) || misaligned(p.dh, el) ||
        misaligned(p.dr, el) || misaligned(d_workspace, 16))
        return CF_ERR_INVALID_ARG;
    const int parts = grad_parts(p.rows, p.H);
    if (workspace_bytes < grad_workspace(p.rows, p.H)) return CF_ERR_INVALID_ARG;
    p.partial = static_cast<float*>(d_workspace);
    p.part_amax = p.partial + static_cast<size_t>(parts) * p.H;
    hipStream_t st = as_stream(stream);
    auto go = [&](auto stream_f32, auto quant) {
        constexpr bool F32 = decltype(stream_f32)::value, QUANT = decltype(quant)::value;
        if (p.H % 8 != 0) launch_grad<F32, QUANT, true>(p, parts, st);
        else launch_grad<F32, QUANT, false>(p, parts, st);
    };
    if (f32) p.q ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
    else p.q ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
    k_sum_parts<<<ceil_div(p.H, kSumColumns) + (p.q ? 1 : 0), kSumThreads, 0, st>>>(p.partial, d_grad_scale, p.H, parts, accumulate, p.part_amax, p.amax);
    return launch_status();
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" {

int cf_add_rmsnorm_quantize_rows(const void* d_residual, const uint16_t* d_x, int stream_is_f32, const uint16_t* d_scale, int rows,
                                 int H, float eps, int is_e5m2, void* d_sum, uint16_t* d_normed, float* d_rms, void* d_q,
                                 float* d_row_scale, float* d_row_descale, cf_stream_t stream) {
    const int chk = check_shape(rows, H);
    if (chk != 0) return chk < 0 ? chk : CF_OK;
    if (const int rc = check_forward(d_residual, d_x, stream_is_f32, d_scale, d_sum, d_normed, d_rms, d_q)) return rc;
    if (!d_row_scale || !d_row_descale || misaligned(d_row_scale, 4) || misaligned(d_row_descale, 4)) return CF_ERR_INVALID_ARG;
    AddNormArgs p = forward_args(d_residual, d_x, d_scale, H, eps, d_sum, d_normed, d_rms, d_q);
    p.scale = d_row_scale; p.descale = d_row_descale;
    return add_norm<Q_ROWS>(p, stream_is_f32 != 0, is_e5m2 != 0, rows, stream);
}

int cf_add_rmsnorm_quantize_block_1x128(const void* d_residual, const uint16_t* d_x, int stream_is_f32, const uint16_t* d_scale,
                                        int rows, int H, float eps, void* d_sum, uint16_t* d_normed, float* d_rms, void* d_q,
                                        float* d_group_scale, float* d_group_descale, cf_stream_t stream) {
    const int chk = check_shape(rows, H);
    if (chk != 0) return chk < 0 ? chk : CF_OK;
    if (const int rc = check_forward(d_residual, d_x, stream_is_f32, d_scale, d_sum, d_normed, d_rms, d_q)) return rc;
    if (!d_group_scale || !d_group_descale || misaligned(d_group_scale, 4) || misaligned(d_group_descale, 4)) return CF_ERR_INVALID_ARG;
    AddNormArgs p = forward_args(d_residual, d_x, d_scale, H, eps, d_sum, d_normed, d_rms, d_q);
    p.scale = d_group_scale; p.descale = d_group_descale;
    return add_norm<Q_BLOCK>(p, stream_is_f32 != 0, false, rows, stream);
}

int cf_add_rmsnorm_quantize_record(const void* d_residual, const uint16_t* d_x, int stream_is_f32, const uint16_t* d_scale, int rows,
                                   int H, float eps, int is_e5m2, void* d_sum, uint16_t* d_normed, float* d_rms, void* d_q,
                                   const float* d_qscale, float* d_amax, cf_stream_t stream) {
    const int chk = check_shape(rows, H);
    if (chk != 0) return chk < 0 ? chk : CF_OK;
    if (const int rc = check_forward(d_residual, d_x, stream_is_f32, d_scale, d_sum, d_normed, d_rms, d_q)) return rc;
    if (!d_qscale || !d_amax || misaligned(d_qscale, 4) || misaligned(d_amax, 4)) return CF_ERR_INVALID_ARG;
    AddNormArgs p = forward_args(d_residual, d_x, d_scale, H, eps, d_sum, d_normed, d_rms, d_q);
    p.qscale = d_qscale; p.amax = d_amax;
    return add_norm<Q_RECORD>(p, stream_is_f32 != 0, is_e5m2 != 0, rows, stream);
}

int cf_add_rmsnorm_backward_workspace_bytes(int rows, int H, size_t* bytes) {
    if (rows < 0 || H < 0 || !bytes) return CF_ERR_INVALID_ARG;
    if (H > kMaxH) return CF_ERR_UNSUPPORTED;
    *bytes = grad_workspace(rows, H);
    return CF_OK;
}

int cf_add_rmsnorm_backward(const uint16_t* d_grad_normed, const void* d_sum, int stream_is_f32, const uint16_t* d_scale,
                            const float* d_rms, const void* d_grad_sum, int rows, int H, void* d_grad_residual, float* d_grad_scale,
                            int accumulate, void* d_workspace, size_t workspace_bytes, cf_stream_t stream) {
    const int chk = check_shape(rows, H);
    if (chk < 0) return chk;
    AddNormGradArgs p{};
    p.dy = d_grad_normed; p.sum = d_sum; p.weight = d_scale; p.rms = d_rms; p.dh = d_grad_sum; p.dr = d_grad_residual; p.rows = rows; p.H = H;
    return add_norm_grad(p, stream_is_f32, d_grad_scale, accumulate, d_workspace, workspace_bytes, stream);
}

int cf_add_rmsnorm_backward_quant_e5m2(const uint16_t* d_grad_normed, const void* d_sum, int stream_is_f32, const uint16_t* d_scale,
                                       const float* d_rms, const void* d_grad_sum, int rows, int H, void* d_grad_residual,
                                       float* d_grad_scale, int accumulate, void* d_grad8, const float* d_qscale, float* d_amax,
                                       void* d_workspace, size_t workspace_bytes, cf_stream_t stream) {
    const int chk = check_shape(rows, H);
    if (chk < 0) return chk;
    AddNormGradArgs p{};
    p.dy = d_grad_normed; p.sum = d_sum; p.weight = d_scale; p.rms = d_rms; p.dh = d_grad_sum; p.dr = d_grad_residual; p.rows = rows; p.H = H;
    p.q = static_cast<uint8_t*>(d_grad8); p.qscale = d_qscale; p.amax = d_amax;
    if (rows > 0 && H > 0 && (!d_grad8 || !d_qscale || !d_amax || misaligned(d_qscale, 4) || misaligned(d_amax, 4))) return CF_ERR_INVALID_ARG;
    return add_norm_grad(p, stream_is_f32, d_grad_scale, accumulate, d_workspace, workspace_bytes, stream);
}

}  // extern "C"
