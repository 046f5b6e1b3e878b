// Residual addition, RMS norm and the 8-bit output with its scales in one pass, and the gradient of it.
//
// Forward, per row:  h = T(r + x),  rms = sqrt(mean(h^2) + eps),  y = h / rms * w,  q = sat_rne(y * F / max|y| of the scale group).
// T is the type the residual stream is kept in (bf16 or fp32).  The norm reads h as it is stored: the backward pass, which has only
// h, then differentiates the function that was computed.  y stays in fp32 up to the 8-bit rounding, the only one it takes on that way.
//
// Backward, per row:  xh = h / rms,  g = dy * w,  c = mean(g * xh),  dr = dh + (g - xh * c) / rms;  over the rows:  dw = sum(dy * xh).
#include "common.hpp"

namespace cf {
namespace {

constexpr int kMaxH = 16384;
constexpr int kThreads = 256;

enum { Q_ROWS = 0, Q_BLOCK = 1, Q_RECORD = 2 };

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
    int H;
    float eps;
};

template <bool F32>
__device__ __forceinline__ float load_stream(const void* p, size_t i) {
    if constexpr (F32) return static_cast<const float*>(p)[i];
    else return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
}
template <bool F32>
__device__ __forceinline__ void store_stream(void* p, size_t i, float v) {
    if constexpr (F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
}

// sum (or maximum) over the workgroup of four wavefronts, the same in every thread
__device__ __forceinline__ float block_sum(float v, float* sh) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}
__device__ __forceinline__ float block_max(float v, float* sh) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
}

// One workgroup per row, the row in LDS as fp32.
template <bool F32, int QMODE, bool E5M2>
__global__ __launch_bounds__(kThreads) void k_add_norm(const AddNormArgs p) {
    extern __shared__ float ys[];
    __shared__ float sh[4];
    const int t = threadIdx.x, H = p.H;
    const size_t base = static_cast<size_t>(blockIdx.x) * H;
    float ss = 0.0f;
    for (int i = t; i < H; i += kThreads) {
        float h = load_stream<F32>(p.residual, base + i);
        if (p.x) {
            h += bf16_to_f32(p.x[base + i]);
            if constexpr (!F32) h = bf16_to_f32(f32_to_bf16(h));
        }
        if (p.sum) store_stream<F32>(p.sum, base + i, h);
        ys[i] = h;
        ss = __builtin_fmaf(h, h, ss);
    }
    const float rms = sqrtf(block_sum(ss, sh) / static_cast<float>(H) + p.eps);
    if (t == 0 && p.rms) p.rms[blockIdx.x] = rms;
    const float inv = 1.0f / rms;
    float amax = 0.0f;
    for (int i = t; i < H; i += kThreads) {
        const float y = ys[i] * inv * bf16_to_f32(p.weight[i]);
        ys[i] = y;
        amax = fmaxf(amax, fabsf(y));
        if (p.normed) p.normed[base + i] = f32_to_bf16(y);
    }
    constexpr float F = E5M2 ? 57344.0f : 448.0f;
    if constexpr (QMODE == Q_BLOCK) {
        __syncthreads();
        const int groups = (H + 127) / 128, wave = t >> 6, lane = t & 63;
        for (int g = wave; g < groups; g += kThreads / kWave) {
            const int i0 = g * 128 + lane, i1 = i0 + 64;
            const float a0 = i0 < H ? ys[i0] : 0.0f, a1 = i1 < H ? ys[i1] : 0.0f;
            const float a = fmaxf(wave_max(fmaxf(fabsf(a0), fabsf(a1))), 1e-12f), s = F / a;
            if (lane == 0) {
                p.scale[static_cast<size_t>(blockIdx.x) * groups + g] = s;
                p.descale[static_cast<size_t>(blockIdx.x) * groups + g] = a / F;
            }
            if (i0 < H) p.q[base + i0] = cvt1_fp8<E5M2>(a0 * s);
            if (i1 < H) p.q[base + i1] = cvt1_fp8<E5M2>(a1 * s);
        }
    } else {
        amax = block_max(amax, sh);
        float s;
        if constexpr (QMODE == Q_ROWS) {
            const float a = fmaxf(amax, 1e-12f);
            s = F / a;
            if (t == 0) { p.scale[blockIdx.x] = s; p.descale[blockIdx.x] = a / F; }
        } else {
            s = *p.qscale;
            if (t == 0) atomic_max_nonneg(p.amax, amax);
        }
        for (int i = t; i < H; i += kThreads) p.q[base + i] = cvt1_fp8<E5M2>(ys[i] * s);
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
    uint8_t* q;               // [rows, H] E5M2, or null
    const float* qscale;
    float* amax;
    int rows, H;
};

// Workgroup b takes rows b, b + parts, ... and leaves its share of dw, gathered in LDS, in partial[b].
template <bool F32>
__global__ __launch_bounds__(kThreads) void k_add_norm_grad(const AddNormGradArgs p) {
    extern __shared__ float dw[];
    __shared__ float sh[4];
    const int t = threadIdx.x, H = p.H;
    for (int i = t; i < H; i += kThreads) dw[i] = 0.0f;
    float amax = 0.0f;
    const float s = p.q ? *p.qscale : 0.0f;
    for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const size_t base = static_cast<size_t>(row) * H;
        const float inv = 1.0f / p.rms[row];
        float dot = 0.0f;
        for (int i = t; i < H; i += kThreads) {
            const float xh = load_stream<F32>(p.sum, base + i) * inv, dy = bf16_to_f32(p.dy[base + i]);
            dw[i] = __builtin_fmaf(dy, xh, dw[i]);
            dot = __builtin_fmaf(dy * bf16_to_f32(p.weight[i]), xh, dot);
        }
        const float c = block_sum(dot, sh) / static_cast<float>(H);
        for (int i = t; i < H; i += kThreads) {
            const float xh = load_stream<F32>(p.sum, base + i) * inv, g = bf16_to_f32(p.dy[base + i]) * bf16_to_f32(p.weight[i]);
            const float d = __builtin_fmaf(__builtin_fmaf(-xh, c, g), inv, p.dh ? load_stream<F32>(p.dh, base + i) : 0.0f);
            store_stream<F32>(p.dr, base + i, d);
            if (p.q) {
                p.q[base + i] = cvt1_fp8<true>(d * s);
                amax = fmaxf(amax, fabsf(d));
            }
        }
    }
    if (p.q) {
        amax = block_max(amax, sh);
        if (t == 0) atomic_max_nonneg(p.amax, amax);
    }
    for (int i = t; i < H; i += kThreads) p.partial[static_cast<size_t>(blockIdx.x) * H + i] = dw[i];
}

// dw[i] = (dw[i] +) the parts' shares, in their order
__global__ __launch_bounds__(kThreads) void k_sum_parts(const float* partial, float* dw, int H, int parts, int accumulate) {
    const int i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= H) return;
    float v = 0.0f;
    for (int b = 0; b < parts; ++b) v += partial[static_cast<size_t>(b) * H + i];
    dw[i] = accumulate ? dw[i] + v : v;
}

// 0: run, 1: nothing to do, < 0: error
int check_shape(int rows, int H) {
    if (rows < 0 || H < 0) return CF_ERR_INVALID_ARG;
    if (rows == 0 || H == 0) return 1;
    return H > kMaxH ? CF_ERR_UNSUPPORTED : 0;
}
bool misaligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

template <int QMODE>
int add_norm(const AddNormArgs& p, bool f32, bool e5m2, int rows, cf_stream_t stream) {
    hipStream_t st = as_stream(stream);
    auto go = [&](auto kernel) {
        kernel<<<rows, kThreads, static_cast<size_t>(p.H) * 4, st>>>(p);
        return launch_status();
    };
    if (f32) return e5m2 ? go(k_add_norm<true, QMODE, true>) : go(k_add_norm<true, QMODE, false>);
    return e5m2 ? go(k_add_norm<false, QMODE, true>) : go(k_add_norm<false, QMODE, false>);
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

int grad_parts(int rows) { return rows < 1024 ? rows : 1024; }

int add_norm_grad(AddNormGradArgs p, int f32, float* d_grad_scale, int accumulate, void* d_workspace, size_t workspace_bytes,
                  cf_stream_t stream) {
    if (p.H == 0) return CF_OK;
    if (!d_grad_scale || misaligned(d_grad_scale, 4)) return CF_ERR_INVALID_ARG;
    if (p.rows == 0) {              // no rows: their sum is zero
        if (accumulate) return CF_OK;
        k_sum_parts<<<ceil_div(p.H, kThreads), kThreads, 0, as_stream(stream)>>>(nullptr, d_grad_scale, p.H, 0, 0);
        return launch_status();
    }
    if (!p.dy || !p.sum || !p.weight || !p.rms || !p.dr || !d_workspace) return CF_ERR_INVALID_ARG;
    const unsigned el = f32 ? 4 : 2;
    if (misaligned(p.dy, 2) || misaligned(p.sum, el) || misaligned(p.weight, 2) || misaligned(p.rms, 4) || misaligned(p.dh, el) ||
        misaligned(p.dr, el) || misaligned(d_workspace, 16))
        return CF_ERR_INVALID_ARG;
    const int parts = grad_parts(p.rows);
    if (workspace_bytes < static_cast<size_t>(parts) * p.H * 4) return CF_ERR_INVALID_ARG;
    p.partial = static_cast<float*>(d_workspace);
    hipStream_t st = as_stream(stream);
    const size_t lds = static_cast<size_t>(p.H) * 4;
    if (f32) k_add_norm_grad<true><<<parts, kThreads, lds, st>>>(p);
    else k_add_norm_grad<false><<<parts, kThreads, lds, st>>>(p);
    k_sum_parts<<<ceil_div(p.H, kThreads), kThreads, 0, st>>>(p.partial, d_grad_scale, p.H, parts, accumulate);
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
    *bytes = static_cast<size_t>(grad_parts(rows)) * H * 4;
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
