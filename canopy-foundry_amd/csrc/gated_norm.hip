// A block's output normed, gated and added to the scaled residual stream, then the next norm with its 8-bit output, in one pass; and its gradient.
//
// Forward, per row:  px = sqrt(mean(x^2) + eps),  xh = x / px,  h = T(res * r + gate * (xh * wp)),  p = sqrt(mean(h^2) + eps),  hh = h / p,
// y = hh * w,  q = sat_rne(y * F / max|y| of the scale group).  T is the type the residual stream is kept in; the second norm reads h as it is stored.
// Kept for the backward pass: px, p, and either the rows themselves or 8-bit checkpoints of the normalised rows, e4m3(xh * S) and e4m3(hh * S).  No element of
// a normalised row is above sqrt(H), so S is the largest power of two with S * sqrt(H) <= 448, the same for every row: no maximum to look for, no scale to keep.
//
// Backward, per row:  g = dy * w,  D = dh + (g - hh * mean(g * hh)) / p,  dr = T(res * D),  e = D * gate * wp,  dx = (e - xh * mean(e * xh)) / px;
// over the rows:  dw = sum(dy * hh);  over a gate's rows:  P = sum(D * xh),  dgate = wp * P;  over the gates:  dwp = sum(gate * P).
#include "gated_norm_plan.hpp"
#include "rows.hpp"

#include <cmath>
#include <type_traits>

namespace cf {
namespace {

struct GatedNormArgs {
    const void* residual;         // [rows, H] bf16 or fp32
    const uint16_t* x;            // [rows, H] bf16
    const uint16_t* gate;         // [ceil(rows / gate_rows), H] bf16 or null
    const uint16_t* post_weight;  // [H] bf16
    const uint16_t* weight;       // [H] bf16
    void* sum;                    // [rows, H] like residual, or null
    uint16_t* normed;             // [rows, H] bf16 or null
    float *post_rms, *rms;        // [rows] or null
    uint8_t *x8, *sum8;           // [rows, H] or null
    uint8_t* q;                   // [rows, H]
    float *scale, *descale;       // Q_ROWS: [rows]; Q_BLOCK: [rows, ceil(H / 128)]
    const float* qscale;          // Q_RECORD
    float* amax;
    int rows, H, gate_rows;
    unsigned row0;                // the launch's first row
    float eps, res, kept;
    int e5m2;
};

__device__ __forceinline__ float pair_at(const u32x4_any& v, int i) { return (i & 1) ? bf16_hi(v[i >> 1]) : bf16_lo(v[i >> 1]); }

// One row in registers, V chunks of eight elements a thread (forward_chunks() says how many), as k_add_norm holds it: everything is read and written once.  Bound by HBM, 9 or 13
// bytes an element with both checkpoints: 8192 x 4096 59 us on a bf16 stream (5.1 TB/s), 83 on an fp32 one (5.2), 1000 x 7168 13 to 14.5; a row alone takes 3.2, launch, load and two
// reductions.  Recording a maximum adds 6 us to 8192 rows (see raise_last()).  Odd widths move whole chunks that straddle lines: 8192 x 4095 75 us.
template <bool F32, int QMODE, bool TAIL, bool ONE_WAVE, int V>
__global__ __launch_bounds__(ONE_WAVE ? 256 : V == 4 ? 512 : 1024) void k_gated_norm(const GatedNormArgs p) {
    __shared__ double sh_post[2][16];
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
    Raw8<F32> r[V];
    u32x4_any w[V], wp[V], gate[V];
    const uint16_t* gates = p.gate ? p.gate + static_cast<size_t>(row / static_cast<unsigned>(p.gate_rows)) * H : nullptr;
    {
        Raw8<false> x[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            clear8(r[j]);
            clear8(x[j]);
            w[j] = wp[j] = gate[j] = u32x4_any{0, 0, 0, 0};
            if (has(j)) {
                const int at = (t + j * T) * 8;
                load8<false, TAIL>(p.x, base + at, left(j), follows, x[j]);
                load8<F32, TAIL>(p.residual, base + at, left(j), follows, r[j]);
                wp[j] = load_weight<TAIL>(p.post_weight, at, left(j), H);
                if (gates) gate[j] = load_weight<TAIL>(gates, at, left(j), H);
                w[j] = load_weight<TAIL>(p.weight, at, left(j), H);
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) h[j][i] = value8<false, TAIL>(x[j], i, left(j));
    }
    // the checkpoint of eight normalised values, none of which is above sqrt(H) but by roundings
    auto keep = [&](uint8_t* to, int j, float scale) {
        if (!to || !has(j)) return;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = h[j][i] * scale;
        store8_bytes<TAIL>(to, base + (t + j * T) * 8, left(j), convert8_fp8<false>(v));
    };

    // Each operation up to h is rounded to fp32 as it is written, the mean of the squares from a 64-bit sum, so that h has the bits that the formula
    // has in fp32: a bf16 stream takes the next value where h lies next to the border of two, and through the maximum of a group one such value can be all of a scale's
    // difference (some 160 of 7 million values lie there).  The squares in 64 bits cost nothing that shows: 8192 x 4096 58.8 us without, 59.2 with them, 1000 x 7168 14.3 and 13.5.  x / px is x times the inverse and a correction by what that leaves.
    int e;
    const float post_rms = row_rms<ONE_WAVE, V>(h, H, p.eps, sh_post, sh_max[1], e);
    if (t == 0 && p.post_rms) p.post_rms[row] = ldexpf(post_rms, e);
    const float post_inv = 1.0f / post_rms, divisor = post_rms < __builtin_inff() ? post_rms : 0.0f;         // infinite: 0 or NaN
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = h[j][i] * post_inv;
            h[j][i] = __builtin_fmaf(__builtin_fmaf(-q, divisor, h[j][i]), post_inv, q);
        }
        keep(p.x8, j, p.kept);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float z = h[j][i] * pair_at(wp[j], i);
            if (gates) z *= pair_at(gate[j], i);
            h[j][i] = p.res * value8<F32, TAIL>(r[j], i, left(j)) + z;
            if constexpr (!F32) h[j][i] = round_bf16_hw(h[j][i]);
        }
        if (p.sum && has(j)) store8_stream<F32, TAIL, !TAIL>(p.sum, base + (t + j * T) * 8, left(j), h[j]);
    }

    const float rms = row_rms<ONE_WAVE, V>(h, H, p.eps, sh_sum, sh_max[2], e);
    if (t == 0 && p.rms) p.rms[row] = ldexpf(rms, e);
    const float inv = 1.0f / rms;
    const float F = p.e5m2 ? 57344.0f : 448.0f;
    float top[V];           // a chunk's largest |y| without its NaNs
#pragma unroll
    for (int j = 0; j < V; ++j) {
        keep(p.sum8, j, inv * p.kept);
        top[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            h[j][i] = h[j][i] * inv * pair_at(w[j], i);        // y from here on
            top[j] = fmaxf(top[j], fabsf(h[j][i]));
        }
        if (p.normed && has(j)) store8_bf16<TAIL>(p.normed, base + (t + j * T) * 8, left(j), h[j]);
    }
    // what has been divided by its own maximum needs no clamp, and the conversion keeps NaNs
    auto quantize = [&](int j, float s) {
        if (!has(j)) return;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = h[j][i] * s;
        const size_t to = base + (t + j * T) * 8;
        if constexpr (QMODE == Q_RECORD) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
            store8_fp8<TAIL>(p.q, to, left(j), p.e5m2, __all(m <= kInf), v);
        } else {
            store8_bytes<TAIL>(p.q, to, left(j), p.e5m2 ? convert8_fp8<true>(v) : convert8_fp8<false>(v));
        }
    };
    if constexpr (QMODE == Q_BLOCK) {
        const int groups = (H + 127) >> 7;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float a = fmaxf(__uint_as_float(max16(__float_as_uint(top[j]))), 1e-12f), s = F / a;
            const int c = t + j * T;
            if ((c & 15) == 0 && has(j)) {
                p.scale[static_cast<size_t>(row) * groups + (c >> 4)] = s;
                p.descale[static_cast<size_t>(row) * groups + (c >> 4)] = a / F;
            }
            quantize(j, s);
        }
    } else {
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) m = fmaxf(m, top[j]);
        const uint32_t bits = row_max<ONE_WAVE>(__float_as_uint(m), sh_max[0]);
        float s, before = 0.0f;
        if constexpr (QMODE == Q_ROWS) {
            const float a = fmaxf(__uint_as_float(bits), 1e-12f);
            s = F / a;
            if (t == 0) { p.scale[row] = s; p.descale[row] = a / F; }
        } else {
            s = *p.qscale;
            if (t == 0) raise_first(p.amax, bits, row, p.rows, before);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) quantize(j, s);
        if constexpr (QMODE == Q_RECORD) {
            if (t == 0) raise_last(p.amax, bits, row, p.rows, before);
        }
    }
}

struct GatedGradArgs {
    const uint16_t* dy;           // [rows, H] bf16: the gradient of y
    const void *sum, *x;          // [rows, H] h and x, or hh and xh in 8 bits
    const uint16_t *gate, *post_weight, *weight;
    const float *post_rms, *rms;  // [rows]
    const void* dh;               // [rows, H] the residual stream's gradient, or null
    void* dr;                     // [rows, H]
    uint16_t* dx;                 // [rows, H] bf16 or null
    uint8_t* q;                   // [rows, H] E5M2 of dx, or null
    const float* qscale;
    float* amax;
    float* dgate;                 // GROUPS: [groups, H], written here for a group that one worker has whole
    int accumulate_gate;
    float* part_w;                // [parts, H] shares of dw
    float* part_p;                // [parts, H] shares of P (GROUPS: of dwp)
    float* part_amax;             // [parts]
    float* segments;              // GROUPS: [workers, 2, H] shares of P of the groups that several workers have
    double* far_dwp;              // GROUPS, H above 8192: [parts, 16, kT], where neither registers nor LDS have room for it
    int rows, H, gate_rows, groups, workers;
    unsigned share;
    float res, kept_inv;
};

// Eight elements of a saved row: as it was, or the normalised row in 8 bits.
template <bool F32, bool KEPT>
struct Saved8 {
    std::conditional_t<KEPT, u32x2_any, Raw8<F32>> v;
    // what follows is made of the elements as they were loaded, not of values kept from before
    __device__ __forceinline__ void hold() {
        if constexpr (KEPT) {
            asm volatile("" : "+v"(v));
        } else {
            asm volatile("" : "+v"(v.v[0]));
            if constexpr (F32) asm volatile("" : "+v"(v.v[F32 ? 1 : 0]));
        }
    }
    template <bool TAIL>
    __device__ __forceinline__ void load(const void* p, size_t at, int n, bool whole) {
        if constexpr (!KEPT) {
            clear8(v);
            if (n > 0) load8<F32, TAIL>(p, at, n, whole, v);
        } else {
            v = u32x2_any{0, 0};
            if (n > 0) v = load8_bytes<TAIL>(static_cast<const uint8_t*>(p), at, n, whole);
        }
    }
    // the normalised values; inv: 1 / rms, or of a checkpoint 1 / S
    template <bool TAIL>
    __device__ __forceinline__ void values(float (&o)[8], int n, float inv) const {
        if constexpr (!KEPT) {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = value8<F32, TAIL>(v, i, n) * inv;
        } else {
            unpack8_e4m3(v, inv, o);
            if constexpr (TAIL) {
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = i < n ? o[i] : 0.0f;
            }
        }
    }
};

// Which rows a worker has where groups of them share a gate, and in which order.  With many groups a worker takes every workers-th one.  Otherwise the rows are cut
// into equal shares, `share` rows each, without regard to the groups, so a group is a piece of one worker's share or of several that follow each other; the workers
// of a group take turns at its rows (the shares' rows as they lie: 8192 x 4096 83.8 us, 76.0 in turns, so much do neighbouring rows help HBM).
struct Walk {
    unsigned worker, workers, rows, gate_rows, groups, share;
    unsigned group, start, m, n, others, first_n, last_n, lead;
    unsigned whole;                     // the group is this worker's alone

    __device__ __forceinline__ bool begin() {
        if (whole_groups(groups, workers)) {
            group = worker;
        } else {
            if (static_cast<unsigned long long>(worker) * share >= rows) return false;
            group = worker * share / gate_rows;
        }
        return piece();
    }
    // the worker's piece of the group: n rows; of the group's other pieces the first has first_n rows, the last last_n, and the `others` between have `share`
    __device__ __forceinline__ bool piece() {
        if (group >= groups) return false;
        start = group * gate_rows;
        const unsigned end = gate_rows < rows - start ? start + gate_rows : rows;
        m = lead = others = last_n = 0;
        n = first_n = end - start;
        whole = 1;
        if (whole_groups(groups, workers)) return true;
        const unsigned k0 = start / share, k1 = (end - 1) / share, mine = worker * share;
        if (start >= mine + share) return false;
        if (k0 == k1) return true;
        whole = 0;
        first_n = (k0 + 1) * share - start;
        last_n = end - k1 * share;
        others = k1 - k0 - 1;
        lead = worker - k0;
        n = worker == k0 ? first_n : worker == k1 ? last_n : share;
        return true;
    }
    __device__ __forceinline__ unsigned row() const {
        const unsigned before = start + others * m + (m < first_n ? m : first_n) + (m < last_n ? m : last_n);
        return lead == 0 ? before : before + lead - 1 + (m < first_n ? 1 : 0);
    }
    __device__ __forceinline__ bool last_of_piece() const { return m + 1 == n; }
    __device__ __forceinline__ bool advance() {
        if (++m < n) return true;
        group += whole_groups(groups, workers) ? workers : 1;
        return piece();
    }
};

template <bool TAIL>
__device__ __forceinline__ void store8_f32(float* p, size_t at, int n, const float (&v)[8]) {
    float* q = p + at;
    if (!TAIL || n >= 8) {
        reinterpret_cast<f32x4_any*>(q)[0] = f32x4_any{v[0], v[1], v[2], v[3]};
        reinterpret_cast<f32x4_any*>(q)[1] = f32x4_any{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) q[i] = v[i];
    }
}

// A worker (a workgroup; ONE_WAVE: a wavefront) holds a row as k_gated_norm does and loads the next row's operands before it works on one.  Its shares of
// the sums over rows are kept in 64 bits and rounded to fp32 once on their way through memory, as in k_add_norm_grad.  Without groups of rows
// workers take turns at the rows; GROUPS: as Walk has it, and at the end of a piece of a group P is left, dgate itself where the worker had the whole group.
// Bound by HBM: 8192 x 4096 from bf16 rows 73 us (5.5 TB/s), from checkpoints with the E5M2 bytes 54 (5.6), and 5 for k_gated_sum.  What it took: registers.  Two sums of
// 64 bits a column, two rows of five tensors and three weights for eight or sixteen columns a thread: with 1024 threads of 128 registers, 2000 x 7168 (fp32 stream,
// gates by sequence) took 159 us, with 512 of 256 94, and 64 with dw in LDS, a row ahead and Walk's order, for which 129 to 209 registers are enough.  Above H = 8192 there is room for
// few rows ahead, and spills cost the most: 2730 x 12288 87 us (4.6 TB/s), 2048 x 16384 98 (4.1).
template <bool F32, bool KEPT, bool GROUPS, bool TAIL, bool ONE_WAVE, int V, Width WIDTH>
__global__ __launch_bounds__((ONE_WAVE ? 256 : kGradThreads<GROUPS, WIDTH>)) void k_gated_norm_grad(const GatedGradArgs p) {
    constexpr int kT = kGradThreads<GROUPS, WIDTH>;
    constexpr bool FAR = GROUPS && WIDTH != USUAL;
    constexpr bool TIGHT = V > 1;       // of registers: dw in LDS, values made from the loaded elements as often as they are used
    __shared__ float sh[2][16];         // each is written again only behind the other one's barrier
    __shared__ double sh_sum[ONE_WAVE ? 4 : 1][ONE_WAVE ? 512 : 1];
    __shared__ double sh_dw[TIGHT ? V * 8 * kT : 1];
    __shared__ double sh_dwp[GROUPS && !ONE_WAVE && !FAR ? V * 8 * kT : 1];
    const int H = p.H, T = ONE_WAVE ? kWave : blockDim.x;
    const int t = ONE_WAVE ? threadIdx.x & 63 : threadIdx.x;
    const unsigned worker = ONE_WAVE ? __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)) : blockIdx.x;
    const unsigned rows = p.rows;
    const int chunks = TAIL ? (H + 7) / 8 : H / 8;
    auto left = [&](int j) { return TAIL ? H - (t + j * T) * 8 : 8; };
    auto has = [&](int j) { return t + j * T < chunks; };

    struct Row {
        Raw8<false> dy[V];
        Saved8<F32, KEPT> h[V];
        Saved8<false, KEPT> x[V];
        Raw8<F32> dh[V];
        float rms, post_rms;
    };
    auto load = [&](Row& r, unsigned row) {
        const size_t base = static_cast<size_t>(row) * H;
        const bool follows = static_cast<size_t>(rows - 1 - row) * H >= 7;
        r.rms = p.rms[row];
        r.post_rms = p.post_rms[row];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int at = (t + j * T) * 8, n = has(j) ? left(j) : 0;
            clear8(r.dy[j]);
            clear8(r.dh[j]);
            r.h[j].template load<TAIL>(p.sum, base + at, n, follows);
            r.x[j].template load<TAIL>(p.x, base + at, n, follows);
            if (n > 0) {
                load8<false, TAIL>(p.dy, base + at, n, follows, r.dy[j]);
                if (p.dh) load8<F32, TAIL>(p.dh, base + at, n, follows, r.dh[j]);
            }
        }
    };
    u32x4_any w[V], wp[V], gate[V];         // GROUPS: the gate is loaded where its rows begin
    float gw[TIGHT ? 1 : V][8];                  // gate * wp
    double dw[TIGHT ? 1 : V][8], ps[V][8], dwp[GROUPS && ONE_WAVE ? V : 1][8];
    // dwp, which changes at a group's end only; constant distances between a thread's sums, which need no registers
    double* far_dwp = p.far_dwp + static_cast<size_t>(blockIdx.x) * (V * 8 * kT);
    auto dwp_at = [&](int j, int i) -> double& {
        if constexpr (ONE_WAVE) return dwp[j][i];
        else if constexpr (FAR) return far_dwp[(j * 8 + i) * kT + t];
        else return sh_dwp[(j * 8 + i) * kT + t];
    };
#pragma unroll
    for (int j = 0; j < V; ++j) {
        w[j] = wp[j] = u32x4_any{0, 0, 0, 0};
        gate[j] = u32x4_any{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};           // 1
        if (has(j)) {
            w[j] = load_weight<TAIL>(p.weight, (t + j * T) * 8, left(j), H);
            wp[j] = load_weight<TAIL>(p.post_weight, (t + j * T) * 8, left(j), H);
            if constexpr (!GROUPS)
                if (p.gate) gate[j] = load_weight<TAIL>(p.gate, (t + j * T) * 8, left(j), H);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            ps[j][i] = 0.0;
            if constexpr (!TIGHT) gw[j][i] = pair_at(gate[j], i) * pair_at(wp[j], i);
            if constexpr (TIGHT) sh_dw[(j * 8 + i) * kT + t] = 0.0;
            else dw[j][i] = 0.0;
            if constexpr (GROUPS && !FAR) dwp_at(j, i) = 0.0;
        }
    }
    const float s = p.q ? *p.qscale : 0.0f;
    const bool s_finite = abs_bits(s) < kInf;
    float amax = 0.0f;
    constexpr bool AHEAD = WIDTH == USUAL || (WIDTH == WIDE && !F32 && !GROUPS);            // where the registers have room for a second row
    Row r, next;
    Walk walk{worker, static_cast<unsigned>(p.workers), rows, static_cast<unsigned>(p.gate_rows), static_cast<unsigned>(p.groups), p.share}, then;
    unsigned row = worker;
    bool more = row < rows;
    if constexpr (GROUPS) {
        more = worker < static_cast<unsigned>(p.workers) && walk.begin();
        if (more) row = walk.row();
    }
    unsigned pieces = 0;                    // of groups, behind the worker
    if (AHEAD && more) load(next, row);
    while (more) {
        unsigned row_then = row + p.workers;
        bool more_then = row_then < rows;
        if constexpr (GROUPS) {
            then = walk;
            more_then = then.advance();
            if (more_then) row_then = then.row();
        }
        if constexpr (AHEAD) r = next;
        if constexpr (GROUPS) {             // before the next row's loads, or they would be waited for with it
            if (walk.m == 0) {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (has(j)) gate[j] = load_weight<TAIL>(p.gate + static_cast<size_t>(walk.group) * H, (t + j * T) * 8, left(j), H);
            }
        }
        if constexpr (AHEAD) {
            if (more_then) load(next, row_then);
        } else {
            load(r, row);
        }
        const size_t base = static_cast<size_t>(row) * H;
        const float inv = 1.0f / r.rms, post_inv = 1.0f / r.post_rms;
        if constexpr (TIGHT) {
#pragma unroll
            for (int j = 0; j < V; ++j) asm volatile("" : "+v"(w[j]), "+v"(wp[j]), "+v"(gate[j]));        // kept as pairs, not as fp32 from row to row
        }
        const float hh_scale = KEPT ? p.kept_inv : inv, xh_scale = KEPT ? p.kept_inv : post_inv;
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float hh[8];
            r.h[j].template values<TAIL>(hh, left(j), hh_scale);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float dy = value8<false, TAIL>(r.dy[j], i, left(j));
                if constexpr (TIGHT) unsafeAtomicAdd(&sh_dw[(j * 8 + i) * kT + t], static_cast<double>(dy * hh[i]));
                else dw[j][i] += static_cast<double>(dy * hh[i]);
                dot = __builtin_fmaf(dy * pair_at(w[j], i), hh[i], dot);
            }
        }
        const float c = row_sum<ONE_WAVE>(dot, sh[0]) / static_cast<float>(H);
        dot = 0.0f;
        if constexpr (GROUPS && !TIGHT) {
            if (walk.m == 0) {
#pragma unroll
                for (int j = 0; j < V; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) gw[j][i] = pair_at(gate[j], i) * pair_at(wp[j], i);
            }
        }
        float e[V][8];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if constexpr (TIGHT) {
                r.h[j].hold();
                r.x[j].hold();
            }
            float hh[8], xh[8], o[8];
            r.h[j].template values<TAIL>(hh, left(j), hh_scale);
            r.x[j].template values<TAIL>(xh, left(j), xh_scale);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float g = value8<false, TAIL>(r.dy[j], i, left(j)) * pair_at(w[j], i);
                const float v = __builtin_fmaf(__builtin_fmaf(-hh[i], c, g), inv, value8<F32, TAIL>(r.dh[j], i, left(j)));
                o[i] = v * p.res;
                ps[j][i] += static_cast<double>(v * xh[i]);
                if constexpr (TIGHT) asm volatile("" : "+v"(ps[j][i]));         // added here, not at the row's end, to which its terms would be kept
                e[j][i] = v * (TIGHT ? pair_at(gate[j], i) * pair_at(wp[j], i) : gw[TIGHT ? 0 : j][i]);
                dot = __builtin_fmaf(e[j][i], xh[i], dot);
            }
            if (has(j)) store8_stream<F32, TAIL, false>(p.dr, base + (t + j * T) * 8, left(j), o);
        }
        const float post_c = row_sum<ONE_WAVE>(dot, sh[1]) / static_cast<float>(H);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if constexpr (TIGHT) r.x[j].hold();
            float xh[8], o[8];
            r.x[j].template values<TAIL>(xh, left(j), xh_scale);
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                o[i] = __builtin_fmaf(-xh[i], post_c, e[j][i]) * post_inv;
                amax = fmaxf(amax, fabsf(o[i]));
                top = max(top, abs_bits(o[i]));
            }
            if (p.dx && has(j)) store8_bf16<TAIL>(p.dx, base + (t + j * T) * 8, left(j), o);
            if (p.q) {
                const bool finite = __all(top < kInf) && s_finite;
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] *= s;
                if (has(j)) store8_fp8<TAIL>(p.q, base + (t + j * T) * 8, left(j), true, finite, o);
            }
        }
        if constexpr (GROUPS) {
            if (walk.last_of_piece()) {
                if constexpr (FAR) asm volatile("" : "+s"(far_dwp));          // its addresses are made here, not kept in registers from row to row
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float o[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const double term = ps[j][i] * static_cast<double>(pair_at(gate[j], i));
                        if constexpr (FAR) {                // the first piece finds nothing there, the last leaves the share
                            const double sum = pieces == 0 ? term : dwp_at(j, i) + term;
                            if (more_then) dwp_at(j, i) = sum;
                            o[i] = static_cast<float>(sum);
                        } else {
                            dwp_at(j, i) += term;
                        }
                    }
                    if constexpr (FAR)
                        if (!more_then && has(j)) store8_f32<TAIL>(p.part_p + static_cast<size_t>(worker) * H, (t + j * T) * 8, left(j), o);
                    if (has(j)) {
                        const int at = (t + j * T) * 8;
                        if (walk.whole) {
                            float* to = p.dgate + static_cast<size_t>(walk.group) * H;
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                double v = ps[j][i] * static_cast<double>(pair_at(wp[j], i));
                                if (p.accumulate_gate && i < left(j)) v += static_cast<double>(to[at + i]);
                                o[i] = static_cast<float>(v);
                            }
                            store8_f32<TAIL>(to, at, left(j), o);
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] = static_cast<float>(ps[j][i]);
                            store8_f32<TAIL>(p.segments + (static_cast<size_t>(worker) * 2 + (walk.lead == 0 ? 1 : 0)) * H, at, left(j), o);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) ps[j][i] = 0.0;
                }
                ++pieces;
            }
            walk = then;
        }
        row = row_then;
        more = more_then;
    }
    // the workgroup's shares
    auto leave = [&](auto at, float* to) {
        float* part = to + static_cast<size_t>(blockIdx.x) * H;
        if constexpr (ONE_WAVE) {
            static_assert(V == 1);
            const int wave = threadIdx.x >> 6;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) sh_sum[wave][t * 8 + i] = at(0, i);
            __syncthreads();
            for (int i = threadIdx.x; i < H; i += 256) part[i] = static_cast<float>((sh_sum[0][i] + sh_sum[1][i]) + (sh_sum[2][i] + sh_sum[3][i]));
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (has(j)) {
                    float o[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = static_cast<float>(at(j, i));
                    store8_f32<TAIL>(part, (t + j * T) * 8, left(j), o);
                }
        }
    };
    leave([&](int j, int i) {
        if constexpr (TIGHT) return sh_dw[(j * 8 + i) * kT + t];
        else return dw[j][i];
    }, p.part_w);
    if (!FAR || pieces == 0)
        leave([&](int j, int i) {
            if constexpr (FAR) return 0.0;
            else if constexpr (GROUPS) return dwp_at(j, i);
            else return ps[j][i];
        }, p.part_p);
    if (p.q) {
        __syncthreads();
        const uint32_t m = row_max<false>(__float_as_uint(amax), reinterpret_cast<uint32_t*>(sh[0]));
        if (threadIdx.x == 0) p.part_amax[blockIdx.x] = __uint_as_float(m);
    }
}

struct GatedSumArgs {
    const float *part_w, *part_p, *part_amax, *segments;
    const uint16_t *gate, *post_weight;
    float *dw, *dwp, *dgate, *amax;
    int rows, H, gate_rows, parts, accumulate, accumulate_gate;
    unsigned share;                 // rows a worker
    int groups;                     // 0 = no gate, 1 = one for all rows, which the shares of P do not hold yet
    int sum_blocks;                 // workgroups for each of the two weights; behind them amax's, if there is one, then the segments'
    int shares;                     // threads for a column of the segments
};

// The parts' shares added up in 64 bits, 32 columns a workgroup, 32 threads to a column that take every 32nd part: first dw's columns, then P's or dwp's; the
// workgroup behind them raises *amax to the parts' maxima.  The rest make dgate of the groups whose rows several workers had, from their segments in the order of the rows.
constexpr int kSumThreads = 1024, kSumColumns = 32, kSumShares = kSumThreads / kSumColumns;
struct Sum4 { double v[4]; };
__global__ __launch_bounds__(kSumThreads) void k_gated_sum(const GatedSumArgs p) {
    __shared__ Sum4 sh[kSumThreads];
    const int t = threadIdx.x;
    int block = blockIdx.x;
    if (block < 2 * p.sum_blocks) {
        const bool second = block >= p.sum_blocks;
        const float* part = second ? p.part_p : p.part_w;
        const int c = (block - (second ? p.sum_blocks : 0)) * kSumColumns + t % kSumColumns;
        double* one = &sh[0].v[0];
        double sum = 0.0;
        if (c < p.H) {
#pragma unroll 8
            for (int b = t / kSumColumns; b < p.parts; b += kSumShares) sum += part[static_cast<size_t>(b) * p.H + c];
        }
        one[t] = sum;
        __syncthreads();
        if (t < kSumColumns && c < p.H) {
            sum = 0.0;
#pragma unroll
            for (int g = 0; g < kSumShares; ++g) sum += one[g * kSumColumns + t];
            if (second && p.groups == 1) {
                const double d = sum * static_cast<double>(bf16_to_f32(p.post_weight[c]));
                p.dgate[c] = static_cast<float>(p.accumulate_gate ? static_cast<double>(p.dgate[c]) + d : d);
                sum *= static_cast<double>(bf16_to_f32(p.gate[c]));
            }
            float* to = second ? p.dwp : p.dw;
            to[c] = static_cast<float>(p.accumulate ? static_cast<double>(to[c]) + sum : sum);
        }
        return;
    }
    block -= 2 * p.sum_blocks;
    if (p.amax && block-- == 0) {
        uint32_t m = 0;
        for (int b = t; b < p.parts; b += kSumThreads) m = max(m, __float_as_uint(p.part_amax[b]));
        m = row_max<false>(m, reinterpret_cast<uint32_t*>(sh));
        if (t == 0) atomic_max_nonneg(p.amax, __uint_as_float(m));
        return;
    }
    const int quads = kSumThreads / p.shares, across = (p.H + 4 * quads - 1) / (4 * quads);
    const unsigned group = block / across, start = group * p.gate_rows, rows = p.rows;
    const unsigned end = p.gate_rows < static_cast<int>(rows - start) ? start + p.gate_rows : rows;
    const unsigned k0 = start / p.share, k1 = (end - 1) / p.share;
    if (k0 == k1) return;
    const int first = (block % across) * quads * 4, column = first + t % quads * 4;
    Sum4 v{};
    if (column < p.H) {
        const int n = p.H - column;
        for (unsigned k = k0 + t / quads; k <= k1; k += 4 * p.shares) {         // four loads on their way
            f32x4_any part[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const unsigned from = k + u * p.shares <= k1 ? k + u * p.shares : k;
                const float* at = p.segments + (static_cast<size_t>(from) * 2 + (from == k0 ? 1 : 0)) * p.H + column;
                if (n >= 4) part[u] = *reinterpret_cast<const f32x4_any*>(at);
                else part[u] = f32x4_any{at[0], n > 1 ? at[1] : 0.0f, n > 2 ? at[2] : 0.0f, 0.0f};
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (k + u * p.shares <= k1) v.v[i] += static_cast<double>(part[u][i]);
        }
    }
    sh[t] = v;
    __syncthreads();
    for (int c = t; c < quads * 4 && first + c < p.H; c += kSumThreads) {
        double sum = 0.0;
        for (int k = 0; k < p.shares; ++k) sum += sh[k * quads + c / 4].v[c % 4];
        sum *= static_cast<double>(bf16_to_f32(p.post_weight[first + c]));
        float* to = p.dgate + static_cast<size_t>(group) * p.H + first + c;
        *to = static_cast<float>(p.accumulate_gate ? static_cast<double>(*to) + sum : sum);
    }
}

float kept_scale(int H) {
    int e = 0;
    while (e < 8 && std::ldexp(1.0, 2 * (e + 1)) * H <= 448.0 * 448.0) ++e;
    return std::ldexp(1.0f, e);
}

// Chunks of a row that a thread has.  Two reductions follow each other here, which many rows hide best with some four workgroups a CU, whole rows behind each other's;
// a row alone wants as many threads as it can have.  1, 2, 4 chunks, us, rows of both checkpoints, 33.6 M elements (the first line: one row, by events over many calls):
//     1 row of 4096, bf16       3.7   4.4   5.8             H = 1024, f32     82.5  82.6  85.0
//     H = 1024, bf16           60.3  57.3  68.8             H = 4096, f32     82.9  83.9  89.3
//     H = 4096, bf16           61.4  58.5  61.0             H = 5120, f32     93.5  86.2  88.8
//     H = 5120, bf16           76.6  62.8  62.2             H = 7168, f32     93.1  87.3  89.3
//     H = 6144, bf16           73.8  65.1  60.6             H = 12288, f32      -   91.1 100.0
//     H = 7168, bf16           78.5  65.2  61.4             H = 16384, f32      -   91.5  94.0
//     H = 12288, bf16            -   63.7  74.2             H = 16384, bf16     -   70.9  63.3
//     H = 8200, bf16             -   72.2  78.0             H = 13312, bf16     -   75.6  65.0
//     H = 10240, bf16            -   66.3  69.6             H = 14336, bf16     -   77.4  64.0
// Four are ahead from somewhere between 12288 and 13312 on, the rule's border lies above that.
int forward_chunks(int rows, int H, bool f32) {
    if (rows <= 256 && H <= kOneChunkH) return 1;
    return !f32 && ((H >= 5120 && H <= kOneChunkH) || H > 14336) ? 4 : 2;
}

template <bool F32, int QMODE, bool TAIL>
int launch_gated_norm(GatedNormArgs p, hipStream_t st) {
    for (; p.row0 < static_cast<unsigned>(p.rows); p.row0 += kLaunchRows) {
        const unsigned left = static_cast<unsigned>(p.rows) - p.row0, n = left < kLaunchRows ? left : kLaunchRows;
        const int V = forward_chunks(p.rows, p.H, F32);
        if (p.H <= kOneWaveH) k_gated_norm<F32, QMODE, TAIL, true, 1><<<(n + 3) / 4, 4 * kWave, 0, st>>>(p);
        else if (V == 1) k_gated_norm<F32, QMODE, TAIL, false, 1><<<n, row_threads(p.H, 1), 0, st>>>(p);
        else if (F32 || V == 2) k_gated_norm<F32, QMODE, TAIL, false, 2><<<n, row_threads(p.H, 2), 0, st>>>(p);
        else if constexpr (!F32) k_gated_norm<F32, QMODE, TAIL, false, 4><<<n, row_threads(p.H, 4), 0, st>>>(p);
    }
    return launch_status();
}

template <int QMODE>
int gated_norm(const GatedNormArgs& p, bool f32, cf_stream_t stream) {
    hipStream_t st = as_stream(stream);
    if (p.H % 8 != 0) return f32 ? launch_gated_norm<true, QMODE, true>(p, st) : launch_gated_norm<false, QMODE, true>(p, st);
    return f32 ? launch_gated_norm<true, QMODE, false>(p, st) : launch_gated_norm<false, QMODE, false>(p, st);
}

// what the three forward entry points ask of the arguments they share
int check_forward(const GatedNormArgs& p, int stream_is_f32) {
    if (!p.residual || !p.x || !p.post_weight || !p.weight || !p.q || (p.gate && p.gate_rows <= 0) || !std::isfinite(p.res)) return CF_ERR_INVALID_ARG;
    const unsigned el = stream_is_f32 ? 4 : 2;
    if (misaligned(p.residual, el) || misaligned(p.sum, el) || misaligned(p.x, 2) || misaligned(p.gate, 2) || misaligned(p.post_weight, 2) ||
        misaligned(p.weight, 2) || misaligned(p.normed, 2) || misaligned(p.post_rms, 4) || misaligned(p.rms, 4))
        return CF_ERR_INVALID_ARG;
    return CF_OK;
}

GatedNormArgs forward_args(const void* d_residual, const uint16_t* d_x, float residual_scale, const uint16_t* d_gate, int rows_per_gate,
                           const uint16_t* d_post_scale, const uint16_t* d_scale, int rows, int H, float eps, void* d_sum, uint16_t* d_normed,
                           float* d_post_rms, float* d_rms, void* d_x8, void* d_sum8, void* d_q) {
    GatedNormArgs p{};
    p.residual = d_residual; p.x = d_x; p.res = residual_scale; p.gate = d_gate; p.gate_rows = rows_per_gate; p.post_weight = d_post_scale;
    p.weight = d_scale; p.rows = rows; p.H = H; p.eps = eps; p.sum = d_sum; p.normed = d_normed; p.post_rms = d_post_rms; p.rms = d_rms;
    p.x8 = static_cast<uint8_t*>(d_x8); p.sum8 = static_cast<uint8_t*>(d_sum8); p.q = static_cast<uint8_t*>(d_q);
    p.kept = kept_scale(H);
    return p;
}

template <bool GROUPS>
constexpr int kWidestChunks = GROUPS ? 2 : 4;
template <bool F32, bool KEPT, bool GROUPS, bool TAIL>
void launch_gated_grad(const GatedGradArgs& p, int parts, hipStream_t st) {
    if (p.H <= kOneWaveH) k_gated_norm_grad<F32, KEPT, GROUPS, TAIL, true, 1, USUAL><<<parts, 4 * kWave, 0, st>>>(p);
    else if (p.H <= kTallH) k_gated_norm_grad<F32, KEPT, GROUPS, TAIL, false, 1, USUAL><<<parts, row_threads(p.H, 1), 0, st>>>(p);
    else if (p.H <= kUsualH) k_gated_norm_grad<F32, KEPT, GROUPS, TAIL, false, 2, USUAL><<<parts, row_threads(p.H, 2), 0, st>>>(p);
    else if (p.H <= kWideH) k_gated_norm_grad<F32, KEPT, GROUPS, TAIL, false, 2, WIDE><<<parts, row_threads(p.H, 2), 0, st>>>(p);
    else k_gated_norm_grad<F32, KEPT, GROUPS, TAIL, false, kWidestChunks<GROUPS>, WIDEST><<<parts, row_threads(p.H, kWidestChunks<GROUPS>), 0, st>>>(p);
}

int gated_grad(GatedGradArgs p, bool kept, int f32, float* d_grad_post_scale, float* d_grad_scale, int accumulate, void* d_workspace,
               size_t workspace_bytes, cf_stream_t stream) {
    const int chk = check_shape(p.rows, p.H);
    if (chk < 0) return chk;
    if ((p.gate && p.gate_rows <= 0) || !std::isfinite(p.res) || (accumulate & ~(CF_ACCUMULATE_SCALES | CF_ACCUMULATE_GATE))) return CF_ERR_INVALID_ARG;
    if (p.H == 0) return CF_OK;
    if (!d_grad_post_scale || !d_grad_scale || misaligned(d_grad_post_scale, 4) || misaligned(d_grad_scale, 4)) return CF_ERR_INVALID_ARG;
    GatedSumArgs s{};
    s.dw = d_grad_scale; s.dwp = d_grad_post_scale; s.H = p.H; s.accumulate = accumulate & CF_ACCUMULATE_SCALES;
    s.sum_blocks = static_cast<int>(ceil_div(p.H, kSumColumns));
    if (p.rows == 0) {              // no rows: their sums are zero, and there is no gate
        if (s.accumulate) return CF_OK;
        k_gated_sum<<<2 * s.sum_blocks, kSumThreads, 0, as_stream(stream)>>>(s);
        return launch_status();
    }
    if (!p.dy || !p.sum || !p.x || !p.post_weight || !p.weight || !p.post_rms || !p.rms || !p.dr || (!p.dx && !p.q) || !d_workspace ||
        (p.q && (!p.qscale || !p.amax)) || (p.gate && !p.dgate))
        return CF_ERR_INVALID_ARG;
    const unsigned el = f32 ? 4 : 2;
    if (misaligned(p.dy, 2) || (!kept && (misaligned(p.sum, el) || misaligned(p.x, 2))) || misaligned(p.gate, 2) || misaligned(p.post_weight, 2) ||
        misaligned(p.weight, 2) || misaligned(p.post_rms, 4) || misaligned(p.rms, 4) || misaligned(p.dh, el) || misaligned(p.dr, el) ||
        misaligned(p.dx, 2) || misaligned(p.dgate, 4) || misaligned(p.qscale, 4) || misaligned(p.amax, 4) || misaligned(d_workspace, 16))
        return CF_ERR_INVALID_ARG;
    const GradPlan plan = grad_plan(p.rows, p.H, p.gate ? p.gate_rows : 0);
    if (workspace_bytes < plan.bytes) return CF_ERR_INVALID_ARG;
    const size_t share = static_cast<size_t>(plan.parts) * p.H;
    p.far_dwp = static_cast<double*>(d_workspace);
    p.part_w = reinterpret_cast<float*>(static_cast<char*>(d_workspace) + plan.far);
    p.part_p = p.part_w + share;
    p.segments = p.part_p + share;
    p.part_amax = p.segments + (plan.segments ? 2 * static_cast<size_t>(plan.workers) * p.H : 0);
    p.groups = plan.groups;
    p.workers = plan.workers;
    p.share = plan.share;
    p.accumulate_gate = accumulate & CF_ACCUMULATE_GATE;
    p.kept_inv = 1.0f / kept_scale(p.H);
    hipStream_t st = as_stream(stream);
    auto go = [&](auto stream_f32, auto in_8_bits, auto groups) {
        constexpr bool F32 = decltype(stream_f32)::value, KEPT = decltype(in_8_bits)::value, GROUPS = decltype(groups)::value;
        if (p.H % 8 != 0) launch_gated_grad<F32, KEPT, GROUPS, true>(p, plan.parts, st);
        else launch_gated_grad<F32, KEPT, GROUPS, false>(p, plan.parts, st);
    };
    const std::true_type yes{};
    const std::false_type no{};
    auto by_groups = [&](auto a, auto b) { plan.several ? go(a, b, yes) : go(a, b, no); };
    if (f32) kept ? by_groups(yes, yes) : by_groups(yes, no);
    else kept ? by_groups(no, yes) : by_groups(no, no);
    s.part_w = p.part_w; s.part_p = p.part_p; s.part_amax = p.part_amax; s.segments = p.segments; s.gate = p.gate; s.post_weight = p.post_weight;
    s.dgate = p.dgate; s.amax = p.q ? p.amax : nullptr; s.rows = p.rows; s.gate_rows = p.gate_rows; s.parts = plan.parts; s.share = plan.share;
    s.groups = plan.several ? 0 : plan.groups; s.accumulate_gate = p.accumulate_gate;
    s.shares = plan.shares;
    const unsigned segment_blocks = plan.segments ? static_cast<unsigned>(plan.groups) * ceil_div(p.H, 4 * kSumThreads / s.shares) : 0;
    k_gated_sum<<<2 * s.sum_blocks + (s.amax ? 1 : 0) + segment_blocks, kSumThreads, 0, st>>>(s);
    return launch_status();
}

GatedGradArgs grad_args(const uint16_t* d_grad_normed, const void* d_sum, const void* d_x, float residual_scale, const uint16_t* d_gate,
                        int rows_per_gate, const uint16_t* d_post_scale, const uint16_t* d_scale, const float* d_post_rms, const float* d_rms,
                        const void* d_grad_sum, int rows, int H, void* d_grad_residual, uint16_t* d_grad_x, void* d_grad8, const float* d_qscale,
                        float* d_amax, float* d_grad_gate) {
    GatedGradArgs p{};
    p.dy = d_grad_normed; p.sum = d_sum; p.x = d_x; p.res = residual_scale; p.gate = d_gate; p.gate_rows = rows_per_gate; p.post_weight = d_post_scale;
    p.weight = d_scale; p.post_rms = d_post_rms; p.rms = d_rms; p.dh = d_grad_sum; p.rows = rows; p.H = H; p.dr = d_grad_residual; p.dx = d_grad_x;
    p.q = static_cast<uint8_t*>(d_grad8); p.qscale = d_qscale; p.amax = d_amax; p.dgate = d_grad_gate;
    return p;
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" {

int cf_gated_add_rmsnorm_quantize_rows(const void* d_residual, const uint16_t* d_x, int stream_is_f32, float residual_scale, const uint16_t* d_gate,
                                       int rows_per_gate, const uint16_t* d_post_scale, const uint16_t* d_scale, int rows, int H, float eps,
                                       int is_e5m2, void* d_sum, uint16_t* d_normed, float* d_post_rms, float* d_rms, void* d_x8, void* d_sum8,
                                       void* d_q, float* d_row_scale, float* d_row_descale, cf_stream_t stream) {
    const int chk = check_shape(rows, H);
    if (chk != 0) return chk < 0 ? chk : CF_OK;
    GatedNormArgs p = forward_args(d_residual, d_x, residual_scale, d_gate, rows_per_gate, d_post_scale, d_scale, rows, H, eps, d_sum, d_normed,
                                   d_post_rms, d_rms, d_x8, d_sum8, d_q);
    if (const int rc = check_forward(p, stream_is_f32)) return rc;
    if (!d_row_scale || !d_row_descale || misaligned(d_row_scale, 4) || misaligned(d_row_descale, 4)) return CF_ERR_INVALID_ARG;
    p.scale = d_row_scale; p.descale = d_row_descale; p.e5m2 = is_e5m2 != 0;
    return gated_norm<Q_ROWS>(p, stream_is_f32 != 0, stream);
}

int cf_gated_add_rmsnorm_quantize_block_1x128(const void* d_residual, const uint16_t* d_x, int stream_is_f32, float residual_scale,
                                              const uint16_t* d_gate, int rows_per_gate, const uint16_t* d_post_scale, const uint16_t* d_scale,
                                              int rows, int H, float eps, void* d_sum, uint16_t* d_normed, float* d_post_rms, float* d_rms,
                                              void* d_x8, void* d_sum8, void* d_q, float* d_group_scale, float* d_group_descale, cf_stream_t stream) {
    const int chk = check_shape(rows, H);
    if (chk != 0) return chk < 0 ? chk : CF_OK;
    GatedNormArgs p = forward_args(d_residual, d_x, residual_scale, d_gate, rows_per_gate, d_post_scale, d_scale, rows, H, eps, d_sum, d_normed,
                                   d_post_rms, d_rms, d_x8, d_sum8, d_q);
    if (const int rc = check_forward(p, stream_is_f32)) return rc;
    if (!d_group_scale || !d_group_descale || misaligned(d_group_scale, 4) || misaligned(d_group_descale, 4)) return CF_ERR_INVALID_ARG;
    p.scale = d_group_scale; p.descale = d_group_descale;
    return gated_norm<Q_BLOCK>(p, stream_is_f32 != 0, stream);
}

int cf_gated_add_rmsnorm_quantize_record(const void* d_residual, const uint16_t* d_x, int stream_is_f32, float residual_scale, const uint16_t* d_gate,
                                         int rows_per_gate, const uint16_t* d_post_scale, const uint16_t* d_scale, int rows, int H, float eps,
                                         int is_e5m2, void* d_sum, uint16_t* d_normed, float* d_post_rms, float* d_rms, void* d_x8, void* d_sum8,
                                         void* d_q, const float* d_qscale, float* d_amax, cf_stream_t stream) {
    const int chk = check_shape(rows, H);
    if (chk != 0) return chk < 0 ? chk : CF_OK;
    GatedNormArgs p = forward_args(d_residual, d_x, residual_scale, d_gate, rows_per_gate, d_post_scale, d_scale, rows, H, eps, d_sum, d_normed,
                                   d_post_rms, d_rms, d_x8, d_sum8, d_q);
    if (const int rc = check_forward(p, stream_is_f32)) return rc;
    if (!d_qscale || !d_amax || misaligned(d_qscale, 4) || misaligned(d_amax, 4)) return CF_ERR_INVALID_ARG;
    p.qscale = d_qscale; p.amax = d_amax; p.e5m2 = is_e5m2 != 0;
    return gated_norm<Q_RECORD>(p, stream_is_f32 != 0, stream);
}

int cf_gated_add_rmsnorm_backward_workspace_bytes(int rows, int H, int rows_per_gate, size_t* bytes) {
    if (rows < 0 || H < 0 || rows_per_gate < 0 || !bytes) return CF_ERR_INVALID_ARG;
    if (H > kMaxH) return CF_ERR_UNSUPPORTED;
    *bytes = grad_plan(rows, H, rows_per_gate).bytes;
    return CF_OK;
}

int cf_gated_add_rmsnorm_backward(const uint16_t* d_grad_normed, const void* d_sum, const uint16_t* d_x, int stream_is_f32, float residual_scale,
                                  const uint16_t* d_gate, int rows_per_gate, const uint16_t* d_post_scale, const uint16_t* d_scale,
                                  const float* d_post_rms, const float* d_rms, const void* d_grad_sum, int rows, int H, void* d_grad_residual,
                                  uint16_t* d_grad_x, void* d_grad8, const float* d_qscale, float* d_amax, float* d_grad_post_scale,
                                  float* d_grad_scale, float* d_grad_gate, int accumulate, void* d_workspace, size_t workspace_bytes,
                                  cf_stream_t stream) {
    return gated_grad(grad_args(d_grad_normed, d_sum, d_x, residual_scale, d_gate, rows_per_gate, d_post_scale, d_scale, d_post_rms, d_rms, d_grad_sum,
                                rows, H, d_grad_residual, d_grad_x, d_grad8, d_qscale, d_amax, d_grad_gate),
                      false, stream_is_f32, d_grad_post_scale, d_grad_scale, accumulate, d_workspace, workspace_bytes, stream);
}

int cf_gated_add_rmsnorm_backward_ckpt8(const uint16_t* d_grad_normed, const void* d_sum8, const void* d_x8, int stream_is_f32, float residual_scale,
                                        const uint16_t* d_gate, int rows_per_gate, const uint16_t* d_post_scale, const uint16_t* d_scale,
                                        const float* d_post_rms, const float* d_rms, const void* d_grad_sum, int rows, int H, void* d_grad_residual,
                                        uint16_t* d_grad_x, void* d_grad8, const float* d_qscale, float* d_amax, float* d_grad_post_scale,
                                        float* d_grad_scale, float* d_grad_gate, int accumulate, void* d_workspace, size_t workspace_bytes,
                                        cf_stream_t stream) {
    return gated_grad(grad_args(d_grad_normed, d_sum8, d_x8, residual_scale, d_gate, rows_per_gate, d_post_scale, d_scale, d_post_rms, d_rms, d_grad_sum,
                                rows, H, d_grad_residual, d_grad_x, d_grad8, d_qscale, d_amax, d_grad_gate),
                      true, stream_is_f32, d_grad_post_scale, d_grad_scale, accumulate, d_workspace, workspace_bytes, stream);
}

}  // extern "C"
