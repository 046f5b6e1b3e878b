// SwiGLU with the 8-bit operand of the product behind it and with gate and up kept in 8 bits, and its gradient from those bytes.
//
// Forward, per element:  a = g * s * u,  s = 1 / (1 + e^-g);  per 128 elements of a row:  e4m3(g * 448 / max|g|), e4m3(u * 448 / max|u|);  q = f8(a * scale).
// Backward, with g and u from their bytes:  dg = dO * u * s * (1 + g * (1 - s)),  du = dO * g * s.
#include "rows.hpp"

#include <type_traits>

namespace cf {
namespace {

constexpr int kKeepThreads = 512;
constexpr int kMaxRow = 32768;              // of the form that holds a whole row

// sigmoid(g), by the two units' instructions (1 ulp each).  The rounding of the exponent's argument costs e^-g a relative 1.2 |g| 2^-24, so the result is off by
// (6 + 1.2 |g| (1 - s)) 2^-24 at most; carrying the argument in two terms took four more of eleven instructions.  0 where e^-g leaves fp32.
__device__ __forceinline__ float sigmoid(float g) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504f));
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
    unsigned row0;                  // the launch's first row
    unsigned parts, turns, total;   // pieces of a row, pieces that a workgroup takes, pieces of all the launch's rows
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
// The largest |v| of a group's 16 lanes, without its NaNs: as the bits of bf16 pairs while there are none, which costs half.
__device__ __forceinline__ float group_max(const Raw8<false>& r) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) m = pk_absmax(m, r.v[0][k]);
    m = max(m << 16, m & 0xffff0000u);
    if (__any(m > kInf)) {
        float f = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f = fmaxf(f, fabsf(r.at(i)));
        m = __float_as_uint(f);
    }
    return __uint_as_float(max16(m));
}
// a lane's value for the 16 around it
template <int LANE>
__device__ __forceinline__ float from_lane(float v) { return __uint_as_float(dpp<0x150 + LANE>(__float_as_uint(v))); }
__device__ __forceinline__ float largest(const float (&a)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(a[i]));
    return m;
}

// A thread has V chunks of eight elements of a row, chunk c by thread c % T of the row's workgroup or, where the scale is not the whole row's, of one of its `parts`.  Sixteen
// lanes are a group of 128 elements.  Of the two (Q_BLOCK: three) scales of a group each quarter of its lanes makes one, in the same instructions: a division takes a dozen.
// What has been divided by its own maximum needs no clamp, and no look for NaNs: the conversion keeps them.
// Bound by HBM once the instructions are few enough (30 an element in all; with 41, divisions by every lane, clamps and looks for NaNs, 8192 x 8192 took 90 to 102 us): 7 bytes an element,
// 8192 x 8192 80 us (5.9 TB/s) with a scale a row or a group, 90 where a maximum is recorded, 8192 x 14336 144 (5.8); 1000 x 5461 9.4.
// A whole row wants as few chunks a thread as it can have: 1, 2, 4 of them 78.6, 82.8, 83.9 us at 4096 wide, 81.0, 83.9, 85.3 at 8192, 85 each at 14336; 2048 x 18432
// with three 50, with four 65.  Beyond 24576 a row of four fills a CU and its phases follow each other (2048 x 28672 88 us, 4.7 TB/s; a second one there would spill: 136).
template <int QMODE, bool TAIL, bool ONE_WAVE, int V>
__global__ __launch_bounds__(ONE_WAVE ? 256 : QMODE == Q_ROWS ? 1024 : kKeepThreads) void k_swiglu_keep(const SwigluKeepArgs p) {
    __shared__ uint32_t sh[2][16];
    const int T = ONE_WAVE ? kWave : blockDim.x;
    unsigned row, part = 0;
    int t = threadIdx.x;
    if constexpr (ONE_WAVE) {
        row = __builtin_amdgcn_readfirstlane(p.row0 + blockIdx.x * 4 + (threadIdx.x >> 6));
        t &= 63;
        if (row >= static_cast<unsigned>(p.rows)) return;
    } else if constexpr (QMODE == Q_ROWS) {
        row = p.row0 + blockIdx.x;
    } else {
        const unsigned index = blockIdx.x * (QMODE == Q_RECORD ? p.turns : 1);
        row = p.row0 + index / p.parts;
        part = index % p.parts;
    }
    const unsigned groups = (static_cast<unsigned>(p.I) + 127) / 128;
    const int lane = threadIdx.x & 15;
    auto at = [&](unsigned piece, int j) { return (static_cast<int>(piece) * T * V + t + j * T) * 8; };

    Raw8<false> g[V], u[V];
    auto load = [&] {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int n = p.I - at(part, j);
            clear8(g[j]);
            clear8(u[j]);
            if (n > 0) {
                const size_t from = row * p.ld + at(part, j);
                const bool whole = static_cast<size_t>(static_cast<unsigned>(p.rows) - 1 - row) * p.ld + n >= 8;       // eight elements from here on in the tensor
                load8<false, TAIL>(p.gate, from, n, whole, g[j]);
                load8<false, TAIL>(p.up, from, n, whole, u[j]);
            }
        }
    };
    load();
    const bool e5m2 = QMODE != Q_BLOCK && p.e5m2;
    const float F = e5m2 ? 57344.0f : 448.0f;
    float qs = 0.0f;
    if constexpr (QMODE == Q_RECORD) {
        qs = *p.qscale;
        saturate_fp8(qs);
    }
    float a[QMODE == Q_ROWS ? V : 1][8], most = 0.0f;
    // the descale that this lane writes; the pointers in registers, or the compiler loads the one that is chosen, and waits for it
    float *descale = p.gate_descale, *second = p.up_descale, *third = p.descale;
    asm volatile("" : "+s"(descale), "+s"(second), "+s"(third));
    descale = lane == 0 ? descale : lane == 4 ? second : third;
    auto chunk = [&](Raw8<false> gate, Raw8<false> up, float (&o)[8], unsigned in_row, unsigned piece, int j) {
        const int from = at(piece, j), n = p.I - from;
        const size_t to = static_cast<size_t>(in_row) * p.I + from, slot = static_cast<size_t>(in_row) * groups + (static_cast<unsigned>(from) >> 7);
        cut<TAIL>(gate, n);
        cut<TAIL>(up, n);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = gate.at(i);
            o[i] = v * sigmoid(v) * up.at(i);
        }
        float m = largest(o);
        const float mg = group_max(gate), mu = group_max(up);
        float one = lane < 4 ? mg : mu;
        if constexpr (QMODE == Q_BLOCK) {
            m = __uint_as_float(max16(__float_as_uint(m)));
            one = lane < 8 ? one : m;
        }
        one = fmaxf(one, 1e-12f);
        const float s = 448.0f / one, d = one / 448.0f;
        if ((lane & 3) == 0 && lane < (QMODE == Q_BLOCK ? 12 : 8) && n > -8 * lane) {         // the group's first element is there
            descale[slot] = d;
            if (QMODE == Q_BLOCK && lane == 8) p.scale[slot] = s;
        }
        const float sg = from_lane<0>(s), su = from_lane<4>(s);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = gate.at(i) * sg;
        if (n > 0) store8_bytes<TAIL>(p.gate8, to, n, convert8_fp8<false>(v));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = up.at(i) * su;
        if (n > 0) store8_bytes<TAIL>(p.up8, to, n, convert8_fp8<false>(v));
        most = fmaxf(most, m);
        if constexpr (QMODE != Q_ROWS) {
            const float sa = QMODE == Q_BLOCK ? from_lane<8>(s) : qs;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = o[i] * sa;
            u32x2_any b;
            if (QMODE == Q_RECORD && __any(!(m * fabsf(qs) < __builtin_inff()))) b = pack8_fp8(e5m2, false, v);
            else b = e5m2 ? convert8_fp8<true>(v) : convert8_fp8<false>(v);
            if (n > 0) store8_bytes<TAIL>(p.q, to, n, b);
        }
    };
    if constexpr (QMODE == Q_RECORD) {
        const unsigned turns = p.total - blockIdx.x * p.turns < p.turns ? p.total - blockIdx.x * p.turns : p.turns;
        for (unsigned turn = 0; turn < turns; ++turn) {
            const Raw8<false> now_g = g[0], now_u = u[0];
            const unsigned now_row = row, now_part = part;
            if (turn + 1 < turns) {
                const unsigned index = blockIdx.x * p.turns + turn + 1;
                row = p.row0 + index / p.parts;
                part = index % p.parts;
                load();
            }
            chunk(now_g, now_u, a[0], now_row, now_part, 0);
            if (turn == 0 && turns > 1 && blockIdx.x % 64 == 0) {
                const uint32_t m = row_max<false>(__float_as_uint(most), sh[0]);
                if (threadIdx.x == 0) atomic_max_nonneg(p.amax, __uint_as_float(m));
            }
        }
        const uint32_t m = row_max<false>(__float_as_uint(most), sh[1]);
        if (threadIdx.x == 0) {
            if (turns > 1) {
                if (above_l2_copy(p.amax, m)) atomic_max_nonneg(p.amax, __uint_as_float(m));
            } else {
                float before;
                raise_first(p.amax, m, blockIdx.x, gridDim.x, before);
                raise_last(p.amax, m, blockIdx.x, gridDim.x, before);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) chunk(g[j], u[j], a[QMODE == Q_ROWS ? j : 0], row, part, j);
    }
    if constexpr (QMODE == Q_ROWS) {
        most = __uint_as_float(row_max<ONE_WAVE>(__float_as_uint(most), sh[0]));
        most = fmaxf(most, 1e-12f);
        const float s = F / most;
        if (t == 0) {
            p.scale[row] = s;
            p.descale[row] = most / F;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int n = p.I - at(0, j);
#pragma unroll
            for (int i = 0; i < 8; ++i) a[j][i] *= s;
            if (n > 0) store8_bytes<TAIL>(p.q, static_cast<size_t>(row) * p.I + at(0, j), n, e5m2 ? convert8_fp8<true>(a[j]) : convert8_fp8<false>(a[j]));
        }
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
    unsigned row0, parts;
    unsigned tile0, tiles;          // k_swiglu_grad8: the launch's first tile, and how many it has
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

// bf16 outputs, a chunk a thread; workgroups as k_swiglu_keep's.  Bound by HBM: 10 bytes an element with the activation, 8192 x 8192 114 us (5.9 TB/s).
template <bool TAIL>
__global__ __launch_bounds__(kKeepThreads) void k_swiglu_grad(const SwigluGradArgs p) {
    const unsigned row = p.row0 + blockIdx.x / p.parts, groups = (static_cast<unsigned>(p.I) + 127) / 128;
    const int at = ((blockIdx.x % p.parts) * blockDim.x + threadIdx.x) * 8, n = p.I - at;
    if (n <= 0) return;
    const size_t from = static_cast<size_t>(row) * p.I + at, slot = static_cast<size_t>(row) * groups + (static_cast<unsigned>(at) >> 7);
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

typedef uint32_t u32x4_byte __attribute__((ext_vector_type(4), aligned(1)));

// 8-bit outputs, 9 bytes an element, bound by HBM and by how well lines are filled: 8192 x 14336 214 us (5.0 TB/s), 2000 x 8192 42, whose transposed rows begin anywhere in a line.
// A workgroup has 128 x 128 elements (64 columns: 250 us; 64 rows: 250; 256 rows: 215, and no better where lines are split), a thread four rows of eight of them, whose bytes it writes along the rows and, through LDS, along the columns.
// Pieces that are whole 128-byte lines leave past the L2 (8192 x 14336: 213 us, 223 through it); where they are not (WHOLE_ROWS: of the straight outputs, WHOLE_LINES: of the transposed), the
// L2 puts a line together from neighbouring tiles, which is why one XCD has them: 8191 x 8192 240 us past it, 153 through it, 162 with the tiles in row-major order over all XCDs.
// LDS holds [column][128 bytes of rows] for each of the three outputs.  A wavefront's store instruction writes four bytes for each of 16 column blocks and four row blocks:
// the 16-byte pieces of a column are xor-swizzled by the column block, and the upper eight blocks store their columns in swapped pairs, so that 64 lanes hit 64 banks.
constexpr int kTile = 128, kTileThreads = 512;
constexpr unsigned kLaunchTiles = (1u << 23) - 8;       // a launch has fewer than 2^32 threads
template <bool TAIL, bool WHOLE_ROWS, bool WHOLE_LINES>
__global__ __launch_bounds__(kTileThreads) void k_swiglu_grad8(const SwigluGradArgs p) {
    __shared__ __attribute__((aligned(16))) uint8_t tile[3][kTile * kTile];
    __shared__ uint32_t sh[16];
    // the eight XCDs, which take workgroups in turn, each have an eighth of the launch's tiles, in strips of a few column tiles and down the rows within one
    const unsigned across = (static_cast<unsigned>(p.I) + kTile - 1) / kTile, rows = p.rows, down = (rows + kTile - 1) / kTile;
    const unsigned each = (p.tiles + 7) / 8, here = blockIdx.x % 8 * each + blockIdx.x / 8, index = p.tile0 + here;
    if (blockIdx.x / 8 >= each || here >= p.tiles) return;
    constexpr unsigned kStrip = WHOLE_LINES ? 8 : 4;
    const unsigned strip = index / (kStrip * down) * kStrip, rest = index % (kStrip * down), wide = across - strip < kStrip ? across - strip : kStrip;
    const unsigned r0 = rest / wide * kTile, group = strip + rest % wide;
    const int c0 = static_cast<int>(group) * kTile, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int at = c0 + tx * 8, n = p.I - at;
    float s = *p.qscale, as = p.act8_t ? *p.act_qscale : 0.0f;
    saturate_fp8(s);
    saturate_fp8(as);
    Raw8<false> d[4];
    u32x2_any g8[4], u8[4], bytes[3][4];
    float gs[4], us[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned row = r0 + ty * 4 + i;
        clear8(d[i]);
        g8[i] = u8[i] = u32x2_any{0, 0};
        gs[i] = us[i] = 0.0f;
        if (row < rows && n > 0) {
            const size_t from = static_cast<size_t>(row) * p.I + at, slot = static_cast<size_t>(row) * across + group;
            const bool whole = static_cast<size_t>(rows - 1 - row) * p.I + n >= 8;
            load8<false, TAIL>(p.grad, from, n, whole, d[i]);
            g8[i] = load8_bytes<TAIL>(p.gate8, from, n, whole);
            u8[i] = load8_bytes<TAIL>(p.up8, from, n, whole);
            gs[i] = p.gate_descale[slot];
            us[i] = p.up_descale[slot];
        }
    }
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned row = r0 + ty * 4 + i;
        Grads8 o;
        grads8<TAIL>(d[i], g8[i], u8[i], gs[i], us[i], n, o);
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (!TAIL || k < n) m = fmaxf(fmaxf(m, fabsf(o.dg[k])), fabsf(o.du[k]));
        most = fmaxf(most, m);
        const bool usual = __all(m * fabsf(s) < __builtin_inff() && largest(o.a) * fabsf(as) < __builtin_inff());       // no product an infinity
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            o.dg[k] *= s;
            o.du[k] *= s;
            o.a[k] *= as;
        }
        bytes[0][i] = usual ? convert8_fp8<true>(o.dg) : pack8_fp8(true, false, o.dg);
        bytes[1][i] = usual ? convert8_fp8<true>(o.du) : pack8_fp8(true, false, o.du);
        bytes[2][i] = usual ? convert8_fp8<false>(o.a) : pack8_fp8(false, false, o.a);
        if (row < rows && n > 0) {
            const size_t to = static_cast<size_t>(row) * 2 * p.I + at;
            store8_bytes<TAIL, WHOLE_ROWS>(p.grad8, to, n, bytes[0][i]);
            store8_bytes<TAIL, WHOLE_ROWS>(p.grad8, to + p.I, n, bytes[1][i]);
        }
    }
    auto out_of = [&](int part) { return part == 2 ? p.act8_t : p.grad8_t ? p.grad8_t + (part == 1 ? static_cast<size_t>(p.I) * rows : 0) : nullptr; };
    const bool swap = tx & 8;
#pragma unroll
    for (int part = 0; part < 3; ++part) {
        if (!out_of(part)) continue;            // the same in every thread
        uint8_t* wr = tile[part] + tx * 8 * kTile + (((ty >> 2) ^ (tx & 7)) << 4) + (ty & 3) * 4;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t c[4];
            transpose4x4(bytes[part][0][half], bytes[part][1][half], bytes[part][2][half], bytes[part][3][half], c);
#pragma unroll
            for (int k = 0; k < 4; ++k)          // instruction k stores column k ^ swap
                *reinterpret_cast<uint32_t*>(wr + (half * 4 + (k ^ (swap ? 1 : 0))) * kTile) = swap ? c[k ^ 1] : c[k];
        }
    }
    __syncthreads();
    const int chunk = threadIdx.x & 7, rr = threadIdx.x >> 3;       // 8 lanes cover one 128-byte output row
    const unsigned row = r0 + chunk * 16;
#pragma unroll
    for (int part = 0; part < 3; ++part) {
        uint8_t* out = out_of(part);
        if (!out) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = i * 64 + rr;
            if (c0 + c >= p.I || row >= rows) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(&tile[part][c * kTile + ((chunk ^ ((c >> 3) & 7)) << 4)]);
            uint8_t* to = out + static_cast<size_t>(c0 + c) * rows + row;
            if (!TAIL || row + 16 <= rows) {
                if constexpr (WHOLE_LINES) __builtin_nontemporal_store(u32x4_byte{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4_byte*>(to));
                else *reinterpret_cast<u32x4_byte*>(to) = u32x4_byte{v.x, v.y, v.z, v.w};
            } else {
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (row + k < rows) to[k] = static_cast<uint8_t>(w[k >> 2] >> (8 * (k & 3)));
            }
        }
    }
    const uint32_t m = row_max<false>(__float_as_uint(most), sh);
    if (threadIdx.x == 0) {
        float before;
        raise_first(p.amax, m, blockIdx.x, gridDim.x, before);
        raise_last(p.amax, m, blockIdx.x, gridDim.x, before);
    }
}

// Workgroups of a row with V chunks a thread, and their threads.
struct Parts { unsigned parts, threads; };
Parts row_parts(int I, int V) {
    const unsigned chunks = (static_cast<unsigned>(I) + 7) / 8, most = kKeepThreads * V, parts = (chunks + most - 1) / most;
    const unsigned each = (chunks + parts * V - 1) / (parts * V);
    return {parts, (each + kWave - 1) / kWave * kWave};
}
// rows of a launch: fewer than 2^32 threads; a row of fewer than 2^30 elements has 2^18 parts at most
unsigned launch_rows(unsigned parts) { return (kLaunchRows << 1) / parts; }

// Recording a maximum: a workgroup that takes two pieces in turn has one maximum to report where it had two, and one in 64 raises it after the first piece, before any
// other looks.  8192 x 14336: one piece 151 to 157 us, two 145, three 149, four 154; as many workgroups as run at once 167.  One and two elsewhere, us with the maximum's clearing:
//                 4096 wide       6144            8192            11008           14336           16384
//     1000 rows  11.1   10.6    16.7   13.9    17.1   15.4    22.6   20.4    25.5   24.4    29.6   27.5
//     2048       18.2   15.7    24.4   22.7    29.7   28.6    38.1   35.1    44.4   42.4    48.6   47.2
//     4096       31.3   28.8    40.2   37.4    49.3   49.1    64.8   61.4    80.5   75.6    85.0   86.6
//     8192       51.1   48.8    69.9   66.1    87.3   90.7     118    114     153    145     157    165
// So two are ahead below kTurnPieces as well, and one at powers of two from 8192 wide on with many rows: the rule goes by the number of pieces alone and takes neither.
constexpr unsigned kTurnPieces = 4096;

template <int QMODE, bool TAIL>
int launch_keep(SwigluKeepArgs p, hipStream_t st) {
    const Parts cut = QMODE == Q_ROWS ? Parts{1, 0} : row_parts(p.I, 1);
    p.parts = cut.parts;
    const unsigned rows = p.rows, most = QMODE == Q_ROWS ? kLaunchRows : launch_rows(cut.parts);
    for (p.row0 = 0; p.row0 < rows; p.row0 += most) {
        const unsigned n = rows - p.row0 < most ? rows - p.row0 : most;
        if constexpr (QMODE == Q_ROWS) {
            if (p.I <= kOneWaveH) k_swiglu_keep<QMODE, TAIL, true, 1><<<(n + 3) / 4, 4 * kWave, 0, st>>>(p);
            else if (p.I <= kOneChunkH) k_swiglu_keep<QMODE, TAIL, false, 1><<<n, row_threads(p.I, 1), 0, st>>>(p);
            else if (p.I <= 2 * kOneChunkH) k_swiglu_keep<QMODE, TAIL, false, 2><<<n, row_threads(p.I, 2), 0, st>>>(p);
            else if (p.I <= 3 * kOneChunkH) k_swiglu_keep<QMODE, TAIL, false, 3><<<n, row_threads(p.I, 3), 0, st>>>(p);
            else k_swiglu_keep<QMODE, TAIL, false, 4><<<n, row_threads(p.I, 4), 0, st>>>(p);
        } else {
            p.total = n * cut.parts;
            p.turns = QMODE == Q_RECORD && p.total >= kTurnPieces ? 2 : 1;
            k_swiglu_keep<QMODE, TAIL, false, 1><<<(p.total - 1) / p.turns + 1, cut.threads, 0, st>>>(p);
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
    const Parts cut = row_parts(I, 1);
    p.parts = cut.parts;
    const unsigned most = launch_rows(cut.parts), all = rows;
    for (p.row0 = 0; p.row0 < all; p.row0 += most) {
        const unsigned n = all - p.row0 < most ? all - p.row0 : most;
        if (I % 8 != 0) k_swiglu_grad<true><<<n * cut.parts, cut.threads, 0, st>>>(p);
        else k_swiglu_grad<false><<<n * cut.parts, cut.threads, 0, st>>>(p);
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
    if (tiles >= static_cast<size_t>(1) << 31) return CF_ERR_UNSUPPORTED;         // some 2^45 elements: 70 terabytes of d_grad_out
    hipStream_t st = as_stream(stream);
    auto go = [&](auto rows_whole, auto lines_whole) {
        constexpr bool ROWS = decltype(rows_whole)::value, LINES = decltype(lines_whole)::value;
        for (p.tile0 = 0; p.tile0 < tiles; p.tile0 += kLaunchTiles) {
            p.tiles = tiles - p.tile0 < kLaunchTiles ? static_cast<unsigned>(tiles) - p.tile0 : kLaunchTiles;
            const unsigned grid = (p.tiles + 7) / 8 * 8;
            if constexpr (!(ROWS && LINES)) {           // whole tiles have no tails
                if (rows % 16 != 0 || I % 8 != 0) {
                    k_swiglu_grad8<true, ROWS, LINES><<<grid, kTileThreads, 0, st>>>(p);
                    continue;
                }
            }
            k_swiglu_grad8<false, ROWS, LINES><<<grid, kTileThreads, 0, st>>>(p);
        }
    };
    const std::true_type yes{};
    const std::false_type no{};
    if (I % kTile == 0) rows % kTile == 0 ? go(yes, yes) : go(yes, no);
    else rows % kTile == 0 ? go(no, yes) : go(no, no);
    return launch_status();
}

}  // extern "C"
