// RMSNorm of every query and key head with the rotary rotation in the same pass, forward and backward.
//
// Per row x of D features (one token's head), weight w, r = 1 / sqrt(mean(x^2) + eps), n = x r, z = n w; the first R
// features turn in pairs by their position's angle, pair i (cos c_i, sin s_i from the table's row):
//   (y1, y2) = (z1 c - z2 s, z2 c + z1 s),    y = z past R
// pairs are (i, i + R/2), or (2i, 2i + 1) when interleaved. Backward: dz = the rotation's transpose of dy, then
//   dw = sum over rows of dz n,   dx = r (dz w - n mean(dz w n))
// A pair's angle may come from one of up to four position axes (time, height, width ...): `axis_end[a]` is the first
// pair past axis a. Everything is fp32 with one rounding to the activations' type. A position outside the table
// reads nothing: its rotated features are NaN.
//
// One read of x (and dy) and one write: bound by HBM. At 8 x 4,096 tokens of 16 + 16 bf16 heads of 128, R = 32, the
// forward takes 97 us (0.85 of a copy's rate), the backward 150 us (0.82). What it took, in that shape (both together):
//   * a warp takes one token and a group of its heads, so the table's row is loaded once per group;
//   * a lane holds both members of its pairs; with 8 neighbouring features a lane and the partners by shuffle the
//     forward's instructions alone were 0.6 of the time (both directions 287 us, with the ring 294);
//   * rows come through an asynchronous ring, 8 to 10 KB a warp ahead of their use: plain loads of four rows at a time,
//     in registers that the arithmetic wants too, 290 us, with the ring 247.
// qk_rows_kernel takes any even R, alignment and stride, a warp per row through shared memory. dw: registers, then one
// partial per block, then a second launch that adds the partials in a fixed order (no atomics: the same inputs give the
// same bits).
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "launch.h"

namespace gdn {
namespace qknr {

constexpr int NTHR = 256, NW = NTHR / 32;
constexpr int MAX_AXES = 4, MAX_D = 512;

struct Side {  // the queries or the keys
    const void *x, *dy;
    void* y;        // forward: y, backward: dx; contiguous [B, T, heads, D]
    const void* w;  // [D]
    int64_t sb, st, sh;  // strides of x in elements
    int heads;
};
struct Args {
    Side side[2];
    const float* table;     // [n_pos, R]: cos, then sin
    const void* positions;  // [axes, B * T], int64 or int32
    float* part;            // backward: [blocks][2][D] partial weight gradients
    int64_t tokens, T, n_pos;
    int64_t units;          // (token, head group) pairs
    int groups[2], group;   // head groups of each side, heads per group; groups[1] == 0: a unit is a whole token
    int D, R, axes, pos64, w_dtype;
    int flat;               // consecutive tokens are one stride apart across batch rows too, on both sides
    int axis_end[MAX_AXES];
    float eps;
};

__device__ __forceinline__ float ldw(const void* p, int dtype, int i) { return gate_f(ld_gate_raw(p, dtype, i), dtype); }

__device__ __forceinline__ int axis_of(const Args& a, int pair) {
    int ax = 0;
#pragma unroll
    for (int e = 0; e < MAX_AXES - 1; ++e) ax += (e < a.axes - 1 && pair >= a.axis_end[e]) ? 1 : 0;
    return ax;
}
// the position of token t on an axis, -1 where it is outside the table
__device__ __forceinline__ int64_t position(const Args& a, int64_t t, int ax) {
    const int64_t i = ax * a.tokens + t;
    const int64_t p = a.pos64 ? ((const int64_t*)a.positions)[i] : (int64_t)((const int32_t*)a.positions)[i];
    return p >= 0 && p < a.n_pos ? p : -1;
}
__device__ __forceinline__ void angle(const Args& a, int64_t t, int pair, float& c, float& s) {
    const int64_t p = position(a, t, axis_of(a, pair));
    if (p < 0) {
        c = s = __int_as_float(0x7fc00000);
        return;
    }
    c = a.table[p * a.R + pair];
    s = a.table[p * a.R + a.R / 2 + pair];
}
// cos and sin of the N pairs from `pair` (a multiple of N) on, p the position of token t on the first one's axis;
// vector loads where the pairs share their axis
template <int N>
__device__ __forceinline__ void angles(const Args& a, int64_t t, int64_t p, int pair, float* c, float* s) {
    if (a.axes > 1 && axis_of(a, pair + N - 1) != axis_of(a, pair)) {
#pragma unroll
        for (int e = 0; e < N; ++e) angle(a, t, pair + e, c[e], s[e]);
        return;
    }
    if (p < 0) {
#pragma unroll
        for (int e = 0; e < N; ++e) c[e] = s[e] = __int_as_float(0x7fc00000);
        return;
    }
    ldv<float, N>(a.table, p * a.R + pair, *(float(*)[N])c);
    ldv<float, N>(a.table, p * a.R + a.R / 2 + pair, *(float(*)[N])s);
}
// 4 weights from feature f on (f a multiple of 4, the weights 16-byte aligned)
__device__ __forceinline__ void weights4(const void* w, int dtype, int f, float2& lo, float2& hi) {
    float o[4];
    if (dtype == GDN_FP32) ldv<float, 4>(w, f, o);
    else if (dtype == GDN_BF16) ldv<__nv_bfloat16, 4>(w, f, o);
    else ldv<__half, 4>(w, f, o);
    lo = make_float2(o[0], o[1]);
    hi = make_float2(o[2], o[3]);
}

// 16 bytes from global to shared memory, asynchronously
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// A warp's batches pass through a ring in shared memory: 192 KB of them on an SM.
template <typename TA, int LPR, bool BWD>
struct Ring {
    static constexpr int BLOCKS = 2;  // resident blocks (the backward needs 128 registers; forward: 2 97 us, 3 104)
    static constexpr int U = 8 / (int)sizeof(TA);  // rows of a lane group in a batch
    static constexpr int ROWS = U * 32 / LPR, ROW = LPR * 8 * (int)sizeof(TA);  // rows of a batch, bytes of a row
    static constexpr int SIDE = ROWS * ROW, BATCH = SIDE * (BWD ? 2 : 1);  // bytes: x, then dy
    static constexpr int STAGES = 192 / BLOCKS * 1024 / NW / BATCH;
    static constexpr int BYTES = NW * STAGES * BATCH;
    static_assert(STAGES >= 2, "ring");
};

// Rows of D = 8 LPR features, R a multiple of 8, rows, weights and table aligned to 16 bytes. A lane holds two vectors of
// 4 features, one in each half of the turned features or one in each half of the others: both members of its pairs are
// its own, and a warp's accesses fill whole sectors. A warp takes a unit: one token's heads on both sides
// (groups[1] == 0: the angles are loaded once), or `group` of them on one side.
template <typename TA, int LPR, bool INTER, bool BWD>
__global__ void __launch_bounds__(NTHR, (Ring<TA, LPR, BWD>::BLOCKS)) qk_vec_kernel(const __grid_constant__ Args a) {
    using G = Ring<TA, LPR, BWD>;
    constexpr int RPW = 32 / LPR, U = G::U, D = LPR * 8;
    constexpr float INV_D = 1.f / D;
    using Vec = RawVec<TA, 4>;
    extern __shared__ __align__(16) uint8_t ring[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, l = lane % LPR, sub = lane / LPR;
    const bool turned = l * 8 < a.R;
    const int fa = turned ? l * 4 : a.R / 2 + l * 4, ab = (turned ? a.R : D - a.R) / 2, fb = fa + ab;
    const int pair0 = INTER ? l * 2 : l * 4, axis0 = turned ? axis_of(a, pair0) : 0;
    uint8_t* const slots = ring + warp * (G::STAGES * G::BATCH);
    float dw[2][8] = {};
    const int per_token = a.groups[0] + a.groups[1];
    const int64_t step = (int64_t)gridDim.x * NW;

    // a place in the sequence of the warp's batches: h is the batch's first head
    struct Place {
        int64_t unit, t;
        int z, z1, g0, h, h1;
        bool new_unit, new_side;
    };
    auto enter_side = [&](Place& c) {
        const int heads = a.side[c.z].heads;
        c.h = c.g0;
        c.h1 = a.groups[1] ? min(c.g0 + a.group, heads) : heads;
        c.new_side = true;
    };
    auto enter_unit = [&](Place& c) {
        c.new_unit = true;
        c.t = c.unit;
        c.z = 0;
        c.z1 = 2;
        c.g0 = 0;
        if (a.groups[1]) {
            c.t = c.unit / per_token;
            c.g0 = (int)(c.unit % per_token);
            c.z = c.g0 >= a.groups[0] ? 1 : 0;
            c.z1 = c.z + 1;
            c.g0 = (c.g0 - (c.z ? a.groups[0] : 0)) * a.group;
        } else if (a.side[0].heads == 0) {
            c.z = 1;
        } else if (a.side[1].heads == 0) {
            c.z1 = 1;
        }
        enter_side(c);
    };
    auto advance = [&](Place& c) {
        c.new_unit = c.new_side = false;
        c.h += G::ROWS;
        if (c.h < c.h1) return;
        if (++c.z < c.z1) {
            enter_side(c);
        } else {
            c.unit += step;
            if (c.unit < a.units) enter_unit(c);
        }
    };
    // a lane copies 16 bytes of every LPR-th row piece; the rows of a batch past the side's end are left as they are
    constexpr int PER = G::ROW / 16, CROWS = 32 / PER > 0 ? 32 / PER : 1, COPIES = G::SIDE / 512;
    static_assert(PER <= 32 || PER == 64, "row size");
    auto fetch = [&](const Place& c, int stage) {
        if (c.unit < a.units) {
            const Side& sd = a.side[c.z];
            const int64_t tok = a.flat ? c.t * sd.st : (c.t / a.T) * sd.sb + (c.t % a.T) * sd.st;
            const int row = lane / PER, piece = lane % PER;
            const int h = c.h + row;
            const TA* x = (const TA*)sd.x + tok + h * sd.sh + piece * (16 / (int)sizeof(TA));
            const TA* dy = BWD ? (const TA*)sd.dy + (c.t * sd.heads + h) * D + piece * (16 / (int)sizeof(TA)) : nullptr;
            const uint32_t dst = (uint32_t)__cvta_generic_to_shared(slots) + stage * G::BATCH + lane * 16;
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
                // piece i * 32 + lane of the batch: PER = 64 takes two copies a row
                const int hi = PER == 64 ? i / 2 : i * CROWS, off = PER == 64 ? i % 2 * (512 / (int)sizeof(TA)) : 0;
                if (h + hi < c.h1) {
                    copy16(dst + i * 512, x + off);
                    if (BWD) copy16(dst + G::SIDE + i * 512, dy + hi * D + off);
                }
                if (PER != 64 || i % 2) x += CROWS * sd.sh;
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    Place at{}, ahead{};
    at.unit = (int64_t)blockIdx.x * NW + warp;
    if (at.unit < a.units) enter_unit(at);
    ahead = at;
#pragma unroll 1
    for (int i = 0; i < G::STAGES - 1; ++i) {
        fetch(ahead, i);
        if (ahead.unit < a.units) advance(ahead);
    }
    int stage = 0, stage_ahead = G::STAGES - 1;
    int64_t pos = at.unit < a.units && turned ? position(a, at.t, axis0) : -1;
    // The rotation as y_e = c_e x_e + s_e x_mate(e) over the lane's four float2: mate(e) = e ^ 2, or the float2 itself
    // with its members exchanged (interleaved). The transpose turns the other way.
    float2 c[4], s[4];
    // forward: y = r (x w + mate ws) with the rotation in w and ws; backward: w alone
    float2 w[4], ws[4], acc[4];
#pragma unroll 1
    while (at.unit < a.units) {
        if (at.new_unit) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c[e] = make_float2(1.f, 1.f);
                s[e] = make_float2(0.f, 0.f);
            }
            if (turned) {
                float cp[4], sp[4];
                angles<INTER ? 2 : 4>(a, at.t, pos, pair0, cp, sp);
                if (INTER) {
                    const int ax = axis_of(a, fb / 2);
                    angles<2>(a, at.t, ax == axis0 ? pos : position(a, at.t, ax), fb / 2, cp + 2, sp + 2);
                }
                const int64_t next = at.unit + step;  // the next unit's position, well ahead of its use
                if (next < a.units) pos = position(a, a.groups[1] ? next / per_token : next, axis0);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (BWD) sp[e] = -sp[e];
                    if (INTER) {
                        c[e] = make_float2(cp[e], cp[e]);
                        s[e] = make_float2(-sp[e], sp[e]);
                    }
                }
                if (!INTER) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        c[e] = c[e + 2] = make_float2(cp[2 * e], cp[2 * e + 1]);
                        s[e] = make_float2(-sp[2 * e], -sp[2 * e + 1]);
                        s[e + 2] = make_float2(sp[2 * e], sp[2 * e + 1]);
                    }
                }
            }
        }
        const Side& sd = a.side[at.z];
        if (at.new_side) {
            weights4(sd.w, a.w_dtype, fa, w[0], w[1]);
            weights4(sd.w, a.w_dtype, fb, w[2], w[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[e] = make_float2(0.f, 0.f);
                ws[e] = mul2(INTER ? make_float2(w[e].y, w[e].x) : w[e ^ 2], s[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!BWD) w[e] = mul2(w[e], c[e]);
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(G::STAGES - 2) : "memory");
        __syncwarp();  // the batch is there for the whole warp, and every lane is done with the one before it
        fetch(ahead, stage_ahead);
        if (ahead.unit < a.units) advance(ahead);
        const TA* const bx = (const TA*)(slots + stage * G::BATCH) + sub * D + fa;
        TA* const y = (TA*)sd.y + (at.t * sd.heads + at.h + sub) * D + fa;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (at.h + u * RPW >= at.h1) break;  // the same for the whole warp
            const bool row = at.h + sub + u * RPW < at.h1;  // else leftovers, which reach nothing
            float2 v[4], d[4], s2 = make_float2(0.f, 0.f);
            Vec in[2];
            in[0].load(bx, u * RPW * D);
            in[1].load(bx, u * RPW * D + ab);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = make_float2(in[e / 2].get(e % 2 * 2), in[e / 2].get(e % 2 * 2 + 1));
                s2 = fma2(v[e], v[e], s2);
            }
            float ss = s2.x + s2.y;
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float r = rsqrtf(ss * INV_D + a.eps);
            const float2 r2 = make_float2(r, r);
            if constexpr (!BWD) {
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] = mul2(v[e], w[e]);
                if (turned) {  // not by a zero sine: an infinity would reach its neighbours
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        d[e] = fma2(INTER ? make_float2(v[e].y, v[e].x) : v[e ^ 2], ws[e], d[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] = mul2(d[e], r2);
            } else {
                float2 g[4], g2 = make_float2(0.f, 0.f);
                in[0].load(bx + G::SIDE / (int)sizeof(TA), u * RPW * D);
                in[1].load(bx + G::SIDE / (int)sizeof(TA), u * RPW * D + ab);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    g[e] = make_float2(in[e / 2].get(e % 2 * 2), in[e / 2].get(e % 2 * 2 + 1));
                    d[e] = mul2(g[e], c[e]);
                }
                if (turned) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        d[e] = fma2(INTER ? make_float2(g[e].y, g[e].x) : g[e ^ 2], s[e], d[e]);  // dz
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = mul2(v[e], r2);  // n
                    if (row) acc[e] = fma2(d[e], v[e], acc[e]);
                    d[e] = mul2(d[e], w[e]);
                    g2 = fma2(d[e], v[e], g2);
                }
                float gr = g2.x + g2.y;
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) gr += __shfl_xor_sync(0xffffffffu, gr, o);
                gr *= -INV_D;
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] = mul2(r2, fma2(v[e], make_float2(gr, gr), d[e]));
            }
            if (row) {
                const float o0[4] = {d[0].x, d[0].y, d[1].x, d[1].y}, o1[4] = {d[2].x, d[2].y, d[3].x, d[3].y};
                stv<TA, 4>(y, u * RPW * D, o0);
                stv<TA, 4>(y, u * RPW * D + ab, o1);
            }
        }
        const int z = at.z;
        advance(at);
        if (BWD && (at.new_side || at.unit >= a.units)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                dw[0][2 * e] += z == 0 ? acc[e].x : 0.f;
                dw[0][2 * e + 1] += z == 0 ? acc[e].y : 0.f;
                dw[1][2 * e] += z == 1 ? acc[e].x : 0.f;
                dw[1][2 * e + 1] += z == 1 ? acc[e].y : 0.f;
            }
        }
        stage = stage == G::STAGES - 1 ? 0 : stage + 1;
        stage_ahead = stage_ahead == G::STAGES - 1 ? 0 : stage_ahead + 1;
    }
    if constexpr (BWD) {
        __shared__ float red[NW][2][D];
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float y = dw[z][e];
#pragma unroll
                for (int o = LPR; o < 32; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
                if (sub == 0) red[warp][z][(e < 4 ? fa : fb - 4) + e] = y;
            }
        __syncthreads();
        for (int i = tid; i < 2 * D; i += NTHR) {
            float y = 0.f;
#pragma unroll
            for (int v = 0; v < NW; ++v) y += red[v][i / D][i % D];
            a.part[(int64_t)blockIdx.x * 2 * a.D + i] = y;
        }
    }
}

// Any even R <= D <= MAX_D, any stride and alignment: a warp per row, the row's z (forward) or dy (backward) in
// shared memory for the pair partners. A unit is a (token, head) row here.
template <typename TA, bool BWD>
__global__ void __launch_bounds__(NTHR) qk_rows_kernel(const __grid_constant__ Args a, int inter) {
    constexpr int J = MAX_D / 32;
    __shared__ float buf[NW][MAX_D];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* b = buf[warp];
    float dw[2][J] = {};
    const int per_token = a.side[0].heads + a.side[1].heads;
    for (int64_t unit = (int64_t)blockIdx.x * NW + warp; unit < a.units; unit += (int64_t)gridDim.x * NW) {
        const int64_t t = unit / per_token;
        int h = (int)(unit % per_token);
        const int z = h >= a.side[0].heads ? 1 : 0;
        h -= z ? a.side[0].heads : 0;
        const Side& sd = a.side[z];
        const TA* x = (const TA*)sd.x + (t / a.T) * sd.sb + (t % a.T) * sd.st + h * sd.sh;
        const int64_t row = (t * sd.heads + h) * a.D;
        float v[J], ss = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int f = lane + 32 * j;
            v[j] = f < a.D ? ld(x, f) : 0.f;
            ss = fmaf(v[j], v[j], ss);
        }
        const float r = 1.f / sqrtf(warp_sum(ss) / a.D + a.eps);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int f = lane + 32 * j;
            if (f < a.D) b[f] = BWD ? ld((const TA*)sd.dy, row + f) : v[j] * r * ldw(sd.w, a.w_dtype, f);
        }
        __syncwarp();
        float o[J], g = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int f = lane + 32 * j;
            o[j] = 0.f;
            if (f >= a.D) continue;
            o[j] = b[f];
            if (f < a.R) {
                const int half = a.R / 2, pair = inter ? f / 2 : (f < half ? f : f - half);
                const bool second = inter ? (f & 1) : f >= half;
                const int m = inter ? f ^ 1 : (second ? f - half : f + half);
                float c, s;
                angle(a, t, pair, c, s);
                o[j] = b[f] * c + (second != BWD ? b[m] * s : -b[m] * s);
            }
            if (BWD) {
                const float n = v[j] * r;
                if (z == 0) dw[0][j] = fmaf(o[j], n, dw[0][j]);
                else dw[1][j] = fmaf(o[j], n, dw[1][j]);
                o[j] *= ldw(sd.w, a.w_dtype, f);
                g = fmaf(o[j], n, g);
            }
        }
        if (BWD) g = warp_sum(g) / a.D;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int f = lane + 32 * j;
            if (f < a.D) st((TA*)sd.y, row + f, BWD ? r * (o[j] - v[j] * r * g) : o[j]);
        }
    }
    if constexpr (BWD) {  // the warps' sums, one side after the other through the row buffers
        for (int z = 0; z < 2; ++z) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < J; ++j) b[lane + 32 * j] = z ? dw[1][j] : dw[0][j];
            __syncthreads();
            for (int f = tid; f < a.D; f += NTHR) {
                float y = 0.f;
                for (int v = 0; v < NW; ++v) y += buf[v][f];
                a.part[((int64_t)blockIdx.x * 2 + z) * a.D + f] = y;
            }
        }
    }
}

// dw[z][f] = sum over the blocks' partials, in order: 8 features per block, 128 threads along the partials
__global__ void __launch_bounds__(1024) qk_dw_kernel(const float* part, int blocks, int D, float* dwq, float* dwk) {
    __shared__ float red[128][9];
    const int f = threadIdx.x & 7, s = threadIdx.x >> 3, i = blockIdx.x * 8 + f;
    float y = 0.f;
    if (i < 2 * D)
#pragma unroll 4
        for (int b = s; b < blocks; b += 128) y += part[(int64_t)b * 2 * D + i];
    red[s][f] = y;
    __syncthreads();
#pragma unroll
    for (int k = 64; k > 0; k >>= 1) {
        if (s < k) red[s][f] += red[s + k][f];
        __syncthreads();
    }
    if (s == 0 && i < 2 * D) {
        if (i < D) dwq[i] = red[0][f];
        else dwk[i - D] = red[0][f];
    }
}

// blocks of the backward launch: what the partials' workspace is sized for
static int64_t max_blocks() { return (int64_t)device_sm_count() * 4; }

template <typename TA, int LPR, bool BWD>
static int launch_vec(Args& a, bool inter, cudaStream_t s, int* blocks) {
    // One batch of rows per warp while tokens are few, so that a decode step's rows spread over the SMs; else a token per
    // warp (one load of its angles for all heads). 16 + 16 heads, forward: 64 tokens 3.9 against 6.8 us, 1,024 tokens 7.1
    // against 7.5, 2,048 tokens 11.8 against 9.2.
    if (a.tokens < (int64_t)device_sm_count() * 8) {
        a.group = Ring<TA, LPR, BWD>::ROWS;
        for (int z = 0; z < 2; ++z) a.groups[z] = (a.side[z].heads + a.group - 1) / a.group;
        if (a.groups[1] == 0) {  // no keys: whole tokens after all
            a.groups[0] = 1;
        }
    } else {
        a.group = 0;
        a.groups[0] = 1;
        a.groups[1] = 0;
    }
    a.units = a.tokens * (a.groups[0] + a.groups[1]);
    const int64_t want = (a.units + NW - 1) / NW;
    const unsigned grid = (unsigned)std::min<int64_t>(want, (int64_t)device_sm_count() * Ring<TA, LPR, BWD>::BLOCKS);
    *blocks = (int)grid;
    constexpr int bytes = Ring<TA, LPR, BWD>::BYTES;
    auto* const kernel = inter ? qk_vec_kernel<TA, LPR, true, BWD> : qk_vec_kernel<TA, LPR, false, BWD>;
    if (smem_optin((const void*)kernel, bytes) != cudaSuccess) return GDN_ERR_LAUNCH;
    kernel<<<grid, NTHR, bytes, s>>>(a);
    return GDN_OK;
}

template <typename TA, bool BWD>
static int launch_all(Args& a, bool inter, cudaStream_t s, int* blocks) {
    a.flat = 1;
    for (int z = 0; z < 2; ++z) a.flat = a.flat && (a.side[z].heads == 0 || a.side[z].sb == a.T * a.side[z].st);
    constexpr int V = 16 / (int)sizeof(TA);
    bool vec = (a.D == 64 || a.D == 128 || a.D == 256) && a.R % 8 == 0 && !((uintptr_t)a.table & 15);
    for (int z = 0; z < 2; ++z) {
        const Side& sd = a.side[z];
        vec = vec && !((uintptr_t)sd.w & 15) && !(((uintptr_t)sd.x | (uintptr_t)sd.y | (uintptr_t)sd.dy) & 15) &&
              sd.sb % V == 0 && sd.st % V == 0 && sd.sh % V == 0;
    }
    if (vec) {
        if (a.D == 64) return launch_vec<TA, 8, BWD>(a, inter, s, blocks);
        if (a.D == 128) return launch_vec<TA, 16, BWD>(a, inter, s, blocks);
        return launch_vec<TA, 32, BWD>(a, inter, s, blocks);
    }
    a.units = a.tokens * (a.side[0].heads + a.side[1].heads);
    const unsigned grid = (unsigned)std::min<int64_t>((a.units + NW - 1) / NW, max_blocks());
    *blocks = (int)grid;
    qk_rows_kernel<TA, BWD><<<grid, NTHR, 0, s>>>(a, inter ? 1 : 0);
    return GDN_OK;
}

static bool dtype_ok(int32_t d) { return d == GDN_BF16 || d == GDN_FP16 || d == GDN_FP32; }

// The arguments that both directions share; `any`: there is at least one row.
static int fill(Args& a, const gdn_qk_norm_rope_problem* p, const void* q, const void* k, const void* wq,
                const void* wk, const float* table, const void* positions, bool& any) {
    if (!p) return GDN_ERR_ARGUMENT;
    if (p->B < 0 || p->T < 0 || p->HQ < 0 || p->HK < 0 || p->HQ > (1 << 20) || p->HK > (1 << 20) || p->D <= 0 ||
        p->D > MAX_D || p->R < 0 || p->R > p->D || p->R % 2 || p->n_pos < 0 || p->axes < 1 || p->axes > MAX_AXES)
        return GDN_ERR_SHAPE;
    if (!dtype_ok(p->act_dtype) || !dtype_ok(p->w_dtype)) return GDN_ERR_DTYPE;
    int64_t end = 0;
    for (int i = 0; i < p->axes; ++i) {
        if (p->axes > 1 && p->sections[i] < 0) return GDN_ERR_SHAPE;
        end += p->axes > 1 ? p->sections[i] : p->R / 2;
        a.axis_end[i] = (int)std::min<int64_t>(end, 1 << 20);
    }
    if (end != p->R / 2) return GDN_ERR_SHAPE;
    any = p->B > 0 && p->T > 0 && p->HQ + p->HK > 0;
    if (any && ((p->HQ && !q) || (p->HK && !k) || !wq || !wk || (p->R && (!positions || (p->n_pos && !table)))))
        return GDN_ERR_ARGUMENT;
    a.side[0].x = q; a.side[1].x = k;
    a.side[0].w = wq; a.side[1].w = wk;
    a.side[0].sb = p->q_strides[0]; a.side[0].st = p->q_strides[1]; a.side[0].sh = p->q_strides[2];
    a.side[1].sb = p->k_strides[0]; a.side[1].st = p->k_strides[1]; a.side[1].sh = p->k_strides[2];
    a.side[0].heads = (int)p->HQ; a.side[1].heads = (int)p->HK;
    a.table = table;
    a.positions = positions;
    a.tokens = p->B * p->T;
    a.T = p->T;
    a.n_pos = p->n_pos;
    a.D = (int)p->D; a.R = (int)p->R; a.axes = p->axes; a.pos64 = p->positions_int64; a.w_dtype = p->w_dtype;
    a.eps = p->eps;
    return GDN_OK;
}

}  // namespace qknr
}  // namespace gdn

using namespace gdn;

extern "C" {

int gdn_qk_norm_rope_fwd(const gdn_qk_norm_rope_problem* p, const void* q, const void* k, const void* q_weight,
                         const void* k_weight, const float* table, const void* positions, void* q_out, void* k_out,
                         gdn_stream_t stream) {
    using namespace qknr;
    Args a{};
    bool any = false;
    const int st = fill(a, p, q, k, q_weight, k_weight, table, positions, any);
    if (st != GDN_OK) return st;
    if (!any) return GDN_OK;
    if ((p->HQ && !q_out) || (p->HK && !k_out)) return GDN_ERR_ARGUMENT;
    a.side[0].y = q_out; a.side[1].y = k_out;
    int blocks = 0;
    GDN_DISPATCH_DTYPE(p->act_dtype, TA, (launch_all<TA, false>(a, p->interleaved != 0, (cudaStream_t)stream, &blocks)))
    count_launch();
    return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

size_t gdn_qk_norm_rope_bwd_workspace_size(const gdn_qk_norm_rope_problem* p) {
    if (!p || p->D <= 0 || p->D > qknr::MAX_D) return 0;
    return (size_t)qknr::max_blocks() * 2 * p->D * sizeof(float);
}

int gdn_qk_norm_rope_bwd(const gdn_qk_norm_rope_problem* p, const void* q, const void* k, const void* q_weight,
                         const void* k_weight, const float* table, const void* positions, const void* dq_out,
                         const void* dk_out, void* dq, void* dk, float* dq_weight, float* dk_weight, void* workspace,
                         size_t workspace_bytes, gdn_stream_t stream) {
    using namespace qknr;
    Args a{};
    bool any = false;
    const int st = fill(a, p, q, k, q_weight, k_weight, table, positions, any);
    if (st != GDN_OK) return st;
    if (!dq_weight || !dk_weight) return GDN_ERR_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    if (!any) {
        if (cudaMemsetAsync(dq_weight, 0, p->D * sizeof(float), s) != cudaSuccess ||
            cudaMemsetAsync(dk_weight, 0, p->D * sizeof(float), s) != cudaSuccess)
            return GDN_ERR_LAUNCH;
        return GDN_OK;
    }
    if ((p->HQ && (!dq_out || !dq)) || (p->HK && (!dk_out || !dk))) return GDN_ERR_ARGUMENT;
    if (!workspace || workspace_bytes < gdn_qk_norm_rope_bwd_workspace_size(p)) return GDN_ERR_WORKSPACE;
    if ((uintptr_t)workspace & 3) return GDN_ERR_ALIGN;
    a.side[0].dy = dq_out; a.side[1].dy = dk_out;
    a.side[0].y = dq; a.side[1].y = dk;
    a.part = (float*)workspace;
    int blocks = 0;
    GDN_DISPATCH_DTYPE(p->act_dtype, TA, (launch_all<TA, true>(a, p->interleaved != 0, s, &blocks)))
    qk_dw_kernel<<<(unsigned)((2 * p->D + 7) / 8), 1024, 0, s>>>(a.part, blocks, a.D, dq_weight, dk_weight);
    count_launch(2);
    return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

}  // extern "C"
