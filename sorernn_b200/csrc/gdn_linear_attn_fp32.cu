// The linear-attention scan (linear_attn.cuh) to fp32 accuracy, for fp32 and fp16 activations and head sizes that the
// tensor-memory kernel does not take.
//
// The products run as warp-level tf32 MMAs on operands split in two, x = hi + lo with hi = tf32(x), lo = tf32(x - hi)
// (2^-22 of x is lost): hi hi + hi lo + lo hi, accumulated in fp32, leaves 2^-22 of each term, as fp32 FMAs would leave
// 2^-24 of each partial sum. 16-bit activations are exact in tf32 and need no lo. fp16's range would not hold the state
// and the in-chunk weights, which is why these activations run here and not as 16-bit operands.
//
// One CTA of 8 warps per (value head, piece), all columns of C. Chunks of 32 tokens: the in-chunk products cost
// 2 x 32 (DB + DC) FLOP a token against 4 DB DC for the state's update and read-out. Per chunk
//   P = A B^T (a 16 x 8 tile a warp)      O = A X, scaled, + W(P) C (16 rows x CW / 4 columns a warp)
//   X <- a^nv X + B^T C (16 x CW, or two warps to 16 rows; accumulators)
// X is copied to shared memory once a chunk for the read-out. The next chunk's rows come in by asynchronous copies (two
// stages, in the activations' type) while this one is worked on; rows that are not whole 16-byte vectors are loaded by
// element. Row strides keep the fragments' loads free of bank conflicts, but for B's transposed ones (two-way). Bound by
// the instructions that split and load the fragments: 4 x 1,024 tokens x 16 heads of 128, forward and backward, 882 us in
// fp32 and 642 us in fp16 (20 and 27 TFLOP/s of what the recurrences need). As fp32 FMAs the same tiling took 1,205
// and 1,176 us, held by shared memory's bandwidth.
#include "launch.h"
#include "linear_attn.cuh"
#include "sm100.cuh"

namespace gdn {
namespace linattn {

namespace sk {
constexpr int NTHR = 256;
constexpr int C = 32;       // tokens per chunk
constexpr int PS = C + 4;   // row stride of P

template <typename TA, int DB, int CW>
struct Smem {
    static constexpr int RS = DB + 16 / (int)sizeof(TA), CS = CW + 8, XS = CW + 8;  // row strides in elements
    static constexpr uint32_t A = 0;
    static constexpr uint32_t B = A + C * RS * sizeof(TA);
    static constexpr uint32_t Ct = B + C * RS * sizeof(TA);
    static constexpr uint32_t STAGE = Ct + C * CS * sizeof(TA);
    static constexpr uint32_t X = 2 * STAGE;
    static constexpr uint32_t P = X + DB * XS * 4;
    static constexpr uint32_t PW = P + C * PS * 4;
    static constexpr uint32_t RED = PW + (C + 4) * 4;
    static constexpr uint32_t BYTES = RED + (NTHR / 32 + 3) * 8;
};
static_assert(Smem<float, 128, 128>::BYTES <= 232448, "shared memory budget");
}  // namespace sk

// 16 bytes global -> shared, or zeros
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
    const int n = in ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
// x = hi + lo in tf32; EXACT: x is a tf32 value already
template <bool EXACT>
struct Split {
    uint32_t hi, lo;
    __device__ __forceinline__ explicit Split(float x) {
        if constexpr (EXACT) {
            hi = __float_as_uint(x);
            lo = 0;
        } else {
            // rounded to nearest on the bits (two integer operations; the conversion instruction is slower); lo's bits
            // past tf32's are dropped by the MMA, towards zero, but lo has either sign, so nothing adds up
            hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
            lo = __float_as_uint(x - __uint_as_float(hi));
        }
    }
    __device__ __forceinline__ Split() {}
};
__device__ __forceinline__ void mma8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d += A B for a 16 x 8 x 8 step. Lane (g, t): A (g, t), (g + 8, t), (g, t + 4), (g + 8, t + 4); B (t, g), (t + 4, g);
// d (g, 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1)
// The cross terms go to e: every MMA drops its sum's last bit or so of the accumulator it adds to, and e's are 2^-11 of
// d's (one accumulator for all three left outputs 1.2e-6 off, two 4e-7).
template <bool EA, bool EB>
__device__ __forceinline__ void mma_step(float (&d)[4], float (&e)[4], const Split<EA> (&a)[4],
                                         const Split<EB> (&b)[2]) {
    if constexpr (!EA) mma8(e, a[0].lo, a[1].lo, a[2].lo, a[3].lo, b[0].hi, b[1].hi);
    if constexpr (!EB) mma8(e, a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[0].lo, b[1].lo);
    mma8(d, a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[0].hi, b[1].hi);
}

template <typename TA, int DB, int CW, bool OUT>
__global__ void __launch_bounds__(sk::NTHR) linear_attn_fp32_kernel(const __grid_constant__ Scans all, int vec) {
    using namespace sk;
    using S = Smem<TA, DB, CW>;
    extern __shared__ __align__(16) uint8_t smem[];
    float* const sX = (float*)(smem + S::X);
    float* const sP = (float*)(smem + S::P);    // [r][m]
    float* const pw = (float*)(smem + S::PW);   // a^0 .. a^C
    const int tid = threadIdx.x;
    const ScanArgs& a = all.s[blockIdx.x % all.n];
    const unsigned cta = blockIdx.x / all.n;
    const int hv = cta % a.HV;
    const int64_t item = cta / a.HV;
    int64_t n, p, bos, eos;
    if (!locate<NTHR>(a, item, (int64_t*)(smem + S::RED), n, p, bos, eos)) return;
    const int64_t len = eos - bos, chunks = (len + C - 1) / C;
    const int64_t pieces = chunks > 0 ? (chunks + a.piece_chunks - 1) / a.piece_chunks : 1;
    const bool last = a.reverse ? p == 0 : p == pieces - 1;   // the piece that leaves the sequence
    if (!OUT && last) return;
    const int64_t ch_lo = p * a.piece_chunks;
    const int64_t ch_hi = ch_lo + a.piece_chunks < chunks ? ch_lo + a.piece_chunks : chunks;
    const int nch = (int)(ch_hi - ch_lo);
    const int cw = a.DC;
    const float g = decay_exponent(a.log_decay, hv);
    if (tid <= C) pw[tid] = expf(g * tid);
    if (a.DB < DB || cw < CW)  // columns past the row sizes stay zero
        for (int e = tid; e < (int)(2 * S::STAGE / 4); e += NTHR) ((uint32_t*)smem)[e] = 0;
    __syncthreads();

    const int hA = hv / a.gA, hB = hv / a.gB, hC = hv / a.gC;
    const int nA = a.HV / a.gA, nB = a.HV / a.gB, nC = a.HV / a.gC;
    auto chunk_tok = [&](int c) { return bos + (a.reverse ? ch_hi - 1 - c : ch_lo + c) * C; };
    auto fetch = [&](int c) {  // chunk c into stage c & 1
        const int64_t t0 = chunk_tok(c);
        const int nv = eos - t0 < C ? (int)(eos - t0) : C;
        uint8_t* const st = smem + (c & 1) * S::STAGE;
        auto rows = [&](uint32_t off, int stride, const void* src, int64_t row, int64_t step, int d) {
            const TA* const from = (const TA*)src + row;
            TA* const to = (TA*)(st + off);
            if (vec) {
                constexpr int V = 16 / (int)sizeof(TA);
                const int q = d / V;
                for (int e = tid; e < C * q; e += NTHR) {
                    const int r = e / q, x = (e - r * q) * V;
                    copy16(sm100::smem_u32(to + r * stride + x), from + (r < nv ? r : 0) * step + x, r < nv);
                }
            } else {
                for (int e = tid; e < C * d; e += NTHR) {
                    const int r = e / d, x = e - r * d;
                    float y = 0.f;
                    if (r < nv) y = ld(from, r * step + x);
                    gdn::st(to, r * stride + x, y);
                }
            }
        };
        if (OUT) rows(S::A, S::RS, a.A, (t0 * nA + hA) * a.DB, (int64_t)nA * a.DB, a.DB);
        rows(S::B, S::RS, a.B, (t0 * nB + hB) * a.DB, (int64_t)nB * a.DB, a.DB);
        rows(S::Ct, S::CS, a.C, (t0 * nC + hC) * a.DC, (int64_t)nC * a.DC, cw);
    };
    if (nch > 0) fetch(0);
    asm volatile("cp.async.commit_group;" ::: "memory");

    constexpr bool EX = sizeof(TA) == 2;
    const int warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tq = lane & 3;
    // the state: 16 rows from xr, NT tiles of 8 columns from xc
    constexpr int MT = DB / 16, NT = CW / 8 / (8 / MT);
    const int xr = (warp % MT) * 16, xc = (warp / MT) * NT * 8;
    float X[NT][4];
    const int64_t xbase = (n * a.HV + hv) * (int64_t)a.DB * a.DC;
    auto x_at = [&](int r, int c) { return xbase + (a.transposed ? (int64_t)c * a.DB + r : (int64_t)r * a.DC + c); };
    const int64_t order = a.reverse ? pieces - 1 - p : p;  // in scan order; only x0 reaches the first
    const int64_t slot = state_slot(a, n, item - p, OUT ? order - 1 : order);
    const bool joined = OUT && order > 0;
    const float* const from = !OUT ? nullptr : joined ? a.local + (slot * a.HV + hv) * (int64_t)a.DB * a.DC : a.x0;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = xr + gr + 8 * (e >> 1), x = xc + 8 * i + 2 * tq + (e & 1);
            X[i][e] = from && r < a.DB && x < cw ? from[joined ? (int64_t)r * a.DC + x : x_at(r, x)] : 0.f;
        }
    // outputs: 16 rows from orw, OT tiles of 8 columns from oc; P: 16 rows from orw, 8 columns from 8 (warp / 2)
    constexpr int OT = CW / 32;
    const int orw = (warp & 1) * 16, oc = (warp >> 1) * OT * 8, pc = (warp >> 1) * 8;

    for (int c = 0; c < nch; ++c) {
        const int64_t t0 = chunk_tok(c);
        const int nv = eos - t0 < C ? (int)(eos - t0) : C;
        const uint8_t* const st = smem + (c & 1) * S::STAGE;
        const TA* const sA = (const TA*)(st + S::A);
        const TA* const sB = (const TA*)(st + S::B);
        const TA* const sC = (const TA*)(st + S::Ct);
        if (OUT) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; e += 2)
                    *(float2*)&sX[(xr + gr + 4 * e) * S::XS + xc + 8 * i + 2 * tq] = make_float2(X[i][e], X[i][e + 1]);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // this chunk and the state are there, and the other stage has been read
        if (c + 1 < nch) fetch(c + 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (OUT) {
            float O[OT][4] = {}, Ox[OT][4] = {}, P[4] = {}, Px[4] = {};  // the second: cross terms
#pragma unroll 2
            for (int k = 0; k < DB; k += 8) {
                const TA* const x = sA + (orw + gr) * S::RS + k + tq;
                const Split<EX> fa[4] = {Split<EX>(ld(x, 0)), Split<EX>(ld(x, 8 * S::RS)), Split<EX>(ld(x, 4)),
                                         Split<EX>(ld(x, 8 * S::RS + 4))};
                const TA* const y = sB + (pc + gr) * S::RS + k + tq;
                const Split<EX> fb[2] = {Split<EX>(ld(y, 0)), Split<EX>(ld(y, 4))};
                mma_step(P, Px, fa, fb);
#pragma unroll
                for (int i = 0; i < OT; ++i) {
                    const float* const z = sX + (k + tq) * S::XS + oc + 8 * i + gr;
                    const Split<false> fx[2] = {Split<false>(z[0]), Split<false>(z[4 * S::XS])};
                    mma_step(O[i], Ox[i], fa, fx);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = orw + gr + 8 * (e >> 1), m = pc + 2 * tq + (e & 1), dist = a.reverse ? m - r : r - m;
                sP[r * PS + m] = dist >= 0 ? (P[e] + Px[e]) * a.sp * pw[dist] : 0.f;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = orw + gr + 8 * h;
                const float f = r < nv ? a.si * pw[a.reverse ? nv - 1 - r : r + 1] : 0.f;
#pragma unroll
                for (int i = 0; i < OT; ++i) {
                    O[i][2 * h] *= f;
                    O[i][2 * h + 1] *= f;
                    Ox[i][2 * h] *= f;
                    Ox[i][2 * h + 1] *= f;
                }
            }
            __syncthreads();  // P is there
            // the columns of P that these 16 rows see
            const int m0 = a.reverse ? orw : 0, m1 = a.reverse ? C : orw + 16;
#pragma unroll 2
            for (int k = m0; k < m1; k += 8) {
                const float* const x = sP + (orw + gr) * PS + k + tq;
                const Split<false> fp[4] = {Split<false>(x[0]), Split<false>(x[8 * PS]), Split<false>(x[4]),
                                            Split<false>(x[8 * PS + 4])};
#pragma unroll
                for (int i = 0; i < OT; ++i) {
                    const TA* const z = sC + (k + tq) * S::CS + oc + 8 * i + gr;
                    const Split<EX> fc[2] = {Split<EX>(ld(z, 0)), Split<EX>(ld(z, 4 * S::CS))};
                    mma_step(O[i], Ox[i], fp, fc);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = orw + gr + 8 * h;
                if (r >= nv) continue;
                const int64_t o = ((t0 + r) * a.HV + hv) * a.DC;
#pragma unroll
                for (int i = 0; i < OT; ++i) {
                    const int x = oc + 8 * i + 2 * tq;
                    const float y[2] = {O[i][2 * h] + Ox[i][2 * h], O[i][2 * h + 1] + Ox[i][2 * h + 1]};
                    if (vec && x < cw) {  // whole pairs
                        if (a.out_fp32) *(float2*)((float*)a.out + o + x) = make_float2(y[0], y[1]);
                        else stv<TA, 2>(a.out, o + x, y);
                    } else {
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (x + e < cw) {
                                if (a.out_fp32) ((float*)a.out)[o + x + e] = y[e];
                                else gdn::st((TA*)a.out, o + x + e, y[e]);
                            }
                    }
                }
            }
        }
        // X <- a^nv X + U, U summed apart: over a long sequence the MMAs' dropped bits would add up in X itself
        const float f = pw[nv];
        Split<false> fb[C / 8][4];
#pragma unroll
        for (int k = 0; k < C / 8; ++k) {  // rows past the end are zeros
            const int m = 8 * k + tq, e0 = a.reverse ? m + 1 : nv - 1 - m, e1 = a.reverse ? e0 + 4 : e0 - 4;
            const float w0 = e0 >= 0 && e0 <= C ? a.su * pw[e0] : 0.f, w1 = e1 >= 0 && e1 <= C ? a.su * pw[e1] : 0.f;
            const TA* const x = sB + m * S::RS + xr + gr;
            fb[k][0] = Split<false>(ld(x, 0) * w0);
            fb[k][1] = Split<false>(ld(x, 8) * w0);
            fb[k][2] = Split<false>(ld(x, 4 * S::RS) * w1);
            fb[k][3] = Split<false>(ld(x, 4 * S::RS + 8) * w1);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            float U[4] = {}, Ux[4] = {};
#pragma unroll
            for (int k = 0; k < C / 8; ++k) {
                const TA* const z = sC + (8 * k + tq) * S::CS + xc + 8 * i + gr;
                const Split<EX> fc[2] = {Split<EX>(ld(z, 0)), Split<EX>(ld(z, 4 * S::CS))};
                mma_step(U, Ux, fb[k], fc);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) X[i][e] = fmaf(f, X[i][e], U[e] + Ux[e]);
        }
        __syncthreads();  // sX and P have been read
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    float* dst = OUT ? (last ? a.x1 : nullptr) : a.local;
    if (!dst) return;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = xr + gr + 8 * (e >> 1), x = xc + 8 * i + 2 * tq + (e & 1);
            if (r < a.DB && x < cw) {
                if (OUT) dst[x_at(r, x)] = X[i][e];
                else dst[(slot * a.HV + hv) * (int64_t)a.DB * a.DC + (int64_t)r * a.DC + x] = X[i][e];
            }
        }
}

template <typename TA, int DB, int CW, bool OUT>
static int launch_fp32(const Scans& b, cudaStream_t s) {
    constexpr int smem = (int)sk::Smem<TA, DB, CW>::BYTES;
    const void* k = (const void*)linear_attn_fp32_kernel<TA, DB, CW, OUT>;
    if (smem_optin(k, smem) != cudaSuccess) return GDN_ERR_LAUNCH;
    const ScanArgs& a = b.s[0];
    constexpr int V = 16 / (int)sizeof(TA);  // whole vectors in every row (bases are 16-byte aligned)
    const int vec = a.DB % V == 0 && a.DC % V == 0 ? 1 : 0;
    linear_attn_fp32_kernel<TA, DB, CW, OUT><<<(unsigned)(a.items * a.HV * b.n), sk::NTHR, smem, s>>>(b, vec);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

template <typename TA, int DB, int CW>
static int fp32_mode(const Scans& b, cudaStream_t s) {
    return b.s[0].states_only ? launch_fp32<TA, DB, CW, false>(b, s) : launch_fp32<TA, DB, CW, true>(b, s);
}

template <typename TA>
static int fp32_typed(const Scans& b, cudaStream_t s) {
    if (b.s[0].DB <= 64) return b.s[0].DC <= 64 ? fp32_mode<TA, 64, 64>(b, s) : fp32_mode<TA, 64, 128>(b, s);
    return b.s[0].DC <= 64 ? fp32_mode<TA, 128, 64>(b, s) : fp32_mode<TA, 128, 128>(b, s);
}

int scan_fp32(const Scans& b, int act_dtype, cudaStream_t s) {
    if (b.s[0].items * b.s[0].HV * b.n > 0x7fffffff) return GDN_ERR_SHAPE;
    switch (act_dtype) {
        case GDN_BF16: return fp32_typed<__nv_bfloat16>(b, s);
        case GDN_FP16: return fp32_typed<__half>(b, s);
        case GDN_FP32: return fp32_typed<float>(b, s);
        default: return GDN_ERR_DTYPE;
    }
}

}  // namespace linattn
}  // namespace gdn
