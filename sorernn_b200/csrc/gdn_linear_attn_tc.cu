// The linear-attention scan (linear_attn.cuh) on the tensor cores: bf16 activations, head sizes 64 and 128.
//
// One CTA per (value head, piece), 128 tokens a chunk. Per chunk, with A, B, C the roles' tiles and X the state:
//   P  = A B^T                       (M = 128 tokens, N = 128 tokens, K = DB)
//   Oi = A (Xhi + Xlo)               (K = DB; X split into two bf16)
//   U^T = C^T (hi + lo)              (M = DC, N = DB, K = 128 tokens; hi + lo = su a^(..) B split into two bf16)
//   Oa = (Whi + Wlo) C               (W(P): in-chunk decay, mask and scale, split into two bf16 in tensor memory)
//   out = Oa + si a^(..) Oi          one rounding
//   X <- a^nv X + U                  (fp32, in registers)
// A, B and C are exact; the two-term splits of X, of W(P) and of the state's operand are good to 2^-17, so outputs are
// within 2e-4 of RMS of their own rounding however slowly a head decays (X in one term left up to 0.018 of RMS more; its
// second term costs the seventh product, a scan of the shape below 121 -> 141 us). A caller that gets the state itself
// (final state, gradient of the initial state) has its operand split in three (`precise`): fp32 accuracy. Two terms of a
// 128 x 128 X do not fit beside the other tiles: its halves along DB, 32 KB of both terms, take turns in one place (the
// staging tile in its stead, with outputs stored directly, made that 158 us).
//
// Keeping X in registers and U in an accumulator of its own takes the state off the tensor pipe's critical path: U of
// a chunk needs nothing of the chunk before. 20 warps, handed over by mbarriers with bounded waits:
//   warps 0-7    W(P), then the outputs: thread = token row, warps 4-7 the upper half of the columns. Every weight
//                from registers; a masked value (NaN or not) is selected away, never multiplied. The outputs leave
//                through shared memory and a bulk store (a warp's direct 16-byte stores touch 32 lines each)
//   warps 8-11   hi and lo of B
//   warps 12-15  the state: thread = a row of X^T, 128 fp32 registers (registers moved here with setmaxnreg)
//   warps 16, 18, 19  issue the MMAs (P and Oa; U; Oi), each in uniform control flow with the issue predicated
//   warp 17      issues the loads (single buffers; L2 prefetch two chunks ahead)
// 8 x 4,096 tokens x 16 heads, DB = DC = 128: a scan takes 147 us, 4.6 us a chunk, 0.56 of a copy's rate over the four
// tensors that it reads and writes; bound by the chain of hand-overs between the roles (tensor pipe 0.44 busy). The
// fp32-accuracy kernel (gdn_linear_attn_fp32.cu) takes 903 us (64 features: 417 against 97; one chunk of 16 heads: 34
// against 8), so bf16 runs here at every size that this one supports. The states-only form runs the split,
// its product and the accumulator in two buffers each and loads B a whole chunk ahead: 2.1 us a chunk (159 us for the pieces
// of 65,536 tokens x 16 heads with one buffer and half a chunk ahead, 124 so). What decided the layout with outputs,
// measured in the shape above (forward):
//   * each role runs its code once a chunk, so the chunk loops have to fit the instruction cache together: 168 KB of
//     unrolled code 12,800 cycles a chunk, 89 KB 6,900 (X in one term; with two, a forward and backward took
//     787 us with 100 KB, the terms written in two passes, and 670 with 90, the halves in turn);
//   * an M = N = 128 product with both operands in shared memory takes nearly all of its read bandwidth (one every 65
//     cycles): beside it a shared load of a warp's 512 bytes takes 60 cycles, a store 7, a global load 8. So the split
//     reads B from global memory (L2) and the weights stay in registers.
// Rows past a sequence's end are zeros in hi, lo, W(P) and C, so that whatever follows in memory (another document)
// reaches nothing.
#include <limits.h>

#include "linear_attn.cuh"
#include "launch.h"
#include "sm100.cuh"
#include "tmap.h"

namespace gdn {
namespace linattn {
using namespace sm100;

// Device error word of this file's kernels (a wait that gave up); read and cleared by read_clear_linear_attn_error().
static __device__ int g_linear_attn_err;

namespace tk {
constexpr int NTHR = 20 * 32;
constexpr int C = 128;  // tokens per chunk
// Registers: 96 a thread at launch (five warpgroups: 480), moved to the roles that need them where there are outputs (the
// outputs' role has two warpgroups); the sum stays 480.
constexpr int REG_OUT = 104, REG_SPLIT = 80, REG_STATE = 160, REG_ISSUE = 32;
static_assert(2 * REG_OUT + REG_SPLIT + REG_STATE + REG_ISSUE == 5 * 96, "register split");
constexpr uint32_t T_P = 0, T_U = 128, T_OI = 256, T_OA = 384, T_COLS = 512;  // TMEM columns
constexpr uint32_t BLK = C * 128;  // bytes of a 64-feature block of a tile

// What a CTA works on. Kept in shared memory, so that each role loads what it needs into its own registers.
struct alignas(16) Info {
    int n, bos, eos;          // sequence, its first token, the token past its end
    int n_precise;            // a chunk's split takes a third term where fewer tokens than this follow in scan order
    int tok_first, tok_step;  // first token of the first chunk in scan order; from chunk to chunk
    int nch, n_u;             // chunks; chunks whose U is formed
    int last, has_x;          // the piece that leaves the sequence; a state comes in
    int slot;                 // place in `local` of that state (-1: it is x0's), or (without outputs) of this piece's own
    uint32_t tm;              // tensor memory
    int failed;               // a warp of the outputs' role gave up
};

template <int DB, int DC, bool OUT>
struct Smem {
    static constexpr uint32_t TB = DB / 64 * BLK, TC = DC / 64 * BLK;
    static constexpr uint32_t B = 0;
    static constexpr uint32_t Ct = B + (OUT ? TB : 0);  // two buffers when only the states are wanted
    static constexpr uint32_t NC = OUT ? 1 : 2;
    static constexpr uint32_t HI = Ct + NC * TC;
    static constexpr uint32_t LO = HI + TB;
    static constexpr uint32_t NS = NC;  // buffers of the split's first two terms
    static constexpr uint32_t LO2 = HI + NS * 2 * TB;  // third term of a precise split, else the output's staging tile
    static constexpr uint32_t ST = LO2;
    static constexpr uint32_t A = LO2 + (TB > TC ? TB : TC);
    // X^T: per 64 columns of DB a block [DC rows][64] of the high terms and one of the low ones; where there is room for
    // 64 columns only (128 by 128 features), the two halves in turn in the same place
    static constexpr uint32_t X = A + (OUT ? TB : 0);
    static constexpr uint32_t BX = DC * 128;
    static constexpr bool TURNS = DB == 128 && DC == 128;
    static constexpr uint32_t NX = TURNS ? 2 : DB / 64 * 2;  // blocks
    static constexpr uint32_t TAB = X + (OUT ? NX * BX : 0);
    static constexpr uint32_t BAR = TAB + 132 * 4;
    static constexpr uint32_t INFO = BAR + 20 * 8;  // NBAR barriers
    static constexpr uint32_t RED = INFO + sizeof(Info);
    static constexpr uint32_t END = RED + (NTHR / 32 + 3) * 8;
    static_assert(TAB % 16 == 0 && BAR % 8 == 0 && INFO % 16 == 0 && RED % 8 == 0, "alignment of the blocks' parts");
    // more than half of an SM's shared memory, so that one CTA holds the SM's tensor memory
    static constexpr uint32_t BYTES = (END > 120 * 1024 ? END : 120 * 1024) + 1024;
};
static_assert(Smem<128, 128, true>::BYTES <= 232448 && Smem<128, 128, false>::BYTES <= 232448, "shared memory budget");

// XR: X is written, AX: it has been multiplied. Where its halves take turns XR and AH are of the first, X2 and AX of the
// second one.
// D16, D18, D19: all products of an issuing warp are done (once, at its end).
enum Bar { FULL_A, FULL_B, FULL_C0, FULL_C1, QK, U, AX, AH, O, HL, XR, X2, UR, P0, P1, E, D16, D18, D19, NBAR };
static_assert(NBAR <= 20, "barriers");
// Without outputs the split, its product and the product's accumulator have two buffers, and a barrier each, by chunk
enum Bar2 { U_ODD = AX, HL_ODD = XR, UR_ODD = P0 };
}  // namespace tk

struct TcArgs {
    CUtensorMap tA, tB, tC, tO;
    ScanArgs s;
};
struct TcBatch {
    TcArgs t[kMaxScans];
    int n;
};

// The low word of the 128-byte-swizzle descriptors (start, LBO); the high word (SBO 1024, version, swizzle) is the same
// for every operand here, so that stepping an operand is one 32-bit addition.
constexpr uint32_t kDescHigh = (1024 >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lbo) { return saddr >> 4 | (lbo >> 4) << 16; }
// D[tmem] (+)= A * B[smem] where `issue` is non-zero; A in shared memory, or (ta) in tensor memory: bf16 pairs, row =
// lane, K along the columns
__device__ __forceinline__ void mma_if(uint32_t issue, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                       uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "mov.b64 da, {%1, %6};\n\t"
        "mov.b64 db, {%2, %6};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(issue), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void mma_ta_if(uint32_t issue, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                          uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "mov.b64 db, {%2, %6};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(issue), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t issue, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
        "r"(issue)
        : "memory");
}
__device__ __forceinline__ void prefetch_tile_l2(const CUtensorMap* map, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"((uint64_t)map), "r"(c0),
                 "r"(c1), "r"(c2)
                 : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"((uint64_t)map),
                 "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}
// Barriers by their shared-memory address (a handful of instructions a use: see the note on the instruction cache).
// A bounded wait: `left` polls remain to the thread (a poll that fails suspends for microseconds, so the budget is
// about a second, where a chunk takes four microseconds); once they are spent, `left` stays 1 and every later wait looks
// once. A warp that gave up hands over and stores nothing from then on, nor writes what a product or a copy may still read:
// the roles end their loops, but for the outputs' one, which meets in named barriers and runs out. So the others give up in
// their turn, no barrier gets an arrival that it does not expect, and what reaches memory was made from complete operands.
// The warps that issue loads and products wait for theirs before the CTA gives its memory back.
constexpr uint32_t kPolls = 1u << 19;
__device__ __forceinline__ void wait_at(uint32_t bar, uint32_t parity, uint32_t& left) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "again:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "@p bra done;\n\t"
        "add.u32 %0, %0, -1;\n\t"
        "setp.ne.u32 p, %0, 0;\n\t"
        "@p bra again;\n\t"
        "mov.u32 %0, 1;\n\t"
        "done:\n\t}"
        : "+r"(left)
        : "r"(bar), "r"(parity)
        : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void expect_at(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
        "[%2];" ::"r"(dst),
        "l"((uint64_t)map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
// 32 bytes to global memory, in one store where they are aligned to that: a whole sector per thread, where two 16-byte
// stores write it by halves
__device__ __forceinline__ void put8(void* p, const uint32_t* w, bool wide) {
    if (wide) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
                     "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                     : "memory");
    } else {
        reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 h) { return *reinterpret_cast<uint32_t*>(&h); }
template <int N> __device__ __forceinline__ void set_regs() {
    if constexpr (N > 96) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    if constexpr (N < 96) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// BATCH: several scans in the launch. Apart, because scans picked by index cost the forward's one scan 5-10 %.
template <int DB, int DC, bool OUT, bool PRECISE, bool BATCH>
__global__ void __launch_bounds__(tk::NTHR, 1) linear_attn_tc_kernel(const __grid_constant__ TcBatch all) {
    using namespace tk;
    using S = Smem<DB, DC, OUT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const TcArgs& args = all.t[BATCH ? blockIdx.x % all.n : 0];
    const unsigned cta = BATCH ? blockIdx.x / all.n : blockIdx.x;
    const ScanArgs& a = args.s;
    float* pw = (float*)(sm + S::TAB);  // a^0 .. a^128
    uint64_t* bar = (uint64_t*)(sm + S::BAR);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

    const int hv = cta % a.HV;
    Info* const info = (Info*)(sm + S::INFO);
    {
        const int64_t item = cta / a.HV;
        int64_t n, p64, bos64, eos64;
        if (!locate<NTHR>(a, item, (int64_t*)(sm + S::RED), n, p64, bos64, eos64)) return;
        // token and chunk numbers fit 32 bits (checked on the host)
        const int p = (int)p64, bos = (int)bos64, eos = (int)eos64, len = eos - bos, chunks = (len + C - 1) / C;
        const int pieces = chunks > 0 ? (chunks + a.piece_chunks - 1) / a.piece_chunks : 1;
        const bool last = a.reverse ? p == 0 : p == pieces - 1;
        if (!OUT && last && !a.end_in_join) return;
        if (tid == 0) {
            const int ch_lo = p * a.piece_chunks, ch_hi = min(ch_lo + a.piece_chunks, chunks), nch = ch_hi - ch_lo;
            info->n = (int)n;
            info->bos = bos;
            info->eos = eos;
            // Two terms leave 2^-18 of a chunk's share; where that share has decayed to 1/64 at the end of the sequence
            // it no longer shows in the end state at fp32 accuracy, so only the chunks after that take the third.
            const float g = decay_exponent(a.log_decay, hv);
            info->n_precise = BATCH && !a.precise ? INT_MIN : g > -1e-6f ? INT_MAX : (int)fminf(4.16f / -g, 2e9f);
            info->tok_first = bos + (a.reverse ? ch_hi - 1 : ch_lo) * C;
            info->tok_step = a.reverse ? -C : C;
            info->nch = nch;
            info->n_u = !OUT || (last && a.x1) ? nch : nch - 1;  // the last chunk's only if its end state is wanted
            info->last = last;
            info->failed = 0;
            const int order = a.reverse ? pieces - 1 - p : p;  // in scan order; only x0 reaches the first
            info->has_x = OUT && (order > 0 || a.x0);
            info->slot = OUT && order == 0 ? -1 : (int)state_slot(a, n, item - p, order - (OUT ? 1 : 0));
        }
    }
    if (tid == 16 * 32) {
        for (int i = 0; i < NBAR; ++i) mbar_init(&bar[i], i >= D16 ? 1 : i >= P0 || (!OUT && i >= HL) ? 8 : i >= HL ? 4 : 1);
        fence_barrier_init();
    }
    if (tid == 17 * 32) {
        if (OUT) prefetch_tmap(&args.tA);
        prefetch_tmap(&args.tB);
        prefetch_tmap(&args.tC);
    }
    if (warp == 0) tmem_alloc(&info->tm, T_COLS);
    const float g = decay_exponent(a.log_decay, hv);
    if (tid <= C) pw[tid] = expf(g * tid);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t sb = smem_u32(sm);
    const uint32_t bars = sb + S::BAR;
    uint32_t polls = kPolls;
    auto at = [&](int b) { return bars + b * 8; };
    auto wait = [&](int b, uint32_t parity) { wait_at(at(b), parity & 1u, polls); };
    // the hand-overs split -> U -> state: of chunk c (two buffers without outputs, so two barriers)
    auto wait_hl = [&](int c) { OUT ? wait(HL, c) : wait(c & 1 ? HL_ODD : HL, c >> 1); };
    auto wait_u = [&](int c) { OUT ? wait(U, c) : wait(c & 1 ? U_ODD : U, c >> 1); };
    auto wait_ur = [&](int c) { OUT ? wait(UR, c) : wait(c & 1 ? UR_ODD : UR, c >> 1); };
    auto odd = [&](int c) { return OUT ? 0u : (uint32_t)c & 1u; };
    constexpr int AHEAD = S::NS;  // buffers of those three
    auto wait_c = [&](int c) { wait(FULL_C0 + (S::NC == 2 ? c & 1 : 0), S::NC == 2 ? c >> 1 : c); };
    auto gave_up = [&]() { return __any_sync(0xffffffffu, polls == 1) != 0; };
    auto arrive = [&](int b) {
        const bool go = !gave_up();
        __syncwarp();
        if (go && lane == 0) arrive_at(at(b));
    };
    // the end of a warp that issues products: they are done
    auto drain = [&](int b) {
        uint32_t left = kPolls;
        commit_if(lane == 0, at(b));
        wait_at(at(b), 0, left);
        tc_fence_after();
    };
    // whether the chunk that starts at t has its split in three terms (see Info)
    auto precise_at = [&](int t) { return PRECISE && (a.reverse ? t - info->bos : info->eos - t - C) < info->n_precise; };
    // tokens of the c-th chunk in scan order
    auto tokens_at = [&](int t) { return min(info->eos - t, C); };
    // zeros in C's rows past the end, by 128 threads
    auto zero_tail = [&](int c, int nv, int t) {
        wait_c(c);
        if (gave_up()) return;
        uint8_t* ct = sm + S::Ct + (S::NC == 2 ? (c & 1) * S::TC : 0);
        for (int e = nv * 8 + t; e < C * 8; e += 128)
#pragma unroll
            for (int kb = 0; kb < DC / 64; ++kb) *reinterpret_cast<uint4*>(ct + kb * BLK + e * 16) = make_uint4(0, 0, 0, 0);
    };

    if (warp >= 16) {
        if constexpr (OUT) set_regs<REG_ISSUE>();
        if (warp == 17 && lane == 0) {
            const int hA = hv / a.gA, hB = hv / a.gB, hC = hv / a.gC;
            const int nch = info->nch, tok_step = info->tok_step;
            int t = info->tok_first, loaded[3] = {0, 0, 0};  // loads issued of A, B, C
#pragma unroll 1
            for (int c = 0; c < nch; ++c, t += tok_step) {
                auto load = [&](const CUtensorMap* map, uint32_t dst, int b, int h, uint32_t bytes) {
                    expect_at(at(b), bytes);
                    for (uint32_t kb = 0; kb < bytes; kb += BLK)
                        load_tile(sb + dst + kb, map, at(b), (int)(kb / BLK) * 64, h, t);
                };
                if (OUT) {
                    if (c > 0) wait(QK, c - 1);
                    if (polls == 1) break;
                    load(&args.tB, S::B, FULL_B, hB, S::TB);
                    ++loaded[1];
                    if (c > 0) wait(AX, c - 1);
                    if (polls == 1) break;
                    load(&args.tA, S::A, FULL_A, hA, S::TB);
                    ++loaded[0];
                    if (c > 0) {  // U and Oa of chunk c - 1 have read C
                        wait(U, c - 1);
                        wait(O, c - 1);
                    }
                } else if (c > 1) {
                    wait_u(c - 2);  // it has read this buffer of C
                }
                if (polls == 1) break;
                const int cb = S::NC == 2 ? c & 1 : 0;
                load(&args.tC, S::Ct + cb * S::TC, FULL_C0 + cb, hC, S::TC);
                ++loaded[2];
                for (int d = c ? c + 2 : 1; d <= c + 2 && d < nch; ++d)  // to L2, two chunks ahead
                    for (int kb = 0; kb < (DB > DC ? DB : DC); kb += 64) {
                        const int td = t + (d - c) * tok_step;
                        if (OUT && kb < DB) prefetch_tile_l2(&args.tA, kb, hA, td);
                        if (kb < DB) prefetch_tile_l2(&args.tB, kb, hB, td);
                        if (kb < DC) prefetch_tile_l2(&args.tC, kb, hC, td);
                    }
            }
            uint32_t left = kPolls;  // the last load of each barrier has landed
            if (loaded[0] > 0) wait_at(at(FULL_A), (loaded[0] - 1) & 1, left);
            if (loaded[1] > 0) wait_at(at(FULL_B), (loaded[1] - 1) & 1, left);
            for (int b = 0; b < (int)S::NC; ++b) {
                const int n = (loaded[2] + (int)S::NC - 1 - b) / (int)S::NC;
                if (n > 0) wait_at(at(FULL_C0 + b), (n - 1) & 1, left);
            }
        } else if (OUT && warp == 16) {
            const uint32_t one = lane == 0;
            constexpr uint32_t id_p = idesc_bf16(128, 128, 0, 0), id_o = idesc_bf16(128, DC, 0, 1);
            const uint32_t dA = desc_low(sb + S::A, 16), dB = desc_low(sb + S::B, 16), dC = desc_low(sb + S::Ct, BLK);
            const uint32_t tm = info->tm;
            const int nch = info->nch;
#pragma unroll 1
            for (int c = 0; c < nch; ++c) {
                wait(FULL_A, c);
                wait(FULL_B, c);
                if (c > 0) wait(O, c - 1);  // W(P) of chunk c - 1 has been read
                if (gave_up()) break;
                tc_fence_after();
#pragma unroll
                for (int ks = 0; ks < DB / 16; ++ks) {
                    const uint32_t o = ((ks >> 2) * BLK + (ks & 3) * 32) >> 4;
                    mma_if(one, tm + T_P, dA + o, dB + o, id_p, ks);
                }
                commit_if(one, at(QK));
                wait_c(c);
                if (c > 0) wait(E, c - 1);  // the outputs of chunk c - 1 have left Oa
#pragma unroll 1
                for (uint32_t half = 0; half < 2; ++half) {
                    wait(half ? P1 : P0, c);
                    if (gave_up()) break;
                    tc_fence_after();
#pragma unroll 1
                    for (uint32_t lo = 0; lo < 2; ++lo) {
                        const uint32_t tw = tm + T_P + half * 64 + lo * 8, d = dC + half * (8192 >> 4);
#pragma unroll
                        for (uint32_t ks = 0; ks < 4; ++ks)
                            mma_ta_if(one, tm + T_OA, tw + ks * 16, d + ks * (2048 >> 4), id_o,
                                      half | lo | ks);
                    }
                }
                if (gave_up()) break;
                commit_if(one, at(O));
            }
            drain(D16);
        } else if (warp == 18) {
            const uint32_t one = lane == 0;
            constexpr uint32_t id_u = idesc_bf16(128, DB, 1, 1);
            const uint32_t dH = desc_low(sb + S::HI, BLK);  // LO follows
            // 64 state rows: the second half of the M = 128 rows reads the first block again, its results are not used
            const uint32_t dCm = desc_low(sb + S::Ct, DC == 128 ? BLK : 0);
            const uint32_t tm = info->tm;
            const int nch = info->nch, n_u = info->n_u, tok_step = info->tok_step;
            int t = info->tok_first;
#pragma unroll 1
            for (int c = 0; c < nch; ++c, t += tok_step) {
                wait_c(c);
                wait_hl(c);
                if (c >= AHEAD) wait_ur(c - AHEAD);
                if (gave_up()) break;
                if (c < n_u) {
                    tc_fence_after();
                    const uint32_t terms = precise_at(t) ? 3 : 2;
                    const uint32_t dC = dCm + (S::NC == 2 ? (c & 1) * (S::TC >> 4) : 0);
#pragma unroll 1
                    for (uint32_t term = 0; term < terms; ++term) {
                        const uint32_t dT = dH + (term == 2 ? (S::LO2 - S::HI) >> 4 : (2 * odd(c) + term) * (S::TB >> 4));
#pragma unroll
                        for (uint32_t ks = 0; ks < 8; ++ks)
                            mma_if(one, tm + (odd(c) ? T_P : T_U), dC + ks * (2048 >> 4), dT + ks * (2048 >> 4), id_u,
                                   term | ks);
                    }
                }
                commit_if(one, at(odd(c) ? (int)U_ODD : (int)U));
            }
            drain(D18);
        } else if (OUT && warp == 19) {
            const uint32_t one = lane == 0;
            constexpr uint32_t id_x = idesc_bf16(128, DC, 0, 0);
            const uint32_t dA = desc_low(sb + S::A, 16), dX = desc_low(sb + S::X, 16);
            const uint32_t tm = info->tm;
            const int nch = info->nch;
            const bool has_x = info->has_x;
#pragma unroll 1
            for (int c = 0; c < nch; ++c) {
                wait(FULL_A, c);  // every phase in turn, also where nothing is issued
                wait(XR, c);
                if (c > 0) wait(E, c - 1);  // the outputs of chunk c - 1 have left Oi
#pragma unroll 1
                for (uint32_t half = 0; half < DB / 64; ++half) {
                    if (S::TURNS && half) {
                        commit_if(one, at(AH));
                        wait(X2, c);
                    }
                    if (gave_up()) break;
                    if (c == 0 && !has_x) continue;
                    tc_fence_after();
#pragma unroll 1
                    for (uint32_t term = 0; term < 2; ++term) {
                        const uint32_t da = dA + half * (BLK >> 4);
                        const uint32_t d = dX + ((S::TURNS ? 0 : half * 2) + term) * (S::BX >> 4);
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            mma_if(one, tm + T_OI, da + ks * 2, d + ks * 2, id_x, half | term | ks);
                    }
                }
                if (gave_up()) break;
                commit_if(one, at(AX));
            }
            drain(D19);
        }
    } else if (OUT ? warp >= 12 : warp < 8) {
        // ---- the state ----
        if constexpr (OUT) set_regs<REG_STATE>();
        // with outputs warps 12-15, a whole row each; without, the warps that then have nothing else, half a row each
        constexpr int XC = OUT ? DB : DB / 2;
        const int row = tid & 127, x0c = OUT ? 0 : (warp >> 2) * XC;  // feature of C; first column
        const bool live = row < DC;
        const uint32_t lb = (uint32_t)(row & 96) << 16;
        float2 x[XC / 2];
        const int64_t xrow = ((int64_t)info->n * a.HV + hv) * (int64_t)DB * DC;               // of x0 and x1
        const int64_t lrow = ((int64_t)info->slot * a.HV + hv) * DB * DC + x0c * DC + row;  // in `local`
        const bool from = OUT && info->has_x && live;
        const bool given = info->slot < 0;
        const float* const src = given ? a.x0 + xrow + (a.transposed ? row * DB : row) : a.local + lrow;
#pragma unroll
        for (int j = 0; j < XC / 2; ++j) x[j] = make_float2(0.f, 0.f);
        if (from && given && a.transposed) {  // a thread's row is contiguous: by 16 bytes
#pragma unroll
            for (int j = 0; j < XC; j += 4) {
                const float4 y = *reinterpret_cast<const float4*>(src + j);
                x[j / 2] = make_float2(y.x, y.y);
                x[j / 2 + 1] = make_float2(y.z, y.w);
            }
        } else if (from) {  // column by column, a warp's threads side by side
#pragma unroll
            for (int j = 0; j < XC; j += 2) x[j / 2] = make_float2(src[j * DC], src[(j + 1) * DC]);
        }
        auto write_x = [&](int c) {  // X^T: row = feature of C, DB along the row
#pragma unroll
            for (int j = 0; j < DB; j += 8) {
                if (S::TURNS && j == 64) {
                    fence_async_smem();
                    arrive(XR);
                    wait(AH, c);
                    if (gave_up()) return;
                }
                if (live) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 y = x[(j / 2 + k) % (XC / 2)];
                        hi[k] = pack2(y.x, y.y);
                        lo[k] = pack2(y.x - lo_f(hi[k]), y.y - hi_f(hi[k]));
                    }
                    uint8_t* const dst = sm + S::X + (S::TURNS ? 0 : (j >> 6) * 2) * S::BX + row * 128 +
                                         (((j >> 3) ^ row) & 7) * 16;
                    *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4*>(dst + S::BX) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            }
            fence_async_smem();
            arrive(S::TURNS ? X2 : XR);
        };
        const int nch = info->nch, n_u = info->n_u;
        const uint32_t tu0 = info->tm + lb + x0c;
#pragma unroll 1
        for (int c = -1; c < n_u; ++c) {  // c = -1: the state that reaches the first chunk
            if (c >= 0) {
                const float f = pw[tokens_at(info->tok_first + c * info->tok_step)];
                const uint32_t tu = tu0 + (odd(c) ? T_P : T_U);
                wait_u(c);
                if (gave_up()) break;
                tc_fence_after();
#pragma unroll
                for (int j = 0; j < XC; j += 16) {
                    float u[16];
                    tmem_ld16(tu + j, u);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; k += 2)
                        x[(j + k) / 2] = fma2(make_float2(f, f), x[(j + k) / 2], make_float2(u[k], u[k + 1]));
                }
                tc_fence_before();
                arrive(odd(c) ? (int)UR_ODD : (int)UR);
            }
            if (OUT && c + 1 < nch) {
                if (c >= 0) wait(AX, c);  // X of this chunk has been read
                if (gave_up()) break;
                write_x(c + 1);
            }
        }
        float* dst = OUT ? (info->last ? a.x1 : nullptr) : a.local;
        if (gave_up()) dst = nullptr;
        if (dst && live) {
            dst += OUT ? xrow + row : lrow;  // x1 is never transposed
#pragma unroll
            for (int j = 0; j < XC; j += 2) {
                dst[j * DC] = x[j / 2].x;
                dst[(j + 1) * DC] = x[j / 2].y;
            }
        }
    } else if (warp >= 8) {
        // ---- hi and lo of B ----
        if constexpr (OUT) set_regs<REG_SPLIT>();
        // B comes from global memory (L2, after the bulk load's prefetch): beside the products, which take nearly all
        // of the shared memory's read bandwidth, a shared load of 512 bytes was measured at 60 cycles, a global one at 8
        // without outputs warps 8-15, twice as many
        constexpr int CT = OUT ? 128 : 256, RS = CT / 8, NR = C / RS;  // threads; rows apart, and per thread
        const int t4 = tid - 256, r0 = t4 >> 3, ch = t4 & 7;  // rows r0 + RS i, 16-byte chunk of a 64-feature block
        const int64_t bstep = (int64_t)(a.HV / a.gB) * DB;    // from token to token
        const __nv_bfloat16* const b0 = (const __nv_bfloat16*)a.B + hv / a.gB * DB + ch * 8;
        uint8_t* const dst0 = sm + S::HI + r0 * 128 + ((ch ^ (r0 & 7)) << 4);  // r & 7 is the same for all i
        constexpr int DEPTH = OUT ? 1 : 2;  // blocks of 64 features loaded ahead
        uint4 u[DEPTH][NR];
        auto load = [&](const __nv_bfloat16* src, uint4& dst, int i, int rows) {
            dst = r0 + RS * i < rows ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0, 0, 0, 0);
        };
        // the rows' factors, as fp32 (precise) or as a pair of bf16, f = fh + fl
        uint32_t fx[NR];
        int nv = -1;
        bool prec = false, good = true;
        const int nch = info->nch, n_u = info->n_u, tok_first = info->tok_first, tok_step = info->tok_step;
        constexpr int NB = DB / 64;
#pragma unroll 1
        for (int step0 = -DEPTH; step0 < nch * NB; step0 += DEPTH)
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int step = step0 + d;
            if (step >= nch * NB) break;
            const int c = step >= 0 ? step / NB : 0, kb = step & (NB - 1);
            if (step >= 0 && kb == 0) {
                const int tc = tok_first + c * tok_step;
                if (nv != tokens_at(tc) || prec != precise_at(tc)) {
                    nv = tokens_at(tc);
                    prec = precise_at(tc);
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        const int r = r0 + RS * i;
                        const float f = r < nv ? a.su * pw[a.reverse ? r + 1 : nv - 1 - r] : 0.f;
                        const uint32_t h = pack2(f, 0.f);
                        fx[i] = prec ? __float_as_uint(f) : h | pack2(0.f, f - lo_f(h));
                    }
                }
                // the split in this buffer has been read; also keeps HL at most one phase ahead of the MMA warp
                if (c >= AHEAD) wait_u(c - AHEAD);
                if (PRECISE && !OUT && prec && c > 0) wait_u(c - 1);  // the third term has one buffer
                if (!OUT) wait_c(c);  // every phase in turn
                good = !gave_up();
                if (nv < C) zero_tail(c, nv, t4 & 127);
            }
            // each row's registers are loaded again as soon as they are used
            const int next = (step + DEPTH) / NB;
            const int tn = tok_first + next * tok_step, rows = next < n_u ? tokens_at(tn) : 0;
            const __nv_bfloat16* src = b0 + (tn + r0) * bstep + (step + DEPTH) % NB * 64;
            if (c < n_u && good) {
                uint8_t* const dst1 = dst0 + odd(c) * (2 * S::TB) + kb * BLK;
#pragma unroll
                for (int i = 0; i < NR; ++i, src += RS * bstep) {
                    if (step < 0) {
                        load(src, u[d][i], i, rows);
                        continue;
                    }
                    const uint32_t w[4] = {u[d][i].x, u[d][i].y, u[d][i].z, u[d][i].w};
                    uint8_t* const dst = dst1 + i * (RS * 128);
                    uint32_t hi[4], lo[4];
                    if (prec) {
                        const float f = __uint_as_float(fx[i]);
                        uint32_t lo2[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            float y0 = lo_f(w[k]) * f, y1 = hi_f(w[k]) * f;
                            hi[k] = pack2(y0, y1);
                            y0 -= lo_f(hi[k]);
                            y1 -= hi_f(hi[k]);
                            lo[k] = pack2(y0, y1);
                            lo2[k] = pack2(y0 - lo_f(lo[k]), y1 - hi_f(lo[k]));
                        }
                        *reinterpret_cast<uint4*>(dst + (S::LO2 - S::HI) - odd(c) * (2 * S::TB)) =
                            make_uint4(lo2[0], lo2[1], lo2[2], lo2[3]);
                    } else {
                        // in bf16 pairs: hi = round(B fh), lo = round(B fl + (B fh - hi)); B fh - hi is exact
                        const __nv_bfloat162 f = as_bf162(fx[i]), fh = __low2bfloat162(f), fl = __high2bfloat162(f);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const __nv_bfloat162 b = as_bf162(w[k]), h = __hmul2_rn(b, fh);
                            hi[k] = as_u32(h);
                            lo[k] = as_u32(__hfma2(b, fl, __hfma2(b, fh, __hneg2(h))));
                        }
                    }
                    *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4*>(dst + S::TB) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    load(src, u[d][i], i, rows);
                }
            }
            if (step >= 0 && kb == NB - 1) {
                fence_async_smem();
                arrive(odd(c) ? (int)HL_ODD : (int)HL);
            }
        }
    } else {
        // ---- W(P), then the outputs ----
        if constexpr (OUT) set_regs<REG_OUT>();
        if (OUT) {
            const int q = warp & 3, h = warp >> 2, r = 32 * q + lane;
            const uint32_t tm = info->tm + ((uint32_t)(32 * q) << 16);
            const int nch = info->nch, eos = info->eos, tok_step = info->tok_step;
            const bool has_x = info->has_x;
            int t0 = info->tok_first;
            // Weights from registers (see the split on shared loads), for 16 columns at a time as a^(distance of r from
            // the columns' near end) a^(distance within them). On the diagonal the first may be negative, down to -15:
            // a head that decays faster than e^-5 a token, where that could overflow, takes every weight by itself.
            float2 w8[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                w8[k] = a.reverse ? make_float2(pw[2 * k], pw[2 * k + 1]) : make_float2(pw[7 - 2 * k], pw[6 - 2 * k]);
            const float g0 = a.reverse ? 1.f : pw[8], g1 = a.reverse ? pw[8] : 1.f;  // first and second 8 columns of 16
            bool staged = false;
            const bool fast = g >= -5.f, wide = ((uintptr_t)a.out & 31) == 0;
#pragma unroll 1
            for (int c = 0; c < nch; ++c, t0 += tok_step) {
                int nv = min(eos - t0, C);
                const int m_end = a.reverse ? nv : C;  // forward: m <= r < nv leaves the tail out by itself
                // A chunk whose split has a third term keeps it in the staging tile. The last tile before that is given
                // up two chunks ahead, and read out before this chunk's W(P): Oa follows it, then the next chunk's U,
                // and only then the third term is written.
                const bool was_staged = staged;
                staged = !precise_at(t0 + 2 * tok_step) && !a.out_fp32 && nv == C;
                if (PRECISE && was_staged && !staged) {
                    if (tid == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    asm volatile("bar.sync 1, 256;" ::: "memory");
                }
                wait(QK, c);
                if (nv < C) {  // not before QK: it came after Oa of the chunk before, whose C is in the same place
                    zero_tail(c, nv, tid & 127);
                    fence_async_smem();
                }
                tc_fence_after();
                // 16 columns -> 8 columns of hi pairs, 8 of lo pairs; the halves of the warps take turns, so that the
                // first 64 columns are ready half way
                auto masked = [&](int m) { return a.reverse ? (m >> 5) < q : (m >> 5) > q; };  // wholly
                auto weigh = [&](int m, float(&v)[16]) {
                    const uint32_t tp = tm + T_P + m;
                    if (masked(m)) {
#pragma unroll
                        for (int k = 0; k < 16; ++k) v[k] = 0.f;
                        tmem_st16(tp, v);
                        return;
                    }
                    const int d0 = a.reverse ? m - r : r - m;  // distance at the first column, rising or falling by one
                    if (fast || (m >> 5) != q) {
                        const float f = a.sp * __expf(g * (float)(a.reverse ? d0 : d0 - 15));
                        const float z0 = f * g0, z1 = f * g1;
#pragma unroll
                        for (int k = 0; k < 16; k += 2) {
                            const float z = k < 8 ? z0 : z1;
                            const float2 y = mul2(make_float2(v[k], v[k + 1]), mul2(w8[k / 2 % 4], make_float2(z, z)));
                            v[k] = y.x;
                            v[k + 1] = y.y;
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 16; ++k) v[k] *= a.sp * __expf(g * fmaxf((float)(a.reverse ? d0 + k : d0 - k), 0.f));
                    }
                    if ((m >> 5) == q || m + 16 > m_end) {
                        // first and last column that counts (reverse: columns past the end are another document's)
                        const int k0 = a.reverse ? -d0 : 0, k1 = a.reverse ? m_end - m : d0 + 1;
#pragma unroll
                        for (int k = 0; k < 16; ++k) v[k] = k >= k0 && k < k1 ? v[k] : 0.f;
                    }
                    float o[16];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t w = pack2(v[2 * k], v[2 * k + 1]);
                        o[k] = __uint_as_float(w);
                        o[8 + k] = __uint_as_float(pack2(v[2 * k] - lo_f(w), v[2 * k + 1] - hi_f(w)));
                    }
                    tmem_st16(tp, o);
                };
                {
                    const int m = 16 * h;
                    float v0[16], v1[16];
                    tmem_ld16(tm + T_P + m, v0);
#pragma unroll 1
                    for (int half = 0; half < 128; half += 64) {
                        tmem_wait_ld();
                        tmem_ld16(tm + T_P + half + m + 32, v1);
                        weigh(half + m, v0);
                        tmem_wait_ld();
                        if (half == 0) tmem_ld16(tm + T_P + m + 64, v0);
                        weigh(half + m + 32, v1);
                        tmem_wait_st();
                        tc_fence_before();
                        arrive(half ? P1 : P0);
                    }
                }

                const bool inter = c > 0 || has_x;  // without a state Oi holds nothing
                const float f = r < nv ? a.si * __expf(g * (float)(a.reverse ? nv - 1 - r : r + 1)) : 0.f;
                if (staged && c > 0) {  // the bulk store of an earlier chunk has read the staging tile
                    if (tid == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    asm volatile("bar.sync 1, 256;" ::: "memory");
                }
                if (inter) wait(AX, c);
                wait(O, c);
                if (gave_up()) {  // nothing of this chunk is stored, nor of a later one
                    nv = 0;
                    if (lane == 0) info->failed = 1;
                }
                tc_fence_after();
                float x0[16], y0[16];
                tmem_ld16(tm + T_OA + DC / 2 * h, x0);
                tmem_ld16(tm + T_OI + DC / 2 * h, y0);
#pragma unroll 1
                for (int j = DC / 2 * h; j < DC / 2 * (h + 1); j += 16) {
                    float x[16];
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        const float2 z = fma2(make_float2(f, f), make_float2(y0[k], y0[k + 1]),
                                              make_float2(x0[k], x0[k + 1]));
                        x[k] = inter ? z.x : x0[k];
                        x[k + 1] = inter ? z.y : x0[k + 1];
                    }
                    if (j + 16 < DC / 2 * (h + 1)) {
                        tmem_ld16(tm + T_OA + j + 16, x0);
                        tmem_ld16(tm + T_OI + j + 16, y0);
                    } else {
                        tc_fence_before();
                        arrive(E);
                    }
                    const int64_t at = ((int64_t)(t0 + r) * a.HV + hv) * DC + j;
                    if (a.out_fp32) {
                        if (r < nv) {
#pragma unroll
                            for (int k = 0; k < 16; k += 8) put8((float*)a.out + at + k, reinterpret_cast<uint32_t*>(x + k), wide);
                        }
                        continue;
                    }
                    uint32_t w[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) w[k] = pack2(x[2 * k], x[2 * k + 1]);
                    if (staged) {  // 16-byte chunks of the row, swizzled by the row
                        uint8_t* const st = sm + S::ST + (j >> 6) * BLK + r * 128;
                        *reinterpret_cast<uint4*>(st + (((j >> 3) ^ r) & 7) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
                        *reinterpret_cast<uint4*>(st + (((j >> 3) + 1 ^ r) & 7) * 16) = make_uint4(w[4], w[5], w[6], w[7]);
                    } else if (r < nv) {
                        put8((__nv_bfloat16*)a.out + at, w, wide);
                    }
                }
                if (staged) {
                    fence_async_smem();
                    asm volatile("bar.sync 1, 256;" ::: "memory");
                    if (tid == 0 && !*(volatile int*)&info->failed) {
#pragma unroll
                        for (int kb = 0; kb < DC / 64; ++kb)
                            tma_store_3d(&args.tO, sm + S::ST + kb * BLK, kb * 64, hv, t0);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                }
            }
            if (tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
    }
    if (polls == 1) atomicCAS(&g_linear_attn_err, 0, GDN_DEV_ERR_LINEAR_ATTN);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) tmem_dealloc(info->tm, T_COLS);
}

bool scan_tc_supported(int64_t DB, int64_t DC, int act_dtype) {
    return act_dtype == GDN_BF16 && (DB == 64 || DB == 128) && (DC == 64 || DC == 128);
}

template <int DB, int DC, bool OUT, bool PRECISE, bool BATCH>
static int launch_tc(const Scans& b, int64_t tokens, cudaStream_t s) {
    const void* k = (const void*)linear_attn_tc_kernel<DB, DC, OUT, PRECISE, BATCH>;
    constexpr int bytes = (int)tk::Smem<DB, DC, OUT>::BYTES;
    if (smem_optin(k, bytes) != cudaSuccess) return GDN_ERR_LAUNCH;
    TcBatch all{};
    all.n = b.n;
    for (int i = 0; i < b.n; ++i) {
        const ScanArgs& a = b.s[i];
        TcArgs& t = all.t[i];
        t.s = a;
        const int64_t nA = a.HV / a.gA, nB = a.HV / a.gB, nC = a.HV / a.gC;
        if (tokens == 0) continue;
        if (!make_tmap_3d_sw128(&t.tC, a.C, DC, nC, tokens, DC, nC * DC, tk::C)) return GDN_ERR_LAUNCH;
        if (!make_tmap_3d_sw128(&t.tB, a.B, DB, nB, tokens, DB, nB * DB, tk::C)) return GDN_ERR_LAUNCH;
        if (OUT && (!make_tmap_3d_sw128(&t.tA, a.A, DB, nA, tokens, DB, nA * DB, tk::C) ||
                    (!a.out_fp32 &&
                     !make_tmap_3d_sw128(&t.tO, a.out, DC, a.HV, tokens, DC, (uint64_t)a.HV * DC, tk::C))))
            return GDN_ERR_LAUNCH;
    }
    const unsigned grid = (unsigned)(b.s[0].items * b.s[0].HV * b.n);
    linear_attn_tc_kernel<DB, DC, OUT, PRECISE, BATCH><<<grid, tk::NTHR, bytes, s>>>(all);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

// The kernels that can form the third term are apart: the branch alone costs the others a fifth (instruction cache).
template <int DB, int DC, bool OUT>
static int launch_mode(const Scans& b, int64_t tokens, cudaStream_t s) {
    bool precise = false;
    for (int i = 0; i < b.n; ++i) precise = precise || b.s[i].precise;
    if (b.n > 1)
        return precise ? launch_tc<DB, DC, OUT, true, true>(b, tokens, s)
                       : launch_tc<DB, DC, OUT, false, true>(b, tokens, s);
    return precise ? launch_tc<DB, DC, OUT, true, false>(b, tokens, s)
                   : launch_tc<DB, DC, OUT, false, false>(b, tokens, s);
}
template <int DB, int DC>
static int launch_sized(const Scans& b, int64_t tokens, cudaStream_t s) {
    return b.s[0].states_only ? launch_mode<DB, DC, false>(b, tokens, s) : launch_mode<DB, DC, true>(b, tokens, s);
}

int scan_tc(const Scans& b, int64_t tokens, cudaStream_t s) {
    if (b.s[0].items * b.s[0].HV * b.n > 0x7fffffff || tokens > 0x7fffffff) return GDN_ERR_SHAPE;
    if (b.s[0].DB == 128) return b.s[0].DC == 128 ? launch_sized<128, 128>(b, tokens, s) : launch_sized<128, 64>(b, tokens, s);
    return b.s[0].DC == 128 ? launch_sized<64, 128>(b, tokens, s) : launch_sized<64, 64>(b, tokens, s);
}

}  // namespace linattn

int read_clear_linear_attn_error(cudaStream_t s, int* out) {
    static const int zero = 0;
    using linattn::g_linear_attn_err;
    if (cudaMemcpyFromSymbolAsync(out, g_linear_attn_err, sizeof(int), 0, cudaMemcpyDeviceToHost, s) != cudaSuccess ||
        cudaMemcpyToSymbolAsync(g_linear_attn_err, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s) != cudaSuccess)
        return GDN_ERR_LAUNCH;
    return GDN_OK;
}

}  // namespace gdn
