// The scan behind linear attention with a fixed decay per head, shared by its kernels.
//
// With a = exp(log_decay[h]) the forward is S_t = a S_(t-1) + k_t v_t^T, o_t = scale S_t^T q_t. Its gradients, with
// R_t = dL/dS_t = a R_(t+1) + scale q_t do_t^T, are dq_t = scale S_t do_t, dk_t = R_t v_t, dv_t = R_t^T k_t: the same
// scan with its operands exchanged, run backwards in time for dk and dv. So one kernel family takes the roles
//             A (reads)  B, C (make the state)   out   direction   state
//   forward   q          k, v                    o     forward     S   [DK, DV]
//   dq        do         v, k                    dq    forward     S^T [DV, DK]
//   dv        k          q, do                   dv    reverse     R   [DK, DV]
//   dk        v          do, q                   dk    reverse     R^T [DV, DK]
// over chunks of tokens, X the state that reaches the chunk (reverse: the gradient of the state that leaves it),
// rows r, m < nv of the chunk:
//   forward   out_r = sp sum_(m <= r) a^(r-m) (A_r . B_m) C_m + si a^(r+1) X^T A_r
//             X'    = a^nv X + su sum_m a^(nv-1-m) B_m C_m^T
//   reverse   out_r = sp sum_(m >= r) a^(m-r) (A_r . B_m) C_m + si a^(nv-1-r) X^T A_r
//             X'    = a^nv X + su sum_m a^(m+1) B_m C_m^T
// Every exponent of a is >= 0, so nothing overflows for a <= 1 however small a is.
//
// Chunks are counted from a sequence's first token in both directions; its last chunk may be partial. A sequence is
// cut into pieces of `piece_chunks` chunks that run side by side: with more than one piece, a first launch
// (states_only) leaves each piece's own end state (from zero) in `local`, a second joins them along the sequence, so that
// `local` holds the state that reaches the next piece, and the third runs the pieces from there, the first one from x0. The
// end state comes from the third launch, or (end_in_join) from the second. Packed sequences keep no state of their last
// piece in scan order, so that the many of one piece take no memory.
#pragma once
#include "common.cuh"
#include "kernels.h"

namespace gdn {
namespace linattn {

struct ScanArgs {
    const void *A, *B, *C;
    void* out;                // act dtype, or fp32 when out_fp32 (one row per value head, summed over groups later)
    const float* log_decay;   // [HV]
    const float* x0;          // incoming state [N, HV, DK, DV], or NULL
    float* x1;                // outgoing state [N, HV, DK, DV], or NULL
    float* local;             // the pieces' states [state_count(), HV, DB, DC], or NULL (one piece per sequence)
    const int64_t* cu;
    int64_t T, N, items;      // items: (sequence, piece) pairs, with cu an upper bound
    int HV;
    int gA, gB, gC;           // value heads per head of A, B, C (1 or HV / H)
    int DB, DC;               // row sizes: of A and B, of C and out
    int piece_chunks;
    int chunk;                // tokens per chunk
    int reverse, transposed;  // transposed: x0 is stored [DC, DB] (such a scan has no x1)
    int states_only;
    int out_fp32;
    int precise;              // the state itself is wanted (x1): keep it to fp32 accuracy
    int end_in_join;          // cut: the join leaves x1, from every piece's own state; the outputs' launch has no x1
    float sp, si, su;
};

// log_decay clamped so that 0 * x is 0 and not NaN for a decay of exactly zero (log_decay = -inf): a^0 = 1, a^n = 0.
// NaN stays NaN.
__device__ __forceinline__ float decay_exponent(const float* log_decay, int hv) {
    const float g = log_decay[hv];
    return g < -1e4f ? -1e4f : g;
}

// Scans that run in one launch (the backward's three): CTA x belongs to scan x % n, so that the scans of one (value head,
// piece), which read the same tiles, run side by side.
constexpr int kMaxScans = 3;
struct Scans {
    ScanArgs s[kMaxScans];
    int n;
};

// (sequence n, piece p) of a work item; false: an item past the last one. The pieces of sequence n are
// max(1, ceil(len / (chunk * piece_chunks))). Called by all NTHR threads of the block; `red` is shared scratch of
// NTHR / 32 + 3 int64.
template <int NTHR>
__device__ __forceinline__ bool locate(const ScanArgs& a, int64_t item, int64_t* red, int64_t& n, int64_t& p,
                                       int64_t& bos, int64_t& eos) {
    const int64_t per = (int64_t)a.chunk * a.piece_chunks;
    if (!a.cu) {
        const int64_t pps = a.T > 0 ? (a.T + per - 1) / per : 1;
        n = item / pps;
        p = item % pps;
        bos = n * a.T;
        eos = bos + a.T;
        return n < a.N;
    }
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int NW = NTHR / 32;
    int64_t base = 0;
    for (int64_t n0 = 0; n0 < a.N; n0 += NTHR) {  // block scan of the piece counts, NTHR sequences at a time
        const int64_t m = n0 + tid;
        int64_t cnt = 0;
        if (m < a.N) {
            const int64_t len = a.cu[m + 1] - a.cu[m];
            cnt = len > 0 ? (len + per - 1) / per : 1;
        }
        int64_t x = cnt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) red[warp] = x;
        if (tid == 0) red[NW] = -1;
        __syncthreads();
        int64_t before = base, total = base;
        for (int w = 0; w < NW; ++w) {
            if (w < warp) before += red[w];
            total += red[w];
        }
        const int64_t first = before + x - cnt;
        if (item >= first && item < first + cnt) {
            red[NW] = m;
            red[NW + 1] = item - first;
        }
        __syncthreads();
        n = red[NW];
        p = red[NW + 1];
        __syncthreads();
        if (n >= 0) {
            bos = a.cu[n];
            eos = a.cu[n + 1];
            return true;
        }
        base = total;
    }
    return false;
}

// The place in `local` of piece i's own end state, and after the join of the state that reaches piece i + 1; i counts the
// pieces of sequence n in scan order, `first` is the sequence's first item.
__device__ __forceinline__ int64_t state_slot(const ScanArgs& a, int64_t n, int64_t first, int64_t i) {
    return first - (a.cu ? n : 0) + i;
}
// Places in `local`: sequences of len tokens have ceil(len / per) pieces, packed ones keep (len - 1) / per states.
inline int64_t state_count(int64_t T, int64_t items, bool varlen, int64_t per) { return varlen ? T / per : items; }

// Pieces per work list: exact for batches, an upper bound for packed sequences.
inline int64_t item_count(int64_t B, int64_t T, int64_t N, bool varlen, int64_t per) {
    return varlen ? T / per + N : B * (T > 0 ? (T + per - 1) / per : 1);
}

// All scans of a batch have the same sizes (DB, DC, HV, items, chunking) and the same states_only.
int scan_fp32(const Scans& b, int act_dtype, cudaStream_t s);
bool scan_tc_supported(int64_t DB, int64_t DC, int act_dtype);
int scan_tc(const Scans& b, int64_t tokens, cudaStream_t s);

}  // namespace linattn
}  // namespace gdn
