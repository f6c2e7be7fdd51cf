// Linear attention with a fixed decay per head: the C entry points (host checks, piece choice, the launches of the
// scan of linear_attn.cuh) and the sum of the gradients of shared query/key heads.
#include "linear_attn.cuh"

#include <algorithm>

#include "launch.h"

namespace gdn {
namespace linattn {

constexpr int kFp32Chunk = 32, kTcChunk = 128;

static bool dtype_ok(int32_t d) { return d == GDN_BF16 || d == GDN_FP16 || d == GDN_FP32; }
static size_t round256(size_t x) { return (x + 255) & ~(size_t)255; }
static bool misaligned(const void* x) { return ((uintptr_t)x & 15) != 0; }

static int check(const gdn_linear_attn_problem* p) {
    if (!p) return GDN_ERR_ARGUMENT;
    if (p->B < 0 || p->T < 0 || p->H <= 0 || p->HV <= 0 || p->DK <= 0 || p->DV <= 0 || p->N < 0) return GDN_ERR_SHAPE;
    if (p->HV % p->H || p->DK > 128 || p->DV > 128 || p->HV > (1 << 20)) return GDN_ERR_SHAPE;
    if (p->cu_seqlens ? p->B != 1 : p->N != p->B) return GDN_ERR_SHAPE;
    if (!dtype_ok(p->act_dtype)) return GDN_ERR_DTYPE;
    return GDN_OK;
}

// Chunks per piece. Time is modelled in units of one chunk's work in one CTA: a launch runs its CTAs in waves of
// `slots`, each as long as its longest piece plus a start-up; cutting (more than one piece for the longest sequence)
// adds a states-only launch that costs `t1` a chunk, a launch gap, and the join of the earlier pieces' states.
struct PieceCost {
    int64_t slots;
    double startup, t1, gap, join;
};
static int choose_piece_chunks(const gdn_linear_attn_problem* p, int chunk, int64_t ctas_per_item, const PieceCost& k) {
    int64_t longest = p->cu_seqlens ? (p->max_seqlen > 0 ? std::min(p->max_seqlen, p->T) : p->T) : p->T;
    // a piece that takes any sequence whole, whatever max_seqlen says: nothing is cut
    const int64_t whole = std::max<int64_t>((p->T + chunk - 1) / chunk, 1);
    longest = (longest + chunk - 1) / chunk;
    if (longest <= 1) return (int)whole;
    double best = 0;
    int64_t best_l = whole;
    for (int64_t pieces = 1; pieces <= 64 && pieces <= longest; ++pieces) {
        const int64_t l = (longest + pieces - 1) / pieces, real = (longest + l - 1) / l;
        double run, pass;
        if (!p->cu_seqlens) {
            const int64_t ctas = p->B * real * ctas_per_item, first = p->B * (real - 1) * ctas_per_item;
            run = (double)((ctas + k.slots - 1) / k.slots) * ((double)l + k.startup);
            pass = (double)((first + k.slots - 1) / k.slots) * ((double)l * k.t1 + k.startup);
        } else {  // uneven lengths: the work spread over the slots, plus the longest piece as its tail; the first
            // launch skips every sequence's last piece, half a piece on average
            const double n = (double)p->N, chunks = (double)p->T / chunk + 0.5 * n, items = chunks / (double)l + 0.5 * n;
            const double share = (double)ctas_per_item / (double)k.slots;
            const double first = std::max(0.0, chunks - 0.5 * n * (double)l);
            run = chunks * share + (double)l + k.startup * (1.0 + items * share);
            pass = (first * share + (double)l) * k.t1 + k.startup * (1.0 + first / (double)l * share);
        }
        const double cost = run + (real > 1 ? pass + k.gap + k.join * (double)(real - 1) : 0.0);
        if (pieces == 1 || cost < best) {
            best = cost;
            best_l = pieces == 1 ? whole : l;
        }
    }
    return (int)best_l;
}

// Geometry of `n_scans` scans of problem p in one launch, with rows of DB and DC features; local_bytes is one scan's.
struct ScanPlan {
    bool tc;  // tensor-memory kernel, else the fp32-accuracy one
    int chunk, piece_chunks;
    int64_t items;
    bool cut;
    // The end state from the join: the tensor-memory kernel with outputs is a fifth slower where it has to keep a state to
    // fp32 (1x65536x16: the whole call 473 us against 412), and the last pieces of equal sequences fit the states' launch
    // without another wave. Packed documents, many of them of one piece, would run their states for nothing else.
    bool end_in_join;
    size_t local_bytes;
};
static ScanPlan plan(const gdn_linear_attn_problem* p, int64_t DB, int64_t DC, int n_scans) {
    ScanPlan s{};
    s.tc = scan_tc_supported(DB, DC, p->act_dtype);
    s.chunk = s.tc ? kTcChunk : kFp32Chunk;
    const int64_t sms = device_sm_count();
    // Measured, on tensor memory (128 tokens): a chunk 4.7 us, its start-up 5.7 (1.2 chunks), a states-only chunk 1.8 to
    // 2.1 (0.4), the two more launches 7 (1.5), a piece more to join 0.15. In tf32 (32 tokens): a chunk 9.7 us in fp32 and
    // 7.1 in fp16 (64 features, two CTAs an SM: 6.2), start-up 0.7 to 0.9 chunks, states-only 0.43, the launches 0.7 to 1.1.
    // The model charges the cut somewhat more than that, for packed windows, where it knows the lengths no better than by
    // the longest: with the measured values single batches of 70 drawn ones gain (2x552 of 4 heads 68 us to 58, all
    // others within 3 %), but forward and backward of 4,295 tokens in 7 documents of 17 bf16 heads go from 166 to 192 us, of
    // 2,969 in 18 documents of 20 fp32 heads from 478 to 590.
    const PieceCost cost = s.tc ? PieceCost{sms, 1.5, 0.55, 1.8, 0.1}
                                : PieceCost{sms * (DB <= 64 && DC <= 64 ? 2 : 1), 0.5, 0.6, 1.8, 0.1};
    s.piece_chunks = choose_piece_chunks(p, s.chunk, p->HV * n_scans, cost);
    const int64_t per = (int64_t)s.chunk * s.piece_chunks;
    s.items = item_count(p->B, p->T, p->N, p->cu_seqlens != nullptr, per);
    s.cut = p->T > per;
    s.end_in_join = s.tc && !p->cu_seqlens;
    const int64_t states = state_count(p->T, s.items, p->cu_seqlens != nullptr, per);
    s.local_bytes = s.cut ? round256((size_t)states * p->HV * DB * DC * sizeof(float)) : 0;
    return s;
}

static int join(const Scans& b, cudaStream_t s);

// Runs a batch of scans of the same sizes. local: n x plan(..., n).local_bytes.
static int scan(const gdn_linear_attn_problem* p, Scans b, void* local, cudaStream_t s) {
    const ScanPlan sp = plan(p, b.s[0].DB, b.s[0].DC, b.n);
    if (sp.items == 0) return GDN_OK;
    for (int i = 0; i < b.n; ++i) {
        ScanArgs& a = b.s[i];
        a.cu = p->cu_seqlens;
        a.T = p->T;
        a.N = p->N;
        a.HV = (int)p->HV;
        a.items = sp.items;
        a.chunk = sp.chunk;
        a.piece_chunks = sp.piece_chunks;
        a.local = sp.cut ? (float*)((uint8_t*)local + i * sp.local_bytes) : nullptr;
        a.precise = a.x1 != nullptr;
        a.end_in_join = sp.cut && sp.end_in_join && a.x1;
    }
    auto launch = [&](int states_only) {
        for (int i = 0; i < b.n; ++i) b.s[i].states_only = states_only;
        return sp.tc ? scan_tc(b, p->B * p->T, s) : scan_fp32(b, p->act_dtype, s);
    };
    if (sp.cut) {
        int st = launch(1);
        if (st == GDN_OK) st = join(b, s);
        if (st != GDN_OK) return st;
        for (int i = 0; i < b.n; ++i)
            if (b.s[i].end_in_join) {
                b.s[i].x1 = nullptr;
                b.s[i].precise = 0;
            }
    }
    return launch(0);
}

// Joins the pieces' own end states along each sequence, in place: a piece's becomes the state that reaches the next one
// (X <- a^len X + local in scan order, X from x0). One thread per 4 elements of a (sequence, value head)'s state; the
// loads of the pieces do not depend on one another, so a chain of P pieces costs about one memory latency for every
// four of them (5 us for 16 heads of a 65,536-token sequence), where each CTA of the scan joining for itself cost two
// microseconds a piece.
__global__ void __launch_bounds__(256) linear_attn_join_kernel(const __grid_constant__ Scans all) {
    __shared__ int64_t red[8];
    const ScanArgs& a = all.s[blockIdx.z];
    const int hv = blockIdx.x % a.HV;
    const int64_t n = blockIdx.x / a.HV, per = (int64_t)a.chunk * a.piece_chunks;
    const int64_t len = a.cu ? a.cu[n + 1] - a.cu[n] : a.T;
    const int pieces = len > 0 ? (int)((len + per - 1) / per) : 1;
    if (pieces == 1 && !a.end_in_join) return;  // nothing to join
    int64_t item0 = n * pieces;
    if (a.cu) {
        int64_t part = 0;  // pieces of the sequences before this one
        for (int64_t m = threadIdx.x; m < n; m += 256) {
            const int64_t l = a.cu[m + 1] - a.cu[m];
            part += l > 0 ? (l + per - 1) / per : 1;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
        if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = part;
        __syncthreads();
        item0 = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) item0 += red[w];
    }
    const int size = a.DB * a.DC, e = (blockIdx.y * 256 + threadIdx.x) * 4;
    if (e >= size) return;
    const int valid = size - e < 4 ? size - e : 4;
    float X[4] = {};
    if (a.x0) {
        const float* x0 = a.x0 + (n * a.HV + hv) * (int64_t)size;
        for (int k = 0; k < valid; ++k) {
            const int r = (e + k) / a.DC, c = (e + k) % a.DC;
            X[k] = x0[a.transposed ? c * a.DB + r : e + k];
        }
    }
    const float g = decay_exponent(a.log_decay, hv);
    const float f = expf(g * (float)per);  // every piece but the sequence's last one is full
    const int last = pieces - 1;
    const float f_last = expf(g * (float)(len - last * per));
    const int own = a.end_in_join ? pieces : last;  // pieces with a state of their own, in scan order
    float* const l = a.local + e + (state_slot(a, n, item0, 0) * a.HV + hv) * (int64_t)size;
    const int64_t step = (int64_t)a.HV * size;
    const bool vec = size % 4 == 0;
    for (int i0 = 0; i0 < own; i0 += 4) {
        float y[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u;
            if (i >= own) continue;
            const float* const src = l + i * step;
            if (vec) *reinterpret_cast<float4*>(y[u]) = *reinterpret_cast<const float4*>(src);
            else
                for (int k = 0; k < valid; ++k) y[u][k] = src[k];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u;
            if (i >= own) continue;
            const float fi = i == (a.reverse ? 0 : last) ? f_last : f;
#pragma unroll
            for (int k = 0; k < 4; ++k) X[k] = fmaf(fi, X[k], y[u][k]);
            float* const dst = l + i * step;
            if (i == last) {  // no piece follows
            } else if (vec) *reinterpret_cast<float4*>(dst) = *reinterpret_cast<float4*>(X);
            else
                for (int k = 0; k < valid; ++k) dst[k] = X[k];
        }
    }
    if (a.end_in_join) {
        float* const x1 = a.x1 + (n * a.HV + hv) * (int64_t)size;
        for (int k = 0; k < valid; ++k) {
            const int r = (e + k) / a.DC, c = (e + k) % a.DC;
            x1[a.transposed ? c * a.DB + r : e + k] = X[k];
        }
    }
}

static int join(const Scans& b, cudaStream_t s) {
    const ScanArgs& a = b.s[0];
    if (a.N * a.HV > 0x7fffffff) return GDN_ERR_SHAPE;
    const dim3 grid((unsigned)(a.N * a.HV), (unsigned)((a.DB * a.DC + 1023) / 1024), (unsigned)b.n);
    linear_attn_join_kernel<<<grid, 256, 0, s>>>(b);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

// The gradients of shared q/k heads (blockIdx.y: dq, dk): out[row, d] = sum over the `group` value heads of a q/k head of
// x[row * group + e, d], VEC features a thread: a stream of 4 (group + 1/2) bytes a feature; 33 us for 8,191 tokens of 20
// value heads of 128 in groups of two (210 MB, at a copy's rate).
template <typename TA, int VEC>
__global__ void __launch_bounds__(256) head_group_sum_kernel(const float* xq, const float* xk, TA* outq, TA* outk, int64_t n,
                                                             int group, int D) {
    const float* const x = blockIdx.y ? xk : xq;
    TA* const out = blockIdx.y ? outk : outq;
    const int per_row = D / VEC;
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per_row;
        const int d = (int)(i - row * per_row) * VEC;
        float acc[VEC] = {};
        for (int e = 0; e < group; ++e) {
            float y[VEC];
            ldv<float, VEC>(x, (row * group + e) * D + d, y);
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] += y[k];
        }
        stv<TA, VEC>(out, row * D + d, acc);
    }
}

static int head_group_sum(const float* xq, const float* xk, void* outq, void* outk, int act_dtype, int64_t rows,
                          int group, int64_t D, cudaStream_t s) {
    if (rows == 0) return GDN_OK;
    const int vec = D % 8 == 0 ? 8 : 1;
    const int64_t n = rows * D / vec;
    const dim3 grid((unsigned)std::min<int64_t>((n + 255) / 256, (int64_t)device_sm_count() * 8), 2);
    GDN_DISPATCH_DTYPE(act_dtype, TA, {
        if (vec == 8) head_group_sum_kernel<TA, 8><<<grid, 256, 0, s>>>(xq, xk, (TA*)outq, (TA*)outk, n, group, (int)D);
        else head_group_sum_kernel<TA, 1><<<grid, 256, 0, s>>>(xq, xk, (TA*)outq, (TA*)outk, n, group, (int)D);
    })
    count_launch();
    return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

}  // namespace linattn
}  // namespace gdn

using namespace gdn;
using namespace gdn::linattn;

extern "C" {

size_t gdn_linear_attn_fwd_workspace_size(const gdn_linear_attn_problem* p) {
    if (check(p) != GDN_OK) return 0;
    return plan(p, p->DK, p->DV, 1).local_bytes;
}

int gdn_linear_attn_fwd(const gdn_linear_attn_problem* p, const void* q, const void* k, const void* v,
                        const float* log_decay, const float* initial_state, void* o, float* final_state,
                        void* workspace, size_t workspace_bytes, gdn_stream_t stream) {
    const int st = check(p);
    if (st != GDN_OK) return st;
    if (p->N == 0) return GDN_OK;
    if (!log_decay || (p->B * p->T > 0 && (!q || !k || !v || !o))) return GDN_ERR_ARGUMENT;
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(o) || misaligned(initial_state) ||
        misaligned(final_state) || misaligned(workspace))
        return GDN_ERR_ALIGN;
    const size_t need = gdn_linear_attn_fwd_workspace_size(p);
    if (need && (!workspace || workspace_bytes < need)) return GDN_ERR_WORKSPACE;
    const int r = (int)(p->HV / p->H);
    Scans b{};
    b.n = 1;
    ScanArgs& a = b.s[0];
    a.A = q; a.B = k; a.C = v; a.out = o;
    a.log_decay = log_decay;
    a.x0 = initial_state; a.x1 = final_state;
    a.gA = r; a.gB = r; a.gC = 1;
    a.DB = (int)p->DK; a.DC = (int)p->DV;
    a.sp = a.si = p->scale; a.su = 1.f;
    return scan(p, b, workspace, (cudaStream_t)stream);
}

// The backward's three scans run in one launch where DK = DV; otherwise dq and dk (rows of DV and DK features) in one and
// dv (DK and DV) in another. Workspace: the pieces' states of a launch, then (HV > H) dq and dk per value head in fp32.
static size_t bwd_local_bytes(const gdn_linear_attn_problem* p) {
    if (p->DK == p->DV) return 3 * plan(p, p->DK, p->DV, 3).local_bytes;
    return std::max(2 * plan(p, p->DV, p->DK, 2).local_bytes, plan(p, p->DK, p->DV, 1).local_bytes);
}
static size_t per_head_bytes(const gdn_linear_attn_problem* p) {
    return p->HV > p->H ? round256((size_t)p->B * p->T * p->HV * p->DK * sizeof(float)) : 0;
}
size_t gdn_linear_attn_bwd_workspace_size(const gdn_linear_attn_problem* p) {
    if (check(p) != GDN_OK) return 0;
    return bwd_local_bytes(p) + 2 * per_head_bytes(p);
}

int gdn_linear_attn_bwd(const gdn_linear_attn_problem* p, const void* q, const void* k, const void* v,
                        const float* log_decay, const float* initial_state, const void* dout, const float* dht,
                        void* dq, void* dk, void* dv, float* dh0, void* workspace, size_t workspace_bytes,
                        gdn_stream_t stream) {
    int st = check(p);
    if (st != GDN_OK) return st;
    if (p->N == 0) return GDN_OK;
    if (!log_decay || (p->B * p->T > 0 && (!q || !k || !v || !dout || !dq || !dk || !dv))) return GDN_ERR_ARGUMENT;
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(dout) || misaligned(dq) || misaligned(dk) ||
        misaligned(dv) || misaligned(dh0) || misaligned(dht) || misaligned(initial_state) || misaligned(workspace))
        return GDN_ERR_ALIGN;
    const size_t need = gdn_linear_attn_bwd_workspace_size(p);
    if (need && (!workspace || workspace_bytes < need)) return GDN_ERR_WORKSPACE;
    cudaStream_t s = (cudaStream_t)stream;
    const int r = (int)(p->HV / p->H);
    float* const dq32 = r > 1 ? (float*)((uint8_t*)workspace + bwd_local_bytes(p)) : nullptr;
    float* const dk32 = r > 1 ? (float*)((uint8_t*)dq32 + per_head_bytes(p)) : nullptr;
    Scans b{};
    ScanArgs &sq = b.s[0], &sk = b.s[1], &sv = b.s[2];
    // dq: forward over (do, v, k), the state transposed
    sq.log_decay = log_decay;
    sq.A = dout; sq.B = v; sq.C = k;
    sq.gA = sq.gB = 1; sq.gC = r;
    sq.DB = (int)p->DV; sq.DC = (int)p->DK;
    sq.x0 = initial_state; sq.transposed = 1;
    sq.sp = sq.si = p->scale; sq.su = 1.f;
    sq.out = r > 1 ? (void*)dq32 : dq; sq.out_fp32 = r > 1;
    // dk: backwards over (v, do, q), the state's gradient transposed
    sk = sq;
    sk.A = v; sk.B = dout; sk.C = q;
    sk.reverse = 1;
    sk.x0 = dht;
    sk.sp = p->scale; sk.si = 1.f; sk.su = p->scale;
    sk.out = r > 1 ? (void*)dk32 : dk;
    // dv: backwards over (k, q, do); it leaves the initial state's gradient
    sv = sk;
    sv.A = k; sv.B = q; sv.C = dout;
    sv.gA = sv.gB = r; sv.gC = 1;
    sv.DB = (int)p->DK; sv.DC = (int)p->DV;
    sv.transposed = 0;
    sv.x1 = dh0;
    sv.out = dv; sv.out_fp32 = 0;
    if (p->DK == p->DV) {
        b.n = 3;
        st = scan(p, b, workspace, s);
    } else {
        b.n = 2;
        st = scan(p, b, workspace, s);
        if (st != GDN_OK) return st;
        b.s[0] = sv;
        b.n = 1;
        st = scan(p, b, workspace, s);
    }
    if (st == GDN_OK && r > 1) st = head_group_sum(dq32, dk32, dq, dk, p->act_dtype, p->B * p->T * p->H, r, p->DK, s);
    return st;
}

}  // extern "C"
