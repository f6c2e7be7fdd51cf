// One token of linear attention with a fixed decay per head on resident fp32 states, in place:
//   S <- a S + k v^T,   o = scale S^T q      (a = exp(log_decay[h]))
// Each state is read once and written once, 8 DK DV bytes against 4 DK + 4 DV of activations, so the kernel is a
// stream at the memory's copy speed. A CTA takes one (request, value head) and a slice of the state's columns
// (columns are independent: no sums cross CTAs). Its threads hold ROWS rows of 4 columns each, all loads issued
// before the first use. Slices are 64 columns: with the whole 128 a CTA's registers leave two on an SM, which then
// load and store in phase (256 requests x 16 heads: 121 us against 90, 0.92 of the copy rate); 32 where there is an
// SM for every such slice (16 states of 128 columns: 2.4 us against 2.7, 32: 2.5 against 2.7, but 64: 2.9 against 2.8 and
// 128: 3.9 against 3.5).
#include "common.cuh"
#include "kernels.h"
#include "launch.h"

namespace gdn {
namespace linstep {

constexpr int NTHR = 256;

struct StepArgs {
    const void *q, *k, *v;
    const float* log_decay;
    float* state;
    const int32_t* slots;  // [N], or NULL: request n's state is state[n]
    void* o;
    int64_t n_slots;
    int H, HV, DK, DV;
    float scale;
};

// VEC columns per thread (4, or 1 for column counts that are not a multiple of 4); COLS = columns per CTA
template <typename TA, int VEC, int COLS>
__global__ void __launch_bounds__(NTHR) linear_attn_step_kernel(const StepArgs a) {
    constexpr int CT = COLS / VEC;     // threads across the columns
    constexpr int RT = NTHR / CT;      // threads across the rows
    constexpr int ROWS = 128 / RT;     // rows per thread
    __shared__ float sq[128], sk[128];
    __shared__ float part[RT][COLS + 4];
    const int tid = threadIdx.x;
    const int64_t n = blockIdx.x / a.HV;
    const int hv = (int)(blockIdx.x % a.HV), hq = hv / (a.HV / a.H);
    const int c = blockIdx.y * COLS + (tid % CT) * VEC, r0 = tid / CT;
    const int64_t slot = a.slots ? (int64_t)a.slots[n] : n;
    TA* o = (TA*)a.o + (n * a.HV + hv) * a.DV;
    if (slot < 0 || slot >= a.n_slots) {  // an idle request (negative): zeros; a slot past the pool: NaN, no access
        const int cc = blockIdx.y * COLS + tid;
        if (tid < COLS && cc < a.DV) st(o, cc, slot < 0 ? 0.f : __int_as_float(0x7fc00000));
        return;
    }
    float* S = a.state + (slot * a.HV + hv) * (int64_t)a.DK * a.DV;
    float x[ROWS][VEC], v[VEC] = {};
    const bool col = c < a.DV;
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        const int r = r0 + u * RT;
        if (col && r < a.DK) {
            if constexpr (VEC == 4) {
                const float4 y = *reinterpret_cast<const float4*>(S + (int64_t)r * a.DV + c);
                x[u][0] = y.x; x[u][1] = y.y; x[u][2] = y.z; x[u][3] = y.w;
            } else {
                x[u][0] = S[(int64_t)r * a.DV + c];
            }
        }
    }
    if (tid < a.DK) sq[tid] = ld((const TA*)a.q, (n * a.H + hq) * a.DK + tid);
    if (tid >= 128 && tid - 128 < a.DK) sk[tid - 128] = ld((const TA*)a.k, (n * a.H + hq) * a.DK + tid - 128);
    if (col) {
#pragma unroll
        for (int w = 0; w < VEC; ++w) v[w] = ld((const TA*)a.v, (n * a.HV + hv) * a.DV + c + w);
    }
    const float decay = expf(a.log_decay[hv]);
    __syncthreads();
    float acc[VEC] = {};
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        const int r = r0 + u * RT;
        if (!col || r >= a.DK) continue;
        const float kr = sk[r], qr = sq[r];
#pragma unroll
        for (int w = 0; w < VEC; ++w) {
            x[u][w] = fmaf(kr, v[w], decay * x[u][w]);
            acc[w] = fmaf(qr, x[u][w], acc[w]);
        }
        if constexpr (VEC == 4)
            *reinterpret_cast<float4*>(S + (int64_t)r * a.DV + c) = make_float4(x[u][0], x[u][1], x[u][2], x[u][3]);
        else S[(int64_t)r * a.DV + c] = x[u][0];
    }
#pragma unroll
    for (int w = 0; w < VEC; ++w) part[r0][(tid % CT) * VEC + w] = acc[w];
    __syncthreads();
    const int cc = blockIdx.y * COLS + tid;
    if (tid < COLS && cc < a.DV) {
        float y = 0.f;
#pragma unroll
        for (int u = 0; u < RT; ++u) y += part[u][tid];
        st(o, cc, a.scale * y);
    }
}

template <typename TA, int VEC, int COLS>
static void launch(const StepArgs& a, int64_t N, cudaStream_t s) {
    const dim3 grid((unsigned)(N * a.HV), (unsigned)((a.DV + COLS - 1) / COLS));
    linear_attn_step_kernel<TA, VEC, COLS><<<grid, NTHR, 0, s>>>(a);
}

}  // namespace linstep
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_linear_attn_step(int64_t N, int64_t H, int64_t HV, int64_t DK, int64_t DV, float scale,
                                    int32_t act_dtype, const void* q, const void* k, const void* v,
                                    const float* log_decay, float* state, int64_t n_slots, const int32_t* slots,
                                    void* o, gdn_stream_t stream) {
    using namespace linstep;
    if (N < 0 || H <= 0 || HV <= 0 || HV % H || DK <= 0 || DK > 128 || DV <= 0 || DV > 128 || n_slots < 0 ||
        (!slots && n_slots < N) || N * HV > 0x7fffffff)
        return GDN_ERR_SHAPE;
    if (act_dtype != GDN_BF16 && act_dtype != GDN_FP16 && act_dtype != GDN_FP32) return GDN_ERR_DTYPE;
    if (N == 0) return GDN_OK;
    if (!q || !k || !v || !log_decay || !o || (n_slots > 0 && !state)) return GDN_ERR_ARGUMENT;
    if (DV % 4 == 0 && ((uintptr_t)state & 15)) return GDN_ERR_ALIGN;  // rows of whole 16-byte vectors
    StepArgs a{};
    a.q = q; a.k = k; a.v = v; a.log_decay = log_decay; a.state = state; a.slots = slots; a.o = o;
    a.n_slots = n_slots;
    a.H = (int)H; a.HV = (int)HV; a.DK = (int)DK; a.DV = (int)DV; a.scale = scale;
    cudaStream_t s = (cudaStream_t)stream;
    const bool few = N * HV * ((DV + 31) / 32) <= device_sm_count();  // an SM for every 32-column slice
    GDN_DISPATCH_DTYPE(act_dtype, TA, {
        if (DV % 4) launch<TA, 1, 32>(a, N, s);
        else if (few) launch<TA, 4, 32>(a, N, s);
        else launch<TA, 4, 64>(a, N, s);
    })
    count_launch();
    return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}
