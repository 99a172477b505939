// gplk_moe_nvfp4.cu - a mixture-of-experts layer for a few tokens, with the
// experts' weights in NVFP4 (the layout gplk_gemm_nvfp4_tn reads):
//   logits = Wr x;  p = softmax(logits);  the `top` experts of largest p
//   h_e = silu(ag_e Wg_e x) * (au_e Wu_e x);  y = sum_j p_j ad_e Wd_e h_e
#include "gplk_ptx.cuh"

namespace gplk {
namespace moe {

using fewtok::aligned;
using fewtok::from_f32;
using fewtok::kMaxTokens;
using fewtok::row_dots;
using fewtok::to_f32;

constexpr int kMaxExperts = 512;
constexpr int kMaxTop = 16;

// Workspace: every part starts on a 256-byte boundary.
struct Layout {
    size_t logits, ids, weights, h, total;
};

static Layout layout(int T, int E, int top, int F) {
    auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    Layout l;
    l.logits = 0;
    l.ids = l.logits + up((size_t)T * E * 4);
    l.weights = l.ids + up((size_t)T * top * 4);
    l.h = l.weights + up((size_t)T * top * 4);
    l.total = l.h + up((size_t)T * top * F * 4);
    return l;
}

struct Params {
    gplk_moe_cfg c;
    float* logits;
    int* ids;
    float* weights;
    float* h;
};

// Router product: one block per expert and 8 tokens.
template <typename XT>
__global__ void __launch_bounds__(128) router_kernel(const Params p) {
    const int e = blockIdx.x, t0 = blockIdx.y * 8;
    const int nx = min(8, p.c.T - t0);
    const XT* r = static_cast<const XT*>(p.c.router) + (size_t)e * p.c.D;
    const XT* x = static_cast<const XT*>(p.c.x) + (size_t)t0 * p.c.ldx;
    float acc[8] = {};
    for (int k = threadIdx.x; k < p.c.D; k += 128) {
        const float w = to_f32(r[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < nx) acc[i] = fmaf(w, to_f32(x[(size_t)i * p.c.ldx + k]), acc[i]);
    }
    __shared__ float part[4][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int o = 16; o; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
        if (lane_id() == 0) part[threadIdx.x / 32][i] = acc[i];
    }
    __syncthreads();
    if (threadIdx.x < (unsigned)nx)
        p.logits[(size_t)(t0 + threadIdx.x) * p.c.E + e] = (part[0][threadIdx.x] + part[1][threadIdx.x]) +
                                                           (part[2][threadIdx.x] + part[3][threadIdx.x]);
}

// Softmax and top-k of one token per warp. A lane holds the logits of experts
// lane, lane + 32, ...; each rank takes the largest left, the lowest index
// among equals. A NaN counts below every number.
__global__ void __launch_bounds__(32 * kMaxTokens) route_kernel(const Params p) {
    const int t = (int)warp_id_uniform();
    const int lane = (int)lane_id();
    if (t >= p.c.T) return;
    constexpr int kPer = kMaxExperts / 32;
    const float* l = p.logits + (size_t)t * p.c.E;
    float v[kPer];
    float best = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = lane + 32 * i;
        v[i] = e < p.c.E ? l[e] : -INFINITY;
        best = fmaxf(best, v[i]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += lane + 32 * i < p.c.E ? expf(v[i] - best) : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    uint32_t taken = 0;
    float chosen = 0.0f, top_sum = 0.0f;
    int chosen_id = 0;
    for (int j = 0; j < p.c.top; ++j) {
        float bv = 0.0f;
        int be = INT_MAX;  // INT_MAX: none yet
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = lane + 32 * i;
            if (e >= p.c.E || (taken >> i & 1)) continue;
            const float a = isnan(v[i]) ? -INFINITY : v[i];
            if (be == INT_MAX || a > bv) {
                bv = a;
                be = e;
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
            const int oe = __shfl_xor_sync(0xffffffffu, be, o);
            if (oe != INT_MAX && (be == INT_MAX || ov > bv || (ov == bv && oe < be))) {
                bv = ov;
                be = oe;
            }
        }
        if ((be & 31) == lane) taken |= 1u << (be >> 5);
        const float pr = expf(l[be] - best) / sum;
        top_sum += pr;
        if (lane == j) {
            chosen = pr;
            chosen_id = be;
        }
    }
    if (lane < p.c.top) {
        p.ids[t * p.c.top + lane] = chosen_id;
        p.weights[t * p.c.top + lane] = p.c.renormalise ? chosen / top_sum : chosen;
    }
}

__device__ __forceinline__ size_t sf_stride(int rows, int k) {
    return (size_t)((rows + 127) / 128) * (size_t)((k + 63) / 64) * 512;
}

template <typename XT>
__global__ void __launch_bounds__(256) gate_up_kernel(const Params p) {
    const int f = blockIdx.x * 8 + (int)warp_id_uniform();
    const int slot = blockIdx.y;
    if (f >= p.c.F) return;
    const int e = p.ids[slot];
    const XT* x[8];
    for (int i = 0; i < 8; ++i) x[i] = static_cast<const XT*>(p.c.x) + (size_t)(slot / p.c.top) * p.c.ldx;
    const size_t wo = (size_t)e * p.c.F * (p.c.D / 2), so = (size_t)e * sf_stride(p.c.F, p.c.D);
    float g[8], u[8];
    row_dots<XT>(p.c.gate + wo, p.c.sf_gate + so, (size_t)f, p.c.D, x, 1, g);
    row_dots<XT>(p.c.up + wo, p.c.sf_up + so, (size_t)f, p.c.D, x, 1, u);
    if (lane_id() == 0) {
        const float gv = g[0] * p.c.alpha_gate[e];
        p.h[(size_t)slot * p.c.F + f] = gv / (1.0f + expf(-gv)) * (u[0] * p.c.alpha_up[e]);
    }
}

template <typename XT>
__global__ void __launch_bounds__(256) down_kernel(const Params p) {
    const int n = blockIdx.x * 8 + (int)warp_id_uniform();
    const int t = blockIdx.y;
    if (n >= p.c.D) return;
    float y = 0.0f;
    for (int j = 0; j < p.c.top; ++j) {
        const int e = p.ids[t * p.c.top + j];
        const float* h[8];
        for (int i = 0; i < 8; ++i) h[i] = p.h + (size_t)(t * p.c.top + j) * p.c.F;
        float o[8];
        row_dots<float>(p.c.down + (size_t)e * p.c.D * (p.c.F / 2), p.c.sf_down + (size_t)e * sf_stride(p.c.D, p.c.F),
                        (size_t)n, p.c.F, h, 1, o);
        y = fmaf(o[0] * p.c.alpha_down[e], p.weights[t * p.c.top + j], y);
    }
    if (lane_id() == 0) static_cast<XT*>(p.c.y)[(size_t)t * p.c.ldy + n] = from_f32<XT>(y);
}

template <typename XT>
static int launch(const Params& p, cudaStream_t stream) {
    const gplk_moe_cfg& c = p.c;
    router_kernel<XT><<<dim3(c.E, (c.T + 7) / 8), 128, 0, stream>>>(p);
    route_kernel<<<1, 32 * c.T, 0, stream>>>(p);
    gate_up_kernel<XT><<<dim3((c.F + 7) / 8, c.T * c.top), 256, 0, stream>>>(p);
    down_kernel<XT><<<dim3((c.D + 7) / 8, c.T), 256, 0, stream>>>(p);
    return launch_status(cudaGetLastError());
}

}  // namespace moe
}  // namespace gplk

extern "C" size_t gplk_moe_nvfp4_workspace_bytes(int T, int E, int top, int D, int F) {
    using namespace gplk;
    if (T <= 0 || E <= 0 || top <= 0 || D <= 0 || F <= 0 || T > moe::kMaxTokens || E > moe::kMaxExperts ||
        top > moe::kMaxTop || top > E)
        return 0;
    return moe::layout(T, E, top, F).total;
}

extern "C" int gplk_moe_nvfp4(const gplk_moe_cfg* cfg, cudaStream_t stream) {
    using namespace gplk;
    if (!cfg) return GPLK_STATUS_BAD_ARG;
    const gplk_moe_cfg& c = *cfg;
    if (c.T < 0 || c.T > moe::kMaxTokens || c.E < 1 || c.E > moe::kMaxExperts || c.top < 1 || c.top > moe::kMaxTop ||
        c.top > c.E)
        return GPLK_STATUS_BAD_ARG;
    if (c.dtype != GPLK_DTYPE_BF16 && c.dtype != GPLK_DTYPE_F16) return GPLK_STATUS_BAD_ARG;
    if (c.D < 64 || c.D % 64 != 0 || c.F < 64 || c.F % 64 != 0) return GPLK_STATUS_BAD_ARG;
    if ((long long)c.E * c.F > INT_MAX || (long long)c.E * c.D > INT_MAX) return GPLK_STATUS_BAD_ARG;
    if (c.T == 0) return GPLK_STATUS_OK;
    if (c.ldx < c.D || c.ldy < c.D) return GPLK_STATUS_BAD_ARG;
    if (!c.x || !c.router || !c.gate || !c.up || !c.down || !c.sf_gate || !c.sf_up || !c.sf_down || !c.alpha_gate ||
        !c.alpha_up || !c.alpha_down || !c.y || !c.workspace)
        return GPLK_STATUS_BAD_ARG;
    for (const void* q : {(const void*)c.gate, (const void*)c.up, (const void*)c.down, (const void*)c.sf_gate,
                          (const void*)c.sf_up, (const void*)c.sf_down, (const void*)c.workspace})
        if (!aligned16(q)) return GPLK_STATUS_BAD_ARG;
    for (const void* q : {(const void*)c.alpha_gate, (const void*)c.alpha_up, (const void*)c.alpha_down,
                          (const void*)c.ids, (const void*)c.weights})
        if (!moe::aligned(q, 4)) return GPLK_STATUS_BAD_ARG;
    if (!moe::aligned(c.x, 2) || !moe::aligned(c.y, 2) || !moe::aligned(c.router, 2)) return GPLK_STATUS_BAD_ARG;
    const moe::Layout l = moe::layout(c.T, c.E, c.top, c.F);
    if (c.workspace_bytes < l.total) return GPLK_STATUS_BAD_ARG;
    DeviceInfo d;
    const int st = require_sm100(&d);
    if (st != GPLK_STATUS_OK) return st;
    uint8_t* ws = static_cast<uint8_t*>(c.workspace);
    const moe::Params p{c,
                        reinterpret_cast<float*>(ws + l.logits),
                        c.ids ? c.ids : reinterpret_cast<int*>(ws + l.ids),
                        c.weights ? c.weights : reinterpret_cast<float*>(ws + l.weights),
                        reinterpret_cast<float*>(ws + l.h)};
    return c.dtype == GPLK_DTYPE_BF16 ? moe::launch<__nv_bfloat16>(p, stream) : moe::launch<__half>(p, stream);
}
