// gplk_moe_nvfp4.cu - a mixture-of-experts layer for a few tokens, with the
// experts' weights in NVFP4 (the layout gplk_gemm_nvfp4_tn reads):
//   logits = Wr x;  p = softmax(logits);  the `top` experts of largest p
//   h_e = silu(ag_e Wg_e x) * (au_e Wu_e x);  y = sum_j p_j ad_e Wd_e h_e
//
// Bound by HBM: the chosen experts' weights, each read once however many
// tokens chose the expert. Four launches, each starting under the previous
// one's tail (programmatic stream serialisation):
//   router    logits, a block per expert and 8 tokens, FP32 sums
//   route     one block: softmax, top-k, and the lists the products follow
//             (which experts, whose tokens)
//   gate/up   stream_kernel (gplk_nvfp4_stream.cu), a cluster per 128 features of
//             a chosen expert: half of its blocks multiply gate rows, half up
//             rows, over slices of D, by the expert's own tokens; the join
//             writes p_j ad_e silu(g) u, FP32, per (token, rank) slot
//   down      stream_kernel, a cluster per 128 outputs: the chosen experts'
//             rows of down, one after another, are one long K of
//             (experts x F) against each token's h (zero where the expert is
//             not the token's), so the weighted sum over experts happens in
//             the accumulator and no atomics or second pass join it.
#include "gplk_ptx.cuh"

namespace gplk {
namespace moe {

using namespace fewtok;

// Whether the experts' down products go to sums of their own, per (token, rank)
// slot, that a last kernel adds.
static bool use_parts(int T) { return T > 8; }

// Whether a block of the per-slot down products takes two tiles.
static bool use_down_pairs(int T) { return T > 0; }

// Workspace: every part starts on a 256-byte boundary.
struct Layout {
    size_t route, amax, logits, ids, weights, h, part, total;
};

static Layout layout(int T, int E, int top, int D, int F) {
    auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    Layout l;
    l.route = 0;
    l.amax = up(sizeof(Route));
    l.logits = l.amax + up(2 * kMaxTokens * sizeof(uint32_t));
    l.ids = l.logits + up((size_t)T * E * 4);
    l.weights = l.ids + up((size_t)T * top * 4);
    l.h = l.weights + up((size_t)T * top * 4);
    l.part = l.h + up((size_t)T * top * F * 4);
    l.total = l.part + (use_parts(T) ? up((size_t)T * top * D * 4) : 0);
    return l;
}

struct RouteParams {
    const void* x;
    const void* router;
    float* logits;
    int* ids;
    float* weights;
    Route* route;
    uint32_t* amax;  // bits of the largest magnitude of x, then of the weighted h, by token
    int T, E, top, D, ldx, renormalise;
    int vec;  // rows of x and of the router are 16-byte aligned
};

// Router product: a block per expert and up to 8 tokens, whose four warps
// share out K. One more block per 8 tokens finds the tokens' largest
// magnitudes, which anchor the conversion of x, and clears those of h.
constexpr int kRouterThreads = 128;

template <typename XT, int NX>
__global__ void __launch_bounds__(kRouterThreads) router_kernel(const RouteParams p) {
    const int e = blockIdx.x, t0 = blockIdx.y * NX;
    const int nx = min(NX, p.T - t0);
    const int warp = (int)warp_id_uniform();
    const int lane = (int)lane_id();
    pdl_wait();
    pdl_launch_dependents();
    const XT* x = static_cast<const XT*>(p.x) + (size_t)t0 * p.ldx;
    const bool vec = p.vec != 0;
    if (e == p.E) {
        for (int t = warp; t < nx; t += kRouterThreads / 32) {
            uint32_t m = 0;
            for (int k0 = lane * 8; k0 < p.D; k0 += 4 * 256) {
                uint4 r[4][2];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    r[c][0] = make_uint4(0, 0, 0, 0);
                    if (k0 + 256 * c < p.D) load_raw(x + (size_t)t * p.ldx + k0 + 256 * c, vec, r[c]);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float v[8];
                    widen<XT>(r[c], v);
                    m = max(m, max_bits(v));
                }
            }
            m = __reduce_max_sync(0xffffffffu, m);
            if (lane == 0) p.amax[t0 + t] = m;
            if (lane == 1) p.amax[kMaxTokens + t0 + t] = 0;
        }
        return;
    }
    const XT* r = static_cast<const XT*>(p.router) + (size_t)e * p.D;
    float acc[NX] = {};
    for (int k = (int)threadIdx.x * 8; k < p.D; k += kRouterThreads * 8) {
        uint4 wr[2], xr[NX][2];
        load_raw(r + k, vec, wr);
#pragma unroll
        for (int i = 0; i < NX; ++i) load_raw(x + (size_t)min(i, nx - 1) * p.ldx + k, vec, xr[i]);
        float w[8];
        widen<XT>(wr, w);
#pragma unroll
        for (int i = 0; i < NX; ++i) {
            float v[8];
            widen<XT>(xr[i], v);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[i] = fmaf(w[j], v[j], acc[i]);
        }
    }
    __shared__ float part[4][NX];
#pragma unroll
    for (int i = 0; i < NX; ++i) {
#pragma unroll
        for (int o = 16; o; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
        if (lane == 0) part[warp][i] = acc[i];
    }
    __syncthreads();
    if (threadIdx.x < (unsigned)nx)
        p.logits[(size_t)(t0 + threadIdx.x) * p.E + e] = (part[0][threadIdx.x] + part[1][threadIdx.x]) +
                                                         (part[2][threadIdx.x] + part[3][threadIdx.x]);
}

// Order-preserving integer of a float, NaN below every number.
__device__ __forceinline__ uint32_t sort_key(float v) {
    const uint32_t b = __float_as_uint(v);
    return isnan(v) ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return k == 0 ? __uint_as_float(0x7FC00000u) : __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// Softmax and top-k of one token per warp, then the routing tables. A lane
// holds the logits of experts lane, lane + 32, ... (PER of them); each rank
// takes the largest left, the lowest index among equals. A NaN counts below
// every number.
template <int PER>
__global__ void __launch_bounds__(32 * kMaxTokens) route_kernel(const RouteParams p) {
    const int warp = (int)warp_id_uniform();
    const int lane = (int)lane_id();
    constexpr int kPer = kMaxExperts / 32;
    __shared__ int ids[kMaxTokens * kMaxTop];
    __shared__ uint32_t chosen_mask[kPer];
    __shared__ int active[kMaxExperts];
    __shared__ int chunks[kMaxExperts];
    if (threadIdx.x < kPer) chosen_mask[threadIdx.x] = 0;
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    if (warp < p.T) {
        const float* l = p.logits + (size_t)warp * p.E;
        float v[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = lane + 32 * i < p.E ? l[lane + 32 * i] : -INFINITY;
        uint32_t key[PER];
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            key[i] = lane + 32 * i < p.E ? sort_key(v[i]) : 0u;
            most = max(most, key[i]);
        }
        const float best = key_value(__reduce_max_sync(0xffffffffu, most));
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += lane + 32 * i < p.E ? expf(v[i] - best) : 0.0f;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        uint32_t taken = 0;
        float chosen = 0.0f, top_sum = 0.0f;
        int chosen_id = 0;
        for (int j = 0; j < p.top; ++j) {
            uint32_t k = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (!(taken >> i & 1)) k = max(k, key[i]);
            const uint32_t m = __reduce_max_sync(0xffffffffu, k);
            uint32_t e = 0xFFFFFFFFu;
#pragma unroll
            for (int i = PER - 1; i >= 0; --i)
                if (!(taken >> i & 1) && key[i] == m && lane + 32 * i < p.E) e = (uint32_t)(lane + 32 * i);
            e = __reduce_min_sync(0xffffffffu, e);  // top <= E: one is left
            if ((int)(e & 31) == lane) taken |= 1u << (e >> 5);
            const float pr = expf(key_value(m) - best) / sum;
            top_sum += pr;
            if (lane == j) {
                chosen = pr;
                chosen_id = (int)e;
            }
        }
        if (lane < p.top) {
            const int slot = warp * p.top + lane;
            p.ids[slot] = chosen_id;
            p.weights[slot] = p.renormalise ? chosen / top_sum : chosen;
            ids[slot] = chosen_id;
            atomicOr(&chosen_mask[chosen_id >> 5], 1u << (chosen_id & 31));
        }
    }
    __syncthreads();
    // The chosen experts in ascending order, and how many tokens each has.
    int n_active = 0, before = 0;
    {
        const int e = (int)threadIdx.x;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t m = chosen_mask[i];
            if (i < (e >> 5)) before += __popc(m);
            n_active += __popc(m);
        }
        if (e < p.E && (chosen_mask[e >> 5] >> (e & 31) & 1))
            active[before + __popc(chosen_mask[e >> 5] & ((1u << (e & 31)) - 1))] = e;
    }
    __syncthreads();
    auto slot_of = [&](int e) {  // this lane's token's slot with expert e
        int slot = -1;
        if (lane < p.T)
            for (int j = 0; j < p.top; ++j)
                if (ids[lane * p.top + j] == e) slot = lane * p.top + j;
        return slot;
    };
    for (int a = warp; a < n_active; a += kMaxTokens) {
        const uint32_t m = __ballot_sync(0xffffffffu, slot_of(active[a]) >= 0);
        if (lane == 0) chunks[a] = (__popc(m) + kMaxEntryTokens - 1) / kMaxEntryTokens;
    }
    __syncthreads();
    for (int a = warp; a < n_active; a += kMaxTokens) {
        // Entries of the experts before this one.
        int base = 0;
        for (int b = lane; b < a; b += 32) base += chunks[b];
        base = __reduce_add_sync(0xffffffffu, base);
        const int slot = slot_of(active[a]);
        const uint32_t m = __ballot_sync(0xffffffffu, slot >= 0);
        const int n = __popc(m), place = __popc(m & ((1u << lane) - 1));
        for (int c = 0; c < chunks[a]; ++c) {
            const int in_chunk = place - c * kMaxEntryTokens;
            const bool mine = slot >= 0 && in_chunk >= 0 && in_chunk < kMaxEntryTokens;
            if (mine) p.route->list[base + c][in_chunk] = (int16_t)slot;
            p.route->slot[base + c][lane] = (int16_t)(mine ? slot : -1);
            if (lane == 0) p.route->head[base + c] = active[a] | min(kMaxEntryTokens, n - c * kMaxEntryTokens) << 16;
        }
    }
    if (warp == 0) {
        int entries = 0;
        for (int b = lane; b < n_active; b += 32) entries += chunks[b];
        entries = __reduce_add_sync(0xffffffffu, entries);
        for (int b = entries + lane; b < kMaxExperts; b += 32) p.route->head[b] = 0;
        if (lane == 0) p.route->n_entries = entries;
    }
}

// y[t] = the sum of a token's slots, in the order of their ranks.
template <typename XT>
__global__ void __launch_bounds__(256) combine_kernel(const float* part, XT* y, int top, int D, int ldy) {
    const int t = blockIdx.y, n = ((int)blockIdx.x * 256 + (int)threadIdx.x) * 4;
    pdl_wait();
    pdl_launch_dependents();
    if (n >= D) return;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int j = 0; j < top; ++j) {
        const float4 v = *reinterpret_cast<const float4*>(part + ((size_t)t * top + j) * D + n);
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
    }
    XT* row = y + (size_t)t * ldy + n;
    row[0] = from_f32<XT>(s.x);
    row[1] = from_f32<XT>(s.y);
    row[2] = from_f32<XT>(s.z);
    row[3] = from_f32<XT>(s.w);
}

template <typename XT>
static int launch(const gplk_moe_cfg& c, const DeviceInfo& d, cudaStream_t stream) {
    const Layout l = layout(c.T, c.E, c.top, c.D, c.F);
    uint8_t* ws = static_cast<uint8_t*>(c.workspace);
    RouteParams r;
    r.x = c.x;
    r.router = c.router;
    r.logits = reinterpret_cast<float*>(ws + l.logits);
    r.ids = c.ids ? c.ids : reinterpret_cast<int*>(ws + l.ids);
    r.weights = c.weights ? c.weights : reinterpret_cast<float*>(ws + l.weights);
    r.route = reinterpret_cast<Route*>(ws + l.route);
    r.amax = reinterpret_cast<uint32_t*>(ws + l.amax);
    r.vec = aligned16(c.router) && aligned16(c.x) && (c.T == 1 || c.ldx % 8 == 0);
    r.T = c.T;
    r.E = c.E;
    r.top = c.top;
    r.D = c.D;
    r.ldx = c.ldx;
    r.renormalise = c.renormalise;

    const int slots = c.T * c.top;
    // Every entry has a token, and all but one of an expert's kMaxEntryTokens.
    const int most = c.E + slots / kMaxEntryTokens;
    const int max_entries = slots < most ? slots : most;
    // Chosen experts to expect of T independent choices, for the splits.
    double miss = 1.0;
    for (int t = 0; t < c.T; ++t) miss *= 1.0 - (double)c.top / c.E;
    double active = c.E * (1.0 - miss);
    if (active < 1.0) active = 1.0;

    const bool parts = use_parts(c.T);

    Params g;
    memset(&g, 0, sizeof(g));
    g.X = c.x;
    g.sf0 = c.sf_gate;
    g.sf1 = c.sf_up;
    g.alpha0 = c.alpha_gate;
    g.alpha1 = c.alpha_up;
    g.alpha2 = c.alpha_down;
    g.Y = ws + l.h;
    g.route = r.route;
    g.weights = r.weights;
    g.amax = r.amax;
    g.amax_out = r.amax + kMaxTokens;
    g.T = c.T;
    g.N = c.F;
    g.K = c.D;
    g.ldx = c.ldx;
    g.ldy = c.F;
    g.x_vec = aligned16(c.x) && (c.T == 1 || c.ldx % 8 == 0);
    g.top = c.top;
    g.tiles = (c.F + kTileRows - 1) / kTileRows;
    g.k_stages = (c.D + kStageK - 1) / kStageK;
    g.kblocks = c.D / 64;
    g.halves = 2;
    const int entry_tokens = c.T < kMaxEntryTokens ? c.T : kMaxEntryTokens;
    const Shape gs = set_shape(g, entry_tokens, true);
    Params o = g;
    o.X = g.Y;
    o.amax = g.amax_out;
    o.sf0 = c.sf_down;
    o.Y = parts ? static_cast<void*>(ws + l.part) : c.y;
    o.N = c.D;
    o.K = c.F;
    o.ldx = c.F;
    o.ldy = parts ? c.D : c.ldy;
    o.x_vec = 1;
    o.tiles = (c.D + kTileRows - 1) / kTileRows;
    o.k_stages = (c.F + kStageK - 1) / kStageK;
    o.kblocks = c.F / 64;
    o.halves = parts && use_down_pairs(c.T) ? 2 : 1;
    const int groups = (o.tiles + o.halves - 1) / o.halves;
    const Shape os = set_shape(o, parts ? entry_tokens : c.T, parts);
    if (gs.smem > (size_t)d.max_smem_optin) return GPLK_STATUS_UNSUPPORTED;
    g.split_log2 = choose_split_log2(g.tiles * active, 2.0 * g.k_stages, 8, gs.per_sm * d.sm_count);
    o.split_log2 = parts ? choose_split_log2(groups * active, o.halves * o.k_stages, 8, os.per_sm * d.sm_count)
                    : choose_split_log2(groups, o.halves * o.k_stages * active, 8, os.per_sm * d.sm_count);

    CUtensorMap tg, tu, td;
    int st = encode_weights(&tg, c.gate, (uint64_t)c.E * c.F, c.D);
    if (st == GPLK_STATUS_OK) st = encode_weights(&tu, c.up, (uint64_t)c.E * c.F, c.D);
    if (st == GPLK_STATUS_OK) st = encode_weights(&td, c.down, (uint64_t)c.E * c.D, c.F);
    if (st != GPLK_STATUS_OK) return st;

    auto router = [&](auto kernel, int nx) {
        return launch_status(launch_pdl(kernel, dim3(c.E + 1, (c.T + nx - 1) / nx), dim3(kRouterThreads), 0, stream, r));
    };
    st = c.T == 1 ? router(router_kernel<XT, 1>, 1) : c.T <= 4 ? router(router_kernel<XT, 4>, 4) : router(router_kernel<XT, 8>, 8);
    if (st == GPLK_STATUS_OK)
        st = launch_status(launch_pdl(c.E <= 128 ? route_kernel<4> : route_kernel<kMaxExperts / 32>, dim3(1),
                                      dim3(32 * kMaxTokens), 0, stream, r));
    if (st == GPLK_STATUS_OK)
        st = launch_stream<Mode::GateUp, XT, float>(tg, tu, g, gs.smem, max_entries * g.tiles, stream);
    if (st != GPLK_STATUS_OK) return st;
    if (!parts) return launch_stream<Mode::Down, float, XT>(td, td, o, os.smem, groups, stream);
    st = launch_stream<Mode::DownPart, float, float>(td, td, o, os.smem, max_entries * groups, stream);
    if (st != GPLK_STATUS_OK) return st;
    return launch_status(launch_pdl(combine_kernel<XT>, dim3((c.D + 1023) / 1024, c.T), dim3(256), 0, stream,
                                    static_cast<const float*>(o.Y), static_cast<XT*>(c.y), c.top, c.D, c.ldy));
}

}  // namespace moe
}  // namespace gplk

extern "C" size_t gplk_moe_nvfp4_workspace_bytes(int T, int E, int top, int D, int F) {
    using namespace gplk;
    if (T <= 0 || E <= 0 || top <= 0 || D <= 0 || F <= 0 || T > fewtok::kMaxTokens || E > fewtok::kMaxExperts ||
        top > fewtok::kMaxTop || top > E)
        return 0;
    return moe::layout(T, E, top, D, F).total;
}

extern "C" int gplk_moe_nvfp4(const gplk_moe_cfg* cfg, cudaStream_t stream) {
    using namespace gplk;
    using namespace gplk::fewtok;
    if (!cfg) return GPLK_STATUS_BAD_ARG;
    const gplk_moe_cfg& c = *cfg;
    if (c.T < 0 || c.T > kMaxTokens || c.E < 1 || c.E > kMaxExperts || c.top < 1 || c.top > kMaxTop || c.top > c.E)
        return GPLK_STATUS_BAD_ARG;
    if (c.dtype != GPLK_DTYPE_BF16 && c.dtype != GPLK_DTYPE_F16) return GPLK_STATUS_BAD_ARG;
    if (c.D < 64 || c.D % 64 != 0 || c.F < 64 || c.F % 64 != 0) return GPLK_STATUS_BAD_ARG;
    // Rows of the expert stacks are TMA coordinates; grids stay below 2^31.
    if ((long long)c.E * c.F > INT_MAX / 8 || (long long)c.E * c.D > INT_MAX / 8) return GPLK_STATUS_BAD_ARG;
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
        if (!aligned(q, 4)) return GPLK_STATUS_BAD_ARG;
    if (!aligned(c.x, 2) || !aligned(c.y, 2) || !aligned(c.router, 2)) return GPLK_STATUS_BAD_ARG;
    if (c.workspace_bytes < moe::layout(c.T, c.E, c.top, c.D, c.F).total) return GPLK_STATUS_BAD_ARG;
    DeviceInfo d;
    const int st = require_sm100(&d);
    if (st != GPLK_STATUS_OK) return st;
    return c.dtype == GPLK_DTYPE_BF16 ? moe::launch<__nv_bfloat16>(c, d, stream) : moe::launch<__half>(c, d, stream);
}
