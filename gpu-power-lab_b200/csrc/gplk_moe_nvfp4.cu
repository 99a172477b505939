// gplk_moe_nvfp4.cu - a mixture-of-experts layer for a few tokens, with the
// experts' weights in NVFP4 (the layout gplk_gemm_nvfp4_tn reads):
//   logits = Wr x;  p = softmax(logits);  the `top` experts of largest p
//   h_e = silu(ag_e Wg_e x) * (au_e Wu_e x);  y = sum_j p_j ad_e Wd_e h_e
//
// Bound by HBM: the chosen experts' weights, each read once however many
// tokens chose the expert (up to 12; a second dozen reads it again, out of L2 for
// the most part). Launches, each starting under the previous one's tail
// (programmatic stream serialisation):
//   router    logits, FP32 sums, and the magnitudes that anchor the conversion of x
//   route     one block: softmax, top-k, and the entries the products follow
//             (a chosen expert with up to 12 of its tokens); for few experts and
//             tokens one launch with the router (few_route_kernel)
//   gate/up   128 features of an entry at a time, gate and up against the same
//             converted tokens; writes p_j ad_e silu(g) u, FP32, per (token, rank)
//             slot. A cluster per item with K split over it (stream_kernel of
//             gplk_nvfp4_stream.cu), or, with two items for every SM, resident
//             blocks (item_kernel)
//   down      by few tokens a cluster per 128 outputs: the entries' rows of down,
//             one after another, are one long K of (entries x F) against each
//             token's h (zero where the entry is not the token's), so the sum over
//             experts happens in the accumulator (stream_kernel). Else resident
//             blocks write a sum per slot, and a last launch adds a token's.
// No atomics order a sum; the maxima that atomics find do not depend on it.
// Measured, us, against the bytes at 6547 GB/s: 1 token 64/8 2048x1024 19 (4.4),
// 8 tokens 128/8 4096x768 69 (42), 16 tokens 16/2 4096x4096 88 (61; FP16 92), 32
// tokens 64/6 4096x2048 165 (133), 32/8 4096x2048 136 (69). Small layers are the
// launches' latencies, 15 us at least; large ones what resident blocks do not
// overlap: routing before the first weight (some 8 us), a last round of items
// that not all SMs have, and with many tokens an expert their conversion, which
// every item repeats.
#include "gplk_ptx.cuh"

namespace gplk {
namespace moe {

using namespace fewtok;

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
    l.total = l.part + up((size_t)T * top * D * 4);
    return l;
}

// Sizes the layer takes.
static bool takes(int T, int E, int top, int D, int F) {
    if (T < 0 || T > kMaxTokens || E < 1 || E > kMaxExperts || top < 1 || top > kMaxTop || top > E) return false;
    if (D < 64 || D % 64 != 0 || F < 64 || F % 64 != 0) return false;
    // Rows of a stack, numbers of stages and grids stay below 2^31.
    return (long long)E * F <= INT_MAX / 8 && (long long)E * D <= INT_MAX / 8;
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

// Largest magnitude of token t, by one warp: it anchors the conversion of x. The
// magnitude of the token's h starts at zero.
template <typename XT>
__device__ __forceinline__ void token_amax(const RouteParams& p, int t) {
    const int lane = (int)lane_id();
    const XT* x = static_cast<const XT*>(p.x) + (size_t)t * p.ldx;
    uint32_t m = 0;
    for (int k0 = lane * 8; k0 < p.D; k0 += 4 * 256) {
        uint4 r[4][2];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            r[c][0] = make_uint4(0, 0, 0, 0);
            if (k0 + 256 * c < p.D) load_raw(x + k0 + 256 * c, p.vec != 0, r[c]);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            float v[8];
            widen<XT>(r[c], v);
            m = max(m, max_bits(v));
        }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) p.amax[t] = m;
    if (lane == 1) p.amax[kMaxTokens + t] = 0;
}

// Sums over this thread's share of K (from k0 in steps of `step`) of the products
// of a router row with the rows of tokens t0 .. t0 + nx - 1.
template <typename XT, int NX>
__device__ __forceinline__ void router_dots(const RouteParams& p, int e, int t0, int nx, int k0, int step,
                                            float (&acc)[NX]) {
    const XT* r = static_cast<const XT*>(p.router) + (size_t)e * p.D;
    const XT* x = static_cast<const XT*>(p.x) + (size_t)t0 * p.ldx;
#pragma unroll
    for (int i = 0; i < NX; ++i) acc[i] = 0.0f;
#pragma unroll(NX == 1 ? 4 : NX <= 4 ? 2 : 1)
    for (int k = k0; k < p.D; k += step) {
        uint4 wr[2], xr[NX][2];
        load_raw(r + k, p.vec != 0, wr);
#pragma unroll
        for (int i = 0; i < NX; ++i) load_raw(x + (size_t)min(i, nx - 1) * p.ldx + k, p.vec != 0, xr[i]);
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
#pragma unroll
    for (int i = 0; i < NX; ++i)
#pragma unroll
        for (int o = 16; o; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
}

// Router product of many experts: a block per expert and up to NX tokens, whose
// warps share out K (a thread's loads are then one round trip up to K = 4096);
// one more block per NX tokens for their magnitudes.
constexpr int kRouterThreads = 512;

template <typename XT, int NX>
__global__ void __launch_bounds__(kRouterThreads) router_kernel(const RouteParams p) {
    const int e = blockIdx.x, t0 = blockIdx.y * NX;
    const int nx = min(NX, p.T - t0);
    const int warp = (int)warp_id_uniform();
    pdl_wait();
    pdl_launch_dependents();
    if (e == p.E) {
        for (int t = warp; t < nx; t += kRouterThreads / 32) token_amax<XT>(p, t0 + t);
        return;
    }
    float acc[NX];
    router_dots<XT, NX>(p, e, t0, nx, (int)threadIdx.x * 8, kRouterThreads * 8, acc);
    __shared__ float part[kRouterThreads / 32][NX];
    if (lane_id() == 0) {
#pragma unroll
        for (int i = 0; i < NX; ++i) part[warp][i] = acc[i];
    }
    __syncthreads();
    if (threadIdx.x < (unsigned)nx) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kRouterThreads / 32; ++w) v += part[w][threadIdx.x];
        p.logits[(size_t)(t0 + threadIdx.x) * p.E + e] = v;
    }
}

// Order-preserving integer of a float, NaN below every number.
__device__ __forceinline__ uint32_t sort_key(float v) {
    const uint32_t b = __float_as_uint(v);
    return isnan(v) ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return k == 0 ? __uint_as_float(0x7FC00000u) : __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// Softmax and top-k of one token per warp, then the routing tables, by one block
// of WARPS warps (at least T of them, and a thread for every expert). A lane holds
// the logits of experts lane, lane + 32, ... (PER of them); each rank takes the
// largest left, the lowest index among equals. A NaN counts below every number.
constexpr int kPer = kMaxExperts / 32;

struct RouteShared {
    alignas(16) int16_t slot[kMaxExperts][kMaxTokens];  // token's slot with an expert, or -1
    uint32_t chosen[kPer];         // experts, as bits
    int active[kMaxExperts];       // the chosen ones, ascending
    uint32_t tokens[kMaxExperts];  // theirs, as bits
};

// What does not wait for the logits.
template <int WARPS>
__device__ __forceinline__ void route_prepare(const RouteParams& p, RouteShared& sh) {
    uint4* slots = reinterpret_cast<uint4*>(&sh.slot[0][0]);
    for (int i = (int)threadIdx.x; i < p.E * kMaxTokens / 8; i += 32 * WARPS) slots[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
    if (threadIdx.x < kPer) sh.chosen[threadIdx.x] = 0;
    __syncthreads();
}

template <int PER, int WARPS>
__device__ __forceinline__ void route_body(const RouteParams& p, RouteShared& sh) {
    static_assert(32 * WARPS >= kMaxExperts, "a thread per expert");
    const int warp = (int)warp_id_uniform();
    const int lane = (int)lane_id();
    if (warp < p.T) {
        const float* l = p.logits + (size_t)warp * p.E;
        float v[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = lane + 32 * i < p.E ? __ldcg(l + lane + 32 * i) : -INFINITY;
        uint32_t key[PER];
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            key[i] = lane + 32 * i < p.E ? sort_key(v[i] + 0.0f) : 0u;  // -0 equals 0
            most = max(most, key[i]);
        }
        const float best = key_value(__reduce_max_sync(0xffffffffu, most));
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += lane + 32 * i < p.E ? expf(v[i] - best) : 0.0f;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        uint32_t taken = 0, my_key = 0;
        int my_expert = 0;  // lane j: the expert of rank j
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
            if (lane == j) {
                my_key = m;
                my_expert = (int)e;
            }
        }
        const float mine = lane < p.top ? expf(key_value(my_key) - best) / sum : 0.0f;
        float top_sum = mine;
#pragma unroll
        for (int o = 16; o; o >>= 1) top_sum += __shfl_xor_sync(0xffffffffu, top_sum, o);
        if (lane < p.top) {
            const int slot = warp * p.top + lane;
            sh.slot[my_expert][warp] = (int16_t)slot;
            atomicOr(&sh.chosen[my_expert >> 5], 1u << (my_expert & 31));
            p.ids[slot] = my_expert;
            p.weights[slot] = p.renormalise ? mine / top_sum : mine;
        }
    }
    __syncthreads();
    int n_active = 0, before = 0;
    {
        const int e = (int)threadIdx.x;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t m = sh.chosen[i];
            if (i < (e >> 5)) before += __popc(m);
            n_active += __popc(m);
        }
        if (e < p.E && (sh.chosen[e >> 5] >> (e & 31) & 1))
            sh.active[before + __popc(sh.chosen[e >> 5] & ((1u << (e & 31)) - 1))] = e;
    }
    __syncthreads();
    auto entry = [&](int at, int expert, int slot, bool mine, int place, int tokens) {
        if (mine) p.route->list[at][place] = (int16_t)slot;
        p.route->slot[at][lane] = (int16_t)(mine ? slot : -1);
        if (lane == 0) p.route->head[at] = expert | tokens << 16;
    };
    // Up to kMaxEntryTokens tokens, an expert is one entry.
    const bool one = p.T <= kMaxEntryTokens;
    for (int a = warp; a < n_active; a += WARPS) {
        const int e = sh.active[a], slot = sh.slot[e][lane];
        const uint32_t m = __ballot_sync(0xffffffffu, slot >= 0);
        if (one) entry(a, e, slot, slot >= 0, __popc(m & ((1u << lane) - 1)), __popc(m));
        else if (lane == 0) sh.tokens[a] = m;
    }
    int entries = n_active;
    if (!one) {
        __syncthreads();
        auto chunks = [&](int a) { return (__popc(sh.tokens[a]) + kMaxEntryTokens - 1) / kMaxEntryTokens; };
        auto entries_before = [&](int a) {
            int n = 0;
            for (int b = lane; b < a; b += 32) n += chunks(b);
            return __reduce_add_sync(0xffffffffu, n);
        };
        for (int a = warp; a < n_active; a += WARPS) {
            const int e = sh.active[a], slot = sh.slot[e][lane], base = entries_before(a);
            const uint32_t m = sh.tokens[a];
            const int n = __popc(m), place = __popc(m & ((1u << lane) - 1));
            for (int c = 0; c * kMaxEntryTokens < n; ++c) {
                const int at = place - c * kMaxEntryTokens;
                entry(base + c, e, slot, slot >= 0 && at >= 0 && at < kMaxEntryTokens, at,
                      min(kMaxEntryTokens, n - c * kMaxEntryTokens));
            }
        }
        if (warp == WARPS - 1) entries = entries_before(n_active);
    }
    if (warp == WARPS - 1) {
        for (int b = entries + lane; b < kMaxExperts; b += 32) p.route->head[b] = 0;
        if (lane == 0) p.route->n_entries = entries;
    }
}

template <int PER>
__global__ void __launch_bounds__(32 * kMaxTokens) route_kernel(const RouteParams p) {
    __shared__ RouteShared sh;
    route_prepare<kMaxTokens>(p, sh);
    pdl_wait();
    pdl_launch_dependents();
    route_body<PER, kMaxTokens>(p, sh);
}

// Router product and routing of few experts and tokens in one launch: a cluster of
// eight blocks shares out the experts and the first block routes. It saves the host
// a launch, which decides small layers that are called one by one, and costs the
// device a little. Called / replayed, us, in one launch and in two: 1 token 8/2
// 1024x512 18.3 and 20.1 / 15.2 and 15.2, 2 tokens 18.3 and 20.1 / 16.4 and 16.0,
// 1 token 32/4 2048x704 18.7 and 20.0 / 17.2 and 17.1; 4 tokens 32/4 2048x704 24.2
// and 23.7 / 22.8 and 22.1; but 1 token 64/8 2048x1024 21.9 and 20.8 / 21.3 and 19.4,
// 4 tokens 64/8 38.1 and 35.2 replayed, so it stops at 65536 weights.
constexpr int kFewBlocks = 8;
constexpr int kFewWarps = 16;
constexpr int kFewPer = 4;  // at most 128 experts

template <typename XT, int NX>
__global__ void __cluster_dims__(kFewBlocks, 1, 1) __launch_bounds__(32 * (kFewWarps + 1))
    few_route_kernel(const RouteParams p, int sub_log2) {
    __shared__ RouteShared sh;
    __shared__ float part[kFewWarps][NX];
    const int rank = (int)cluster_ctarank(), warp = (int)warp_id_uniform(), lane = (int)lane_id();
    if (rank == 0) route_prepare<kFewWarps + 1>(p, sh);
    pdl_wait();
    pdl_launch_dependents();
    // 2^sub_log2 warps share out an expert's K, so that a block's experts take
    // all of its warps.
    // The last warp finds the tokens' magnitudes meanwhile.
    const bool dots = warp < kFewWarps;
    if (!dots)
        for (int t = rank; t < p.T; t += kFewBlocks) token_amax<XT>(p, t);
    const int subs = 1 << sub_log2, mine = warp >> sub_log2, sub = warp & (subs - 1);
    for (int e0 = rank; e0 < p.E; e0 += kFewBlocks * (kFewWarps >> sub_log2)) {
        const int e = e0 + kFewBlocks * mine;
        float acc[NX] = {};
        if (dots && e < p.E) router_dots<XT, NX>(p, e, 0, p.T, (sub * 32 + lane) * 8, subs * 256, acc);
#pragma unroll
        for (int i = 0; i < NX; ++i)
            if (dots && lane == i) part[warp][i] = acc[i];
        __syncthreads();
        if (dots && sub == 0 && e < p.E && lane < p.T) {
            float v = 0.0f;
            for (int q = 0; q < subs; ++q) v += part[warp + q][lane];
            p.logits[(size_t)lane * p.E + e] = v;
        }
        __syncthreads();
    }
    __syncwarp();
    cluster_sync();
    if (rank == 0) route_body<kFewPer, kFewWarps + 1>(p, sh);
}

static bool few_experts(int T, int E, int D) { return T <= 4 && E <= 32 * kFewPer && (long long)E * D <= 1 << 16; }

// ---------------------------------------------------------------- resident experts' products
// With enough work for every SM, one block per SM walks over the items (an
// entry's two tiles: gate and up of 128 features, or 256 rows of down), and its
// roles run ahead of one another from item to item: the copies and the
// conversion fill the rings with the next item's stages while the accumulators
// (two sets) drain. stream_kernel starts a block per item instead, which costs
// about 4 us of an SM's stream each; there K is split over a cluster, which is
// what few items need.
//   warp 0 copies, warp 1 MMAs, warps 2..17 convert, warps 18..21 epilogue
// (8 / 12 / 16 converting warps, us: 32 tokens 32/8 4096x2048 165 / 145 / 137, 64/6
// 4096x2048 176 / 167 / 166, 16 tokens 16/2 4096x4096 FP16 90.2 / 90.1 / 91.8, 8 tokens
// 128/8 4096x768 66.6 / 67.0 / 68.2.)
constexpr int kItemConvWarps = 16;
constexpr int kItemThreads = 32 * (6 + kItemConvWarps);

struct ItemControl {
    uint64_t full[kMaxSlots];
    uint64_t empty[kMaxSlots];
    uint64_t acc_full[2];
    uint64_t acc_empty[2];
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
};

template <bool GATE_UP, typename T>
__global__ void __launch_bounds__(kItemThreads, 1)
    item_kernel(const __grid_constant__ CUtensorMap tm0, const __grid_constant__ CUtensorMap tm1,
                const __grid_constant__ Params p) {
    using XT = std::conditional_t<GATE_UP, T, float>;
    constexpr int kPlanes = kPlanesOf<T>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    ItemControl& sm = *reinterpret_cast<ItemControl*>(ring + p.ring_bytes);
    const uint32_t warp = warp_id_uniform();
    const uint32_t lane = lane_id();
    const Geometry g = p.geo[0];  // for the most tokens an entry can have
    uint8_t* const b_ring = ring + (size_t)g.w_slots * kWSlot;

    if (threadIdx.x < kMaxSlots) {
        mbar_init(&sm.full[threadIdx.x], 1 + kItemConvWarps);
        mbar_init(&sm.empty[threadIdx.x], 1);
        if (threadIdx.x < 2) {
            mbar_init(&sm.acc_full[threadIdx.x], 1);
            mbar_init(&sm.acc_empty[threadIdx.x], 4);
        }
        if (threadIdx.x == 0) {
            mbar_init(&sm.drain, 1);
            sm.abort = 0;
            tma_prefetch_desc(&tm0);
            if (GATE_UP) tma_prefetch_desc(&tm1);
        }
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(&sm.tmem_base, p.tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t sfa_col0 = tmem + 4u * g.acc_cols, sfb_col0 = sfa_col0 + (uint32_t)g.w_slots * 16;
    const int groups = GATE_UP ? p.tiles : (p.tiles + 1) / 2;
    const int items = p.route->n_entries * groups;

    if (warp == 0) {
        // ------------------------------------------------------------ copies
        if (lane == 0) {
            Cursor c;
            long issued = 0;
            bool ok = true;
            const size_t sf_matrix = (size_t)p.tiles * (size_t)p.kblocks * 512;
            for (int it = (int)blockIdx.x; it < items && ok; it += (int)gridDim.x) {
                const int group = it % groups, expert = p.route->head[it / groups] & 0xFFFF;
                const int tile0 = GATE_UP ? group : 2 * group;
                const int nw = GATE_UP || tile0 + 1 < p.tiles ? 2 : 1;
                for (int kb = 0; kb < p.k_stages && ok; ++kb) {
                    const uint32_t sf_bytes = 512u * (uint32_t)min(4, p.kblocks - 4 * kb);
                    for (int h = 0; h < 2; ++h) {
                        if (!mbar_wait(&sm.empty[c.slot], c.phase ^ 1u, &sm.abort, 0x0701)) {
                            ok = false;
                            break;
                        }
                        uint64_t* full = &sm.full[c.slot];
                        if (h < nw) {
                            const bool up = GATE_UP && h == 1;
                            const int tile = GATE_UP ? tile0 : tile0 + h;
                            uint8_t* st = ring + (size_t)c.slot * kWSlot;
                            const uint8_t* sf = (up ? p.sf1 : p.sf0) + (size_t)expert * sf_matrix +
                                                ((size_t)tile * p.kblocks + (size_t)kb * 4) * 512;
                            mbar_arrive_expect_tx(full, kWBytes + sf_bytes);
                            tma_load_3d(st, up ? &tm1 : &tm0, full, kb * 128, tile * kTileRows, expert);
                            bulk_load(st + kWBytes, sf, sf_bytes, full);
                        } else {
                            mbar_arrive(full);  // an odd last tile: its neighbour's slot stays as it is
                        }
                        ++issued;
                        c.advance(g.w_slots);
                    }
                }
            }
            if (!ok || *(volatile int*)&sm.abort) {
                int dummy = 0;
                for (long j = issued > g.w_slots ? issued - g.w_slots : 0; j < issued; ++j)
                    mbar_wait(&sm.full[j % g.w_slots], (uint32_t)(j / g.w_slots) & 1u, &dummy, 0x0702, 100000000ull);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        const uint64_t op_desc = desc_kmajor_sw128(0), sf_desc = smem_desc(0, 0, 128, 0);
        const uint32_t sfb_step = g.sfb_step >> 4;
        Cursor w, b, acc;
        bool ok = true;
        for (int it = (int)blockIdx.x; it < items && ok; it += (int)gridDim.x) {
            const int ntok = p.route->head[it / groups] >> 16;
            const int tile0 = GATE_UP ? 0 : 2 * (it % groups);
            const int nw = GATE_UP || tile0 + 1 < p.tiles ? 2 : 1;
            const uint32_t idesc = idesc_nvf4(kTileRows, (kPlanes * ntok + 7) & ~7);
            if (!mbar_wait(&sm.acc_empty[acc.slot], acc.phase ^ 1u, &sm.abort, 0x0711)) break;
            __syncwarp();
            tc_fence_after();
            for (int kb = 0; kb < p.k_stages && ok; ++kb) {
                const int nblk = min(4, p.kblocks - 4 * kb);
                const uint32_t b_addr = smem_u32(b_ring) + (uint32_t)b.slot * g.b_slot;
                const uint64_t b_desc = op_desc + (b_addr >> 4);
                const uint64_t sfb_desc = sf_desc + ((b_addr + (uint32_t)g.nb * 128) >> 4);
                const uint32_t sfb_col = sfb_col0 + (uint32_t)b.slot * g.sfb_cols;
                for (int h = 0; h < 2; ++h) {
                    ok = mbar_wait(&sm.full[w.slot], w.phase, &sm.abort, 0x0712);
                    if (!ok) break;
                    __syncwarp();
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(ring) + (uint32_t)w.slot * kWSlot;
                    const uint64_t a_desc = op_desc + (a_addr >> 4);
                    const uint32_t sfa_col = sfa_col0 + (uint32_t)w.slot * 16;
                    const uint32_t d = tmem + (uint32_t)(2 * acc.slot + h) * g.acc_cols;
                    const uint64_t sfa_desc = sf_desc + ((a_addr + kWBytes) >> 4);
                    auto scales = [&](int j) {
                        if (h == 0) tmem_cp_32x128b_warpx4(sfb_col + 4 * j, sfb_desc + sfb_step * j);
                        tmem_cp_32x128b_warpx4(sfa_col + 4 * j, sfa_desc + 32 * j);
                    };
                    auto product = [&](int j) {
                        mma_nvf4(d, a_desc + 2 * j, b_desc + 2 * j, idesc, sfa_col + 4 * j, sfb_col + 4 * j,
                                 (kb | j) != 0);
                    };
                    if (elect_one()) {
                        if (h < nw) {
                            if (nblk == 4) {
#pragma unroll
                                for (int j = 0; j < 4; ++j) scales(j);
#pragma unroll
                                for (int j = 0; j < 4; ++j) product(j);
                            } else {
                                for (int j = 0; j < nblk; ++j) scales(j);
                                for (int j = 0; j < nblk; ++j) product(j);
                            }
                        }
                        tc_commit(&sm.empty[w.slot]);
                    }
                    __syncwarp();
                    w.advance(g.w_slots);
                }
                b.advance(g.b_slots);
            }
            if (ok && elect_one()) tc_commit(&sm.acc_full[acc.slot]);
            __syncwarp();
            acc.advance(2);
        }
        // Every MMA issued completes before TMEM is freed.
        if (elect_one()) tc_commit(&sm.drain);
        __syncwarp();
        int dummy = 0;
        mbar_wait(&sm.drain, 0, &dummy, 0x0713, 100000000ull);
        __syncwarp();
    } else if (warp < 2 + kItemConvWarps) {
        // ------------------------------------------------------------ activations
        // Unit u = kb * tokens + t of an item is warp u % 16's.
        const int w = (int)warp - 2;
        struct Unit {
            int it, kb, t, ntok, step_kb, step_t, entry;
        };
        auto enter = [&](Unit& u) {  // the unit is the first of the item, if any is left
            while (u.it < items) {
                u.entry = u.it / groups;
                u.ntok = p.route->head[u.entry] >> 16;
                const uint32_t inverse = p.inverse[u.ntok];
                u.step_kb = (int)(kItemConvWarps * inverse >> 16);
                u.step_t = kItemConvWarps - u.step_kb * u.ntok;
                u.kb = (int)((uint32_t)w * inverse >> 16);
                u.t = w - u.kb * u.ntok;
                if (u.kb < p.k_stages) return;
                u.it += (int)gridDim.x;
            }
        };
        auto next_unit = [&](Unit& u) {
            u.kb += u.step_kb;
            u.t += u.step_t;
            if (u.t >= u.ntok) {
                u.t -= u.ntok;
                ++u.kb;
            }
            if (u.kb >= p.k_stages) {
                u.it += (int)gridDim.x;
                enter(u);
            }
        };
        // The lane's eight elements and the token's anchor.
        auto load = [&](const Unit& u, uint4 (&r)[2], int& anchor) {
            r[0] = r[1] = make_uint4(0, 0, 0, 0);
            if (u.it >= items) return;
            const int slot = p.route->list[u.entry][u.t];
            const int row = GATE_UP ? slot / p.top : slot;
            const int k = u.kb * kStageK + (int)lane * 8;
            if (k < p.K) load_raw(static_cast<const XT*>(p.X) + (size_t)row * p.ldx + k, p.x_vec != 0, r);
            anchor = anchor_of<kPlanes>(p.amax[slot / p.top]);
        };
        Unit cur;
        cur.it = (int)blockIdx.x;
        enter(cur);
        Unit ahead = cur;
        uint4 r0[2], r1[2];
        int a0 = 0, a1 = 0;
        load(ahead, r0, a0);
        if (ahead.it < items) next_unit(ahead);
        load(ahead, r1, a1);
        Cursor c, b;
        bool ok = true;
        for (int it = (int)blockIdx.x; it < items && ok; it += (int)gridDim.x) {
            for (int kb = 0; kb < p.k_stages; ++kb) {
                const int slot0 = c.slot;
                ok = mbar_wait(&sm.empty[c.slot], c.phase ^ 1u, &sm.abort, 0x0721);
                c.advance(g.w_slots);
                const int slot1 = c.slot;
                ok = ok && mbar_wait(&sm.empty[c.slot], c.phase ^ 1u, &sm.abort, 0x0722);
                c.advance(g.w_slots);
                if (!ok) break;
                __syncwarp();
                if (cur.it == it && cur.kb == kb) {
                    uint8_t* b_rows = b_ring + (size_t)b.slot * g.b_slot;
                    uint8_t* sfb = b_rows + (size_t)g.nb * 128;
                    const bool inside = kb * kStageK + (int)lane * 8 < p.K;
                    do {
                        float v[8];
                        widen<XT>(r0, v);
                        const int t = cur.t, anchor = a0;
                        r0[0] = r1[0];
                        r0[1] = r1[1];
                        a0 = a1;
                        next_unit(cur);
                        if (ahead.it < items) next_unit(ahead);
                        load(ahead, r1, a1);
                        convert<kPlanes>(v, anchor, t, inside, b_rows, sfb, g.sfb_step, lane);
                    } while (cur.it == it && cur.kb == kb);
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                if (lane == 0) {
                    mbar_arrive(&sm.full[slot0]);
                    mbar_arrive(&sm.full[slot1]);
                }
                b.advance(g.b_slots);
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ epilogue
        // A thread has one row of both tiles.
        const uint32_t quarter = warp & 3u;
        const int row = (int)(quarter * 32 + lane);
        Cursor acc;
        for (int it = (int)blockIdx.x; it < items; it += (int)gridDim.x) {
            const int entry = it / groups, group = it % groups, head = p.route->head[entry];
            const int ntok = head >> 16, expert = head & 0xFFFF;
            // Lane t: token t's slot, magnitude and, for gate / up, what h is scaled by.
            const int my_slot = (int)lane < ntok ? p.route->list[entry][lane] : 0;
            const uint32_t my_max = (int)lane < ntok ? p.amax[my_slot / p.top] : 0u;
            float ag = 1.0f, au = 1.0f, my_scale = 1.0f;
            if constexpr (GATE_UP) {
                ag = p.alpha0[expert];
                au = p.alpha1[expert];
                my_scale = (int)lane < ntok ? p.weights[my_slot] * p.alpha2[expert] : 0.0f;
            }
            if (!mbar_wait_sleepy(&sm.acc_full[acc.slot], acc.phase, &sm.abort, 0x0731, false)) break;
            __syncwarp();
            tc_fence_after();
            const uint32_t acc0 = tmem + ((quarter * 32u) << 16) + (uint32_t)(2 * acc.slot) * g.acc_cols;
            // Four tokens' columns of both tiles fit a thread's registers up to six planes.
            constexpr int kAtOnce = kPlanes < 7 ? 4 : 2, kLoads = (kPlanes * kAtOnce + 7) / 8;
            for (int t0 = 0; t0 < ntok; t0 += kAtOnce) {
                uint32_t c0[kLoads][8], c1[kLoads][8];
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    tmem_ld_32x32b_x8(acc0 + (uint32_t)(kPlanes * t0 + 8 * i), c0[i]);
                    tmem_ld_32x32b_x8(acc0 + g.acc_cols + (uint32_t)(kPlanes * t0 + 8 * i), c1[i]);
                }
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    if (t0 + i >= ntok) continue;
                    auto col = [&](const uint32_t (&c)[kLoads][8], int n) { return __uint_as_float(c[n >> 3][n & 7]); };
                    float s = col(c0, kPlanes * i + kPlanes - 1), u = col(c1, kPlanes * i + kPlanes - 1);
#pragma unroll
                    for (int q = kPlanes - 2; q >= 0; --q) {
                        s = __fmaf_rn(s, 0.125f, col(c0, kPlanes * i + q));
                        u = __fmaf_rn(u, 0.125f, col(c1, kPlanes * i + q));
                    }
                    const uint32_t mb = __shfl_sync(0xffffffffu, my_max, t0 + i);
                    const int slot = __shfl_sync(0xffffffffu, my_slot, t0 + i);
                    const float unit = __uint_as_float((uint32_t)(anchor_of<kPlanes>(mb) - 8 + 127) << 23);
                    s = s * ag * unit;
                    u = u * au * unit;
                    if (mb >= kInfBits) s = u = __uint_as_float(0x7FC00000u);
                    float* y = static_cast<float*>(p.Y) + (size_t)slot * p.ldy;
                    if constexpr (GATE_UP) {
                        const int n = group * kTileRows + row;
                        const float h = s / (1.0f + expf(-s)) * u * __shfl_sync(0xffffffffu, my_scale, t0 + i);
                        if (n < p.N) y[n] = h;
                        const uint32_t m = __reduce_max_sync(0xffffffffu, n < p.N ? __float_as_uint(h) & 0x7FFFFFFFu : 0u);
                        if (lane == 0 && m) atomicMax(&p.amax_out[slot / p.top], m);
                    } else {
                        const int n = 2 * group * kTileRows + row;
                        if (n < p.N) y[n] = s;
                        if (n + kTileRows < p.N) y[n + kTileRows] = u;
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.acc_empty[acc.slot]);
            acc.advance(2);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, p.tmem_cols);
    }
}

static size_t set_item_shape(Params& p, int planes, int entry_tokens) {
    for (int t = 1; t <= kMaxTokens; ++t) p.inverse[t] = 65536u / (uint32_t)t + 1;
    const Shape s = item_shape(p.geo, planes, entry_tokens, sizeof(ItemControl));
    p.ring_bytes = s.ring_bytes;
    p.tmem_cols = s.tmem_cols;
    return s.smem;
}

template <bool GATE_UP, typename T>
static int launch_items(const CUtensorMap& tm0, const CUtensorMap& tm1, const Params& p, size_t smem, int blocks,
                        cudaStream_t stream) {
    static thread_local uint64_t configured = 0;  // bit per device
    return launch_clusters(item_kernel<GATE_UP, T>, &configured, blocks, kItemThreads, 1, smem, stream, tm0, tm1, p);
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

// Whether gate and up run as resident blocks over `items`: from two for every SM.
// Measured, us of the layer, a block per item / resident: 976 items (32 tokens,
// 64/6, 4096x2048) 177 / 165, 448 (16, 16/2, 4096x4096) 89 / 89, 390 (8, 64/6,
// 2048x1408) 57 / 49, 310 (8, 128/8, 4096x768) 80 / 68, but 256 (8, 8/2, 4096x4096)
// 53 / 53 and (32, 8/2, 4096x4096) 82 / 79, 200 (16, 64/6, 2048x512) 36 / 39, 168 (4,
// 64/8, 4096x768) 50 / 56, 145 (4, 32/4, 4096x1408) 44 / 50, 64 (16, 8/2, 2048x1024)
// 24 / 27.
static bool use_gate_items(double items, int sm_count) { return items >= 2.0 * sm_count; }

// Whether down runs as resident blocks with a sum per slot, or accumulates over the
// experts, which splits K further but converts and multiplies for every token in
// every stage: by the tiles an SM streams, the second's weighed by its tokens.
// Measured, us of the layer, accumulating / resident: 1 token 8/2 4096x14336
// 48 / 71, 64/8 2048x1024 19.3 / 20.8; 2 tokens 16/4 4096x2048 31.4 / 32.2; 3 tokens
// 39 / 42, 4 tokens 52 / 57, 5 tokens 56 / 60, 6 tokens 59 / 62; 4 tokens 32/4 2048x704
// 22.8 / 21.6, 5 tokens 23.9 / 22.3, 6 tokens 26.6 / 25.3; 64/8 2048x1024 5 tokens
// 39.5 / 38.0, 7 tokens 52 / 47; 8/2 4096x4096 5 tokens 54 / 56, 6 tokens 63 / 60, 8
// tokens 66 / 53, 32 tokens 147 / 82; 8 tokens 8/1 1024x14336 70 / 63; 16 tokens 8/2
// 2048x1024 28.5 / 23.1. Where the two are within a tenth, some sizes have the
// slower one (3, 5 and 6 tokens 16/4; 8 tokens 8/1).
static bool use_down_items(int T, double active, int tiles, int k_stages, int split, int sm_count) {
    const int pairs = (tiles + 1) / 2;
    const double resident = 2.0 * k_stages * ceil(active * pairs / sm_count);
    const double accumulated = ceil(active * k_stages / split) * ceil((double)tiles * split / sm_count);
    return resident <= accumulated * (T <= 4 ? 0.8 : 1.0 + T / 8.0);
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

    const int entry_tokens = c.T < kMaxEntryTokens ? c.T : kMaxEntryTokens;

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
    Params o = g;
    o.X = g.Y;
    o.amax = g.amax_out;
    o.sf0 = c.sf_down;
    o.N = c.D;
    o.K = c.F;
    o.ldx = c.F;
    o.x_vec = 1;
    o.tiles = (c.D + kTileRows - 1) / kTileRows;
    o.k_stages = (c.F + kStageK - 1) / kStageK;
    o.kblocks = c.F / 64;
    size_t g_smem, o_smem;
    const bool g_items = use_gate_items(active * g.tiles, d.sm_count);
    if (g_items) {
        g_smem = set_item_shape(g, kPlanesOf<XT>, entry_tokens);
    } else {
        const Shape s = set_shape(g, kPlanesOf<XT>, entry_tokens, true, 2, Fill::Convert, g.k_stages);
        g_smem = s.smem;
        g.split_log2 = choose_split_log2(g.tiles * active, 2.0 * g.k_stages, d.sm_count, s.per_sm);
    }
    const Shape os = set_shape(o, kPlanesOf<XT>, c.T, false, 1, Fill::Convert, o.k_stages * max_entries);
    o.split_log2 = choose_split_log2(o.tiles, o.k_stages * active, d.sm_count, os.per_sm);
    const bool o_items = use_down_items(c.T, active, o.tiles, o.k_stages, 1 << o.split_log2, d.sm_count);
    o_smem = o_items ? set_item_shape(o, kPlanesOf<XT>, entry_tokens) : os.smem;
    o.Y = o_items ? static_cast<void*>(ws + l.part) : c.y;
    o.ldy = o_items ? c.D : c.ldy;
    if (g_smem > (size_t)d.max_smem_optin || o_smem > (size_t)d.max_smem_optin) return GPLK_STATUS_UNSUPPORTED;

    CUtensorMap tg, tu, td;
    int st = encode_weights(&tg, c.gate, c.F, c.E, c.D);
    if (st == GPLK_STATUS_OK) st = encode_weights(&tu, c.up, c.F, c.E, c.D);
    if (st == GPLK_STATUS_OK) st = encode_weights(&td, c.down, c.D, c.E, c.F);
    if (st != GPLK_STATUS_OK) return st;

    auto router = [&](auto kernel, int nx) {
        return launch_status(launch_pdl(kernel, dim3(c.E + 1, (c.T + nx - 1) / nx), dim3(kRouterThreads), 0, stream, r));
    };
    if (few_experts(c.T, c.E, c.D)) {
        int sub_log2 = 4;
        while (sub_log2 > 0 && (c.E + kFewBlocks - 1) / kFewBlocks > kFewWarps >> sub_log2) --sub_log2;
        st = launch_status(launch_pdl(c.T == 1 ? few_route_kernel<XT, 1> : few_route_kernel<XT, 4>, dim3(kFewBlocks),
                                      dim3(32 * (kFewWarps + 1)), 0, stream, r, sub_log2));
    } else {
        st = c.T == 1   ? router(router_kernel<XT, 1>, 1)
             : c.T <= 4 ? router(router_kernel<XT, 4>, 4)
                        : router(router_kernel<XT, 8>, 8);
        if (st == GPLK_STATUS_OK)
            st = launch_status(launch_pdl(c.E <= 128 ? route_kernel<4> : route_kernel<kPer>, dim3(1),
                                          dim3(32 * kMaxTokens), 0, stream, r));
    }
    if (st == GPLK_STATUS_OK)
        st = g_items ? launch_items<true, XT>(tg, tu, g, g_smem, d.sm_count, stream)
                     : launch_stream<Mode::GateUp, XT, float>(tg, tu, g, g_smem, max_entries * g.tiles, stream);
    if (st != GPLK_STATUS_OK) return st;
    if (!o_items) return launch_stream<Mode::Down, float, XT>(td, td, o, o_smem, o.tiles, stream);
    st = launch_items<false, XT>(td, td, o, o_smem, d.sm_count, stream);
    if (st != GPLK_STATUS_OK) return st;
    return launch_status(launch_pdl(combine_kernel<XT>, dim3((c.D + 1023) / 1024, c.T), dim3(256), 0, stream,
                                    static_cast<const float*>(o.Y), static_cast<XT*>(c.y), c.top, c.D, c.ldy));
}

}  // namespace moe
}  // namespace gplk

extern "C" size_t gplk_moe_nvfp4_workspace_bytes(int T, int E, int top, int D, int F) {
    using namespace gplk;
    return T > 0 && moe::takes(T, E, top, D, F) ? moe::layout(T, E, top, D, F).total : 0;
}

extern "C" int gplk_moe_nvfp4(const gplk_moe_cfg* cfg, cudaStream_t stream) {
    using namespace gplk;
    using namespace gplk::fewtok;
    if (!cfg) return GPLK_STATUS_BAD_ARG;
    const gplk_moe_cfg& c = *cfg;
    if (!moe::takes(c.T, c.E, c.top, c.D, c.F)) return GPLK_STATUS_BAD_ARG;
    if (c.dtype != GPLK_DTYPE_BF16 && c.dtype != GPLK_DTYPE_F16) return GPLK_STATUS_BAD_ARG;
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
