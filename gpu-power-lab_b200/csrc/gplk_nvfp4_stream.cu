// gplk_nvfp4_stream.cu - the main loop of the products of a few tokens with NVFP4
// weights (gplk_gemv_nvfp4.cu, gplk_moe_nvfp4.cu):
//   y[t][n] = sum_k x[t][k] * sf[n][k / 16] * w[n][k]
// E2M1 weights and UE4M3 scales in the layout gplk_gemm_nvfp4_tn reads, 16-bit
// or FP32 activations, FP32 sums.
//
// What bounds it: every weight is read once for 2 T operations, so HBM. A
// B200 reads 46 weights per SM and clock; decoding them on the CUDA cores
// takes about that many issue slots (one warp per row with FP32 FMAs measured
// 0.56 TB/s at one token, 16384 x 8192). So the weights are not decoded at all:
// they go from HBM through TMA to the block-scaled tensor-core MMA
// (kind::mxf4nvf4), codes and scales as they lie, and the activations are
// brought to its operand format instead:
//
//   Within a 16-group of a token, 2^b the power of two at or below its largest
//   magnitude, x is rounded to a multiple of 2^b * 2^-(3 P - 2) and written in P
//   balanced base-8 digits  x = 2^b * sum_p d_p / 2 * 8^-p,  p = 0..P - 1,
//   d_0 in -4..4, the others in -4..3. Every d / 2 is an E2M1 value, so digit p
//   of all of k is one E2M1 row ("plane") of the MMA's B operand, and 2^b,
//   relative to the token's largest magnitude 2^A, is the group's UE4M3 scale.
//   P is 6 for BF16 and 7 for FP16: with either, a value down to 2^-9 of its
//   group's 2^b keeps all of its bits (8 and 11), and a smaller one is off by at
//   most 2^-17 and 2^-20 of 2^b, half a step. (In groups 2^14 and more below the
//   token's largest magnitude: 2^-31 and 2^-34 of that.) An MoE layer's h, FP32,
//   is taken to the planes of the layer's type. With one plane less, values next
//   to an outlier lose bits that their type has; it takes as long for a few
//   tokens, and for many of them 32x16384x16384 38.7 instead of 40.2 us, a layer
//   of 32 tokens 8/2 4096x4096 70 instead of 80. The accumulator column of each
//   (token, plane) is exact products in FP32 sums; the epilogue adds 8^-p times
//   the planes' columns.
//
// So T tokens are an MMA of N = P T columns (padded to 8), at most 224 of the
// 256 an instruction takes.
//
// Layout of the work. A block owns 128 weight rows (the MMA's M), or two such
// tiles that share the activations' rows (gate and up of an expert), and a slice
// of K; blocks of a cluster share the rows, split K, and add their partial sums
// in rank order through distributed shared memory, so the bits do not depend on
// timing. Two blocks share an SM where TMEM allows: one's start and end hide
// behind the other's stream.
//   warp 0      TMA producer: 128 rows x 128 bytes of codes and up to 2 KiB of
//               scales (256 elements of K) per slot of the weights' ring
//   warp 1      owns TMEM, copies the scales there and issues one MMA per 64
//               elements of K and tile
//   warps 2..9  convert the same 256 elements of every token into a slot of
//               the activations' ring (a warp per token and slot); warps 2..5
//               then read the accumulators, and all warps add the slices.
//               An Image kernel copies what another kernel converted, and has
//               warps 2..5 only.
// The MMA warp runs its loop converged and elects the issuing lane: with
// addresses and descriptors in uniform registers, 65536 x 8192 at one token
// takes 49 us (6.2 TB/s); issued from a lane of a diverged warp it took 76 us.
// Smaller calls have some 4 us of start and end. At 32 tokens what counts is the
// weights on their way, since activations take half of the shared memory (16384 x
// 16384: 40 us; an earlier build's 42 were 37 without any MMA, scale copy or
// activation), and, with more tiles than SMs, the rounds of blocks, each with a
// start and an end (65536 x 8192: 102 us against 47 at HBM's rate).
// Every mbarrier wait is bounded, as everywhere in this library.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "gplk_nvfp4_shape.cuh"
#include "gplk_ptx.cuh"

namespace gplk {
namespace fewtok {

constexpr int kMaxExperts = 512;
constexpr int kMaxTop = 16;
constexpr int kConvWarps = 8;
constexpr int kPlanesBF16 = 6, kPlanesF16 = 7;

// Gemv: all tokens against one matrix. GateUp: tokens of a chosen expert against
// its gate and up matrices. Down: all tokens against every chosen expert's down
// matrix, accumulated over the experts.
enum class Mode { Gemv, GateUp, Down };

// Planes of the activations in a product of type T.
template <typename T>
constexpr int kPlanesOf = std::is_same<T, __half>::value ? kPlanesF16 : kPlanesBF16;

template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    return static_cast<T>(v);
}

// ---------------------------------------------------------------- routing tables (MoE)
// Written by the route kernel into the layer's workspace. An entry is a chosen
// expert with up to kMaxEntryTokens of its tokens; experts ascend.
struct Route {
    int n_entries;
    int head[kMaxExperts];                      // expert | tokens << 16; 0 behind the last entry
    int16_t list[kMaxExperts][16];              // the tokens' slots (token * top + rank), ascending
    int16_t slot[kMaxExperts][kMaxTokens];      // slot of token t in entry a, or -1
};

struct Params {
    const void* X;       // activations (16-bit rows; for down: FP32 h rows by slot)
    const uint8_t* sf0;  // scales: W, gate or down
    const uint8_t* sf1;  // GateUp: up
    const float* alpha0; // Gemv: one; GateUp: gate's, per expert
    const float* alpha1; // GateUp: up's
    const float* alpha2; // GateUp: down's, folded into h
    void* Y;             // T rows; from gate and up, and from resident down blocks: FP32 rows by slot
    const void* R;
    const Route* route;
    const float* weights;  // MoE: per slot
    const uint8_t* image;  // Image kernels: the converted activations, by stage
    const uint32_t* amax;  // bits of each token's largest magnitude, or NULL: this kernel finds its slice's
    uint32_t* amax_out;    // GateUp: h's, by token
    int T, N, K, ldx, ldy, ldr;
    int x_vec;           // rows of X are 16-byte aligned
    int top;
    uint32_t inverse[kMaxTokens + 1];  // 2^16 / n + 1
    int tiles;           // 128-row tiles of one matrix
    int k_stages;        // stages of one matrix row
    int kblocks;         // K / 64
    int split_log2;      // slices of K, the cluster's size
    uint32_t ring_bytes; // shared memory of the two rings
    uint32_t tmem_cols;
    Geometry geo[kMaxEntryTokens];  // per-expert modes: by tokens - 1; else the first, for T tokens
};

struct Control {
    uint64_t full[kMaxSlots];   // by weights' slot
    uint64_t empty[kMaxSlots];
    uint64_t acc_full;
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
    uint32_t amax[kMaxTokens];  // bits of the largest magnitude in this block's slice
    int16_t slot[kMaxTokens];   // per-expert modes: slots of the block's tokens
    uint8_t dirty[kMaxSlots][kMaxTokens];  // Down: the slot holds digits of that token
};

// A ring position.
struct Cursor {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void advance(int slots) {
        if (++slot == slots) {
            slot = 0;
            phase ^= 1u;
        }
    }
};

__device__ __forceinline__ void tmem_ld_32x32b_x8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}

// True in one lane of a converged warp, always the same one.
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(e));
    return e != 0;
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// Sum of the four floats at the same place of the cluster's n blocks (1, 2, 4 or
// 8), added in rank order, four loads on their way at a time.
__device__ __forceinline__ float4 sum_cluster(uint32_t addr, int n) {
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int c0 = 0; c0 < 8; c0 += 4) {
        if (c0 >= n) break;
        float4 v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (c < n) v[c] = ld_cluster_f32x4(mapa_shared(addr, (uint32_t)(c0 + c)));
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (c < n) {
                s.x += v[c].x;
                s.y += v[c].y;
                s.z += v[c].z;
                s.w += v[c].w;
            }
    }
    return s;
}

// Eight consecutive activations of one lane.
template <typename XT>
__device__ __forceinline__ void load_raw(const XT* x, bool vec, uint4 (&r)[2]) {
    if constexpr (sizeof(XT) == 4) {
        r[0] = *reinterpret_cast<const uint4*>(x);
        r[1] = *reinterpret_cast<const uint4*>(x + 4);
    } else if (vec) {
        r[0] = *reinterpret_cast<const uint4*>(x);
    } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(x);
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (uint32_t)h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
        r[0] = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

template <typename XT>
__device__ __forceinline__ void widen(const uint4 (&r)[2], float (&v)[8]) {
    const uint32_t w[4] = {r[0].x, r[0].y, r[0].z, r[0].w};
    if constexpr (sizeof(XT) == 4) {
        const uint32_t w1[4] = {r[1].x, r[1].y, r[1].z, r[1].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = __uint_as_float(w[i]);
            v[4 + i] = __uint_as_float(w1[i]);
        }
    } else if constexpr (std::is_same<XT, __nv_bfloat16>::value) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = *reinterpret_cast<const __half2*>(&w[i]);
            v[2 * i] = __low2float(h);
            v[2 * i + 1] = __high2float(h);
        }
    }
}

// Bits of the largest magnitude. Integer order is magnitude order, with
// infinity and then NaN above every finite number.
__device__ __forceinline__ uint32_t max_bits(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
}

constexpr uint32_t kInfBits = 0x7F800000u;

// Exponent A of a token's largest magnitude. The anchor stays where a group 2^14
// below it is still a multiple of 2^-127: what is lost there is at most 2^-128,
// in FP32's own subnormal range.
template <int PLANES>
__device__ __forceinline__ int anchor_of(uint32_t amax_bits) {
    return max((int)(amax_bits >> 23) - 127, 3 * PLANES - 115);
}

// Eight nibbles of biased digits (0..7 for -4..3; 8 for the top digit's 4) to
// E2M1 codes of d / 2: magnitude |d| in the low three bits, sign above.
template <bool TOP>
__device__ __forceinline__ uint32_t digit_codes(uint32_t w) {
    uint32_t m = ~(w >> 2);  // 1 in the nibbles of negative digits
    if constexpr (TOP) m &= ~(w >> 3);
    m &= 0x11111111u;
    uint32_t c = ((w ^ (m * 3u)) & 0x33333333u) + m * 9u;  // negative: 8 | (3 - w) + 1
    if constexpr (TOP) c |= (w >> 1) & 0x44444444u;
    return c;
}

// Byte of row r's scale for a lane's 16-group: one block per 64 elements, with
// 16 bytes per row of 32 and 4 per further 32 rows, as the MMA wants them in TMEM.
__device__ __forceinline__ uint32_t sfb_offset(uint32_t r, uint32_t lane, uint32_t step) {
    return (r >> 7) * 2048 + (lane >> 3) * step + (r & 31) * 16 + ((r & 127) >> 5) * 4 + ((lane >> 1) & 3);
}

// One token's 256 elements of a stage, eight per lane: planes PLANES t and on
// of the stage's B rows (128-byte swizzled, K-major) and the 16 groups'
// scales. `on` is false for lanes beyond K, whose blocks no MMA reads.
template <int PLANES>
__device__ __forceinline__ void convert(const float (&v)[8], int anchor, int t, bool on, uint8_t* b_rows,
                                        uint8_t* sfb, uint32_t sfb_step, uint32_t lane) {
    static_assert(PLANES >= 5 && PLANES <= kMaxPlanes, "digits in 22 bits of a word");
    uint32_t m = max_bits(v);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));  // the other half of the 16-group
    const int b = max((int)(m >> 23) - 127, anchor - 14);
    const float scale = __uint_as_float((uint32_t)(3 * PLANES - 2 - b + 127) << 23);
    // x * scale is at most 2^(3 PLANES - 1) in magnitude; adding 1.5 * 2^23 rounds
    // it to an integer, and the bias, a 4 in every digit, makes all of them
    // non-negative.
    constexpr uint32_t kDigitBias = 4u * (((1u << 3 * PLANES) - 1) / 7);
    constexpr float kMagic = 12582912.0f + (float)kDigitBias;
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(__fmaf_rn(v[i], scale, kMagic));
    // Elements i and i + 4 (nibbles i and i + 4 of a word are 16 bits apart): bits 0
    // to 15, and 8 to 23 for the digits above.
    uint32_t low[4], high[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        low[i] = __byte_perm(u[i], u[i + 4], 0x5410);
        high[i] = __byte_perm(u[i], u[i + 4], 0x6521);
    }
    if (!on) return;
#pragma unroll
    for (int p = 0; p < PLANES; ++p) {
        const int sh = 3 * (PLANES - 1 - p);
        const bool upper = sh + (p == 0 ? 4 : 3) > 16;
        const uint32_t mask = p == 0 ? 0x000F000Fu : 0x00070007u;
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= ((upper ? high[i] >> (sh - 8) : low[i] >> sh) & mask) << (4 * i);
        w = p == 0 ? digit_codes<true>(w) : digit_codes<false>(w);
        const uint32_t r = (uint32_t)(PLANES * t + p);
        *reinterpret_cast<uint32_t*>(b_rows + (r >> 3) * 1024 + (r & 7) * 128 + (((lane >> 2) ^ (r & 7)) << 4) +
                                     (lane & 3) * 4) = w;
        if ((lane & 1) == (uint32_t)(p & 1))
            sfb[sfb_offset(r, lane, sfb_step)] = (uint8_t)((b - anchor + 15) << 3);
    }
}

// A token without a part in the stage's expert: zero digits, scale 1.
template <int PLANES>
__device__ __forceinline__ void convert_zero(int t, uint8_t* b_rows, uint8_t* sfb, uint32_t sfb_step,
                                             uint32_t lane) {
#pragma unroll
    for (int p = 0; p < PLANES; ++p) {
        const uint32_t r = (uint32_t)(PLANES * t + p);
        *reinterpret_cast<uint32_t*>(b_rows + (r >> 3) * 1024 + (r & 7) * 128 + lane * 4) = 0u;
        if ((lane & 1) == (uint32_t)(p & 1))
            sfb[sfb_offset(r, lane, sfb_step)] = 0x38;
    }
}

template <bool IMAGE>
constexpr int kThreads = IMAGE ? 64 + 128 : 64 + 32 * kConvWarps;

template <Mode M, typename XT, typename YT, bool IMAGE>
__global__ void __launch_bounds__(kThreads<IMAGE>, 2)
    stream_kernel(const __grid_constant__ CUtensorMap tm0, const __grid_constant__ CUtensorMap tm1,
                  const __grid_constant__ Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    Control& sm = *reinterpret_cast<Control*>(ring + p.ring_bytes);
    const uint32_t warp = warp_id_uniform();
    const uint32_t lane = lane_id();
    const int slice = (int)cluster_ctarank();
    const int split = 1 << p.split_log2;
    const int cid = (int)(blockIdx.x >> p.split_log2);
    constexpr bool kPerExpert = M == Mode::GateUp;
    constexpr int kPlanes = kPlanesOf<std::conditional_t<M == Mode::Down, YT, XT>>;

    // Barriers and TMEM. A slot is full when the copies have landed and the warps
    // with tokens in the stage have converted them (where the tokens are not
    // known yet: when every warp has been there).
    auto set_up = [&](int ntok) {
        if (threadIdx.x < kMaxSlots) {
            const int i = (int)threadIdx.x;
            mbar_init(&sm.full[i], IMAGE ? 2u : 1u + (uint32_t)(kPerExpert ? kConvWarps : min(ntok, kConvWarps)));
            mbar_init(&sm.empty[i], 1);
            if (i == 0) {
                mbar_init(&sm.acc_full, 1);
                mbar_init(&sm.drain, 1);
                sm.abort = 0;
            }
            fence_barrier_init();
        }
        if (threadIdx.x < kMaxTokens) sm.amax[threadIdx.x] = 0;
        if (warp == 1) {
            tmem_alloc(&sm.tmem_base, p.tmem_cols);
            tmem_relinquish();
        }
    };
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm0);
        if (M == Mode::GateUp) tma_prefetch_desc(&tm1);
    }
    set_up(p.T);
    // What is above may overlap the previous kernel's tail. The conversion
    // kernel that an Image kernel follows let it start only once every kernel
    // before the two had completed, with its results in global memory, so weights
    // (which TMA fetches from L2) may be read at once, and what that kernel wrote
    // is read behind a pdl_wait() of the warps that read it. Elsewhere nothing
    // below touches global memory before the previous kernel has completed.
    if constexpr (!IMAGE) pdl_wait();
    pdl_launch_dependents();

    // This block's rows, tokens and stages.
    int tile = cid, expert = 0, ntok = p.T, total = p.k_stages;
    if constexpr (kPerExpert) {
        const int a = cid / p.tiles;
        tile = cid % p.tiles;
        const int head = p.route->head[a];
        if (threadIdx.x < kMaxEntryTokens) sm.slot[threadIdx.x] = p.route->list[a][threadIdx.x];
        expert = head & 0xFFFF;
        ntok = head >> 16;
        if (ntok == 0) {  // behind the last entry: the whole cluster leaves
            tc_fence_before();
            __syncthreads();
            tc_fence_after();
            if (warp == 1) tmem_dealloc(sm.tmem_base, p.tmem_cols);
            return;
        }
    } else if constexpr (M == Mode::Down) {
        total = p.route->n_entries * p.k_stages;
    }
    const int first = (total * slice) >> p.split_log2;
    const int nst = ((total * (slice + 1)) >> p.split_log2) - first;
    constexpr int nw = M == Mode::GateUp ? 2 : 1;  // tiles: GateUp the same rows of gate and of up
    const Geometry g = p.geo[kPerExpert ? ntok - 1 : 0];
    uint8_t* const b_ring = ring + (size_t)g.w_slots * kWSlot;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;
    const uint32_t sfa_col0 = tmem + (uint32_t)nw * g.acc_cols;
    const uint32_t sfb_col0 = sfa_col0 + (uint32_t)g.w_slots * 16;

    if (warp == 0) {
        // ------------------------------------------------------------ copies
        if (lane == 0) {
            Cursor c, b;
            int issued = 0;
            bool ok = true;
            const size_t sf_matrix = (size_t)p.tiles * (size_t)p.kblocks * 512;
            int entry = 0, kb = first;
            if constexpr (M == Mode::Down) {
                entry = first / p.k_stages;
                kb = first % p.k_stages;
                if (nst > 0) expert = p.route->head[entry] & 0xFFFF;
            }
            // An Image kernel fills the ring with weights before it waits for the
            // conversion; then stage i - w + b's activations follow tile i's weights.
            Cursor img;
            int next_image = 0;
            auto load_image = [&]() {
                uint64_t* full = &sm.full[img.slot];
                mbar_arrive_expect_tx(full, g.image);
                bulk_load(b_ring + (size_t)b.slot * g.b_slot, p.image + (size_t)(first + next_image) * g.image, g.image,
                          full);
                ++next_image;
                img.advance(g.w_slots);
                b.advance(g.b_slots);
            };
            auto first_images = [&]() {
                pdl_wait();
                while (next_image < min(nst, g.b_slots)) load_image();
            };
            for (int i = 0; i < nst && ok; ++i) {
                const uint32_t sf_bytes = 512u * (uint32_t)min(4, p.kblocks - 4 * kb);
                for (int h = 0; h < nw; ++h) {
                    if (!mbar_wait(&sm.empty[c.slot], c.phase ^ 1u, &sm.abort, 0x0601)) {
                        ok = false;
                        break;
                    }
                    const bool up = h == 1;
                    uint8_t* st = ring + (size_t)c.slot * kWSlot;
                    const uint8_t* sf = (up ? p.sf1 : p.sf0) + (size_t)expert * sf_matrix +
                                        ((size_t)tile * p.kblocks + (size_t)kb * 4) * 512;
                    uint64_t* full = &sm.full[c.slot];
                    mbar_arrive_expect_tx(full, kWBytes + sf_bytes);
                    tma_load_3d(st, up ? &tm1 : &tm0, full, kb * 128, tile * kTileRows, expert);
                    bulk_load(st + kWBytes, sf, sf_bytes, full);
                    ++issued;
                    if constexpr (IMAGE) {
                        if (issued == min(nst, g.w_slots)) first_images();
                        else if (issued > g.w_slots) load_image();
                    }
                    c.advance(g.w_slots);
                }
                ++kb;
                if constexpr (M == Mode::Down) {
                    if (kb == p.k_stages) {
                        kb = 0;
                        ++entry;
                        if (i + 1 < nst) expert = p.route->head[entry] & 0xFFFF;
                    }
                }
            }
            if constexpr (IMAGE) {
                // The last stages' activations, as their slots come free: stage m's with
                // stage m - b, which is when tile m - b + w could go on.
                if (nst < g.w_slots) {
                    c.slot = 0;
                    c.phase = 1;
                }
                for (; ok && next_image < nst; c.advance(g.w_slots)) {
                    ok = mbar_wait(&sm.empty[c.slot], c.phase ^ 1u, &sm.abort, 0x0603);
                    if (ok) load_image();
                }
            }
            if (!ok || *(volatile int*)&sm.abort) {
                // Drain: every issued copy must land before the block exits.
                int dummy = 0;
                for (int j = max(0, issued - g.w_slots); j < issued; ++j)
                    mbar_wait(&sm.full[j % g.w_slots], (uint32_t)(j / g.w_slots) & 1u, &dummy, 0x0602, 100000000ull);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        // The whole warp runs the loop, so addresses and descriptors stay in
        // uniform registers, and one elected lane issues.
        if (nst > 0) {
            const uint32_t idesc = idesc_nvf4(kTileRows, g.nb);
            const uint64_t op_desc = desc_kmajor_sw128(0), sf_desc = smem_desc(0, 0, 128, 0);
            // A: K-block j at sfa_col + 4 j. B: K-block j at sfb_col + 4 j, or, with
            // two row halves, half q at sfb_col + 8 j + 4 q.
            const uint32_t sfb_step = g.sfb_step >> 4, sfb_next = g.sfb_cols / 4;
            Cursor w, b;
            bool ok = true;
            int kb = M == Mode::Down ? first % p.k_stages : first;
            for (int i = 0; i < nst && ok; ++i) {
                const int nblk = min(4, p.kblocks - 4 * kb);
                const uint32_t b_addr = smem_u32(b_ring) + (uint32_t)b.slot * g.b_slot;
                const uint64_t b_desc = op_desc + (b_addr >> 4);
                const uint64_t sfb_desc = sf_desc + ((b_addr + (uint32_t)g.nb * 128) >> 4);
                const uint32_t sfb_col = sfb_col0 + (uint32_t)b.slot * g.sfb_cols;
                for (int h = 0; h < nw; ++h) {
                    ok = mbar_wait(&sm.full[w.slot], w.phase, &sm.abort, 0x0611);
                    if (!ok) break;
                    __syncwarp();
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(ring) + (uint32_t)w.slot * kWSlot;
                    const uint64_t a_desc = op_desc + (a_addr >> 4);
                    const uint64_t sfa_desc = sf_desc + ((a_addr + kWBytes) >> 4);
                    const uint32_t sfa_col = sfa_col0 + (uint32_t)w.slot * 16;
                    const uint32_t acc = tmem + (uint32_t)h * g.acc_cols;
                    auto scales = [&](int j) { tmem_cp_32x128b_warpx4(sfa_col + 4 * j, sfa_desc + 32 * j); };
                    auto product = [&](int j) {
                        mma_nvf4(acc, a_desc + 2 * j, b_desc + 2 * j, idesc, sfa_col + 4 * j, sfb_col + sfb_next * j,
                                 (i | j) != 0);
                    };
                    if (elect_one()) {
                        if (h == 0) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                tmem_cp_32x128b_warpx4(sfb_col + sfb_next * j, sfb_desc + sfb_step * j);
                                if (sfb_next == 8u) tmem_cp_32x128b_warpx4(sfb_col + 4 + 8 * j, sfb_desc + 128 + 32 * j);
                            }
                        }
                        if (nblk == 4) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) scales(j);
#pragma unroll
                            for (int j = 0; j < 4; ++j) product(j);
                        } else {
                            for (int j = 0; j < nblk; ++j) scales(j);
                            for (int j = 0; j < nblk; ++j) product(j);
                        }
                        tc_commit(&sm.empty[w.slot]);
                    }
                    __syncwarp();
                    w.advance(g.w_slots);
                }
                b.advance(g.b_slots);
                if (++kb == p.k_stages && M == Mode::Down) kb = 0;
            }
            if (elect_one()) {
                tc_commit(&sm.acc_full);
                // Every MMA issued completes before TMEM is freed.
                tc_commit(&sm.drain);
            }
            __syncwarp();
            int dummy = 0;
            mbar_wait(&sm.drain, 0, &dummy, 0x0613, 100000000ull);
        }
        __syncwarp();
    } else {
        const int w = (int)warp - 2;
        if constexpr (IMAGE) {
            pdl_wait();
            if (w == 0) sm.amax[lane] = (int)lane < p.T ? p.amax[lane] : 0u;
            named_sync(1, 128);
        } else {
        // ------------------------------------------------------------ activations
        // Unit u = i * tokens + t, token t in stage i, is warp u % 8's. A lane
        // holds eight elements of it; false: the token has none in the stage.
        struct Unit {
            int i, t;
            int entry, kb;  // of the stage; Down only
        };
        auto row_of = [&](const Unit& n) -> int {
            if constexpr (M == Mode::Down) return p.route->slot[n.entry][n.t];
            if constexpr (M == Mode::GateUp) return sm.slot[n.t] / p.top;
            return n.t;
        };
        auto load = [&](const Unit& n, uint4 (&r)[2]) -> bool {
            const int row = row_of(n), kb = M == Mode::Down ? n.kb : first + n.i;
            const int k = kb * kStageK + (int)lane * 8;
            r[0] = r[1] = make_uint4(0, 0, 0, 0);
            if (row < 0) return false;
            if (k < p.K) load_raw(static_cast<const XT*>(p.X) + (size_t)row * p.ldx + k, p.x_vec != 0, r);
            return true;
        };
        // x / ntok for x <= 8, exactly.
        const uint32_t inverse = p.inverse[ntok];
        const int step_i = (int)(kConvWarps * inverse >> 16), step_t = kConvWarps - step_i * ntok;
        auto next_unit = [&](Unit& u) {
            const int was = u.i;
            u.i += step_i;
            u.t += step_t;
            if (u.t >= ntok) {
                u.t -= ntok;
                ++u.i;
            }
            if constexpr (M == Mode::Down) {
                u.kb += u.i - was;
                while (u.kb >= p.k_stages) {
                    u.kb -= p.k_stages;
                    ++u.entry;
                }
            }
        };
        Unit first_unit;
        first_unit.i = (int)((uint32_t)w * inverse >> 16);
        first_unit.t = w - first_unit.i * ntok;
        first_unit.entry = M == Mode::Down ? (first + first_unit.i) / p.k_stages : 0;
        first_unit.kb = M == Mode::Down ? (first + first_unit.i) % p.k_stages : 0;
        const int units = nst * ntok;
        auto in_k = [&](const Unit& u) {
            return (M == Mode::Down ? u.kb : first + u.i) * kStageK + (int)lane * 8 < p.K;
        };
        auto keep_max = [&](const uint4 (&r)[2], int t, bool valid) {
            float v[8];
            widen<XT>(r, v);
            const uint32_t m = __reduce_max_sync(0xffffffffu, max_bits(v));
            if (lane == 0 && valid) atomicMax(&sm.amax[t], m);
        };
        // A slice of at most four units per warp that the ring holds whole
        // stays in registers between the search for the largest magnitude
        // and the conversion.
        bool done = false;
        if constexpr (M == Mode::Gemv) {
            constexpr int kHeld = 4;
            if (nst <= g.w_slots && units <= kHeld * kConvWarps) {
                uint4 r[kHeld][2];
                Unit u = first_unit;
#pragma unroll
                for (int c = 0; c < kHeld; ++c, next_unit(u))
                    if (u.i < nst) load(u, r[c]);
                u = first_unit;
#pragma unroll
                for (int c = 0; c < kHeld; ++c, next_unit(u))
                    if (u.i < nst) keep_max(r[c], u.t, true);
                named_sync(1, 32 * kConvWarps);
                u = first_unit;
#pragma unroll
                for (int c = 0; c < kHeld; ++c, next_unit(u)) {
                    if (u.i >= nst) continue;
                    float v[8];
                    widen<XT>(r[c], v);
                    uint8_t* b_rows = b_ring + (size_t)u.i * g.b_slot;
                    convert<kPlanes>(v, anchor_of<kPlanes>(sm.amax[u.t]), u.t, in_k(u), b_rows,
                                     b_rows + (size_t)g.nb * 128, g.sfb_step, lane);
                }
                fence_proxy_async_smem();
                __syncwarp();
                // One arrival for each stage in which the warp had a token.
                if (lane == 0)
                    for (int i = 0; i < nst; ++i)
                        if (((w - i * ntok) & (kConvWarps - 1)) < ntok) mbar_arrive(&sm.full[i]);
                done = true;
            }
        }
        if (!done) {
            // Two units' elements are on their way while one is converted.
            Unit cur = first_unit, ahead = first_unit;
            uint4 r0[2], r1[2];
            bool on0 = false, on1 = false;
            if (cur.i < nst) on0 = load(cur, r0);
            next_unit(ahead);
            if (ahead.i < nst) on1 = load(ahead, r1);
            if (p.amax) {
                if (w == 0 && (int)lane < ntok)
                    sm.amax[lane] = p.amax[kPerExpert ? sm.slot[lane] / p.top : (int)lane];
            } else {
                Unit u = first_unit;
                for (int u0 = w; u0 < units; u0 += 4 * kConvWarps) {
                    uint4 r[4][2];
                    int t[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c, next_unit(u)) {
                        t[c] = u.t;
                        r[c][0] = r[c][1] = make_uint4(0, 0, 0, 0);
                        if (u.i < nst) load(u, r[c]);
                    }
#pragma unroll
                    for (int c = 0; c < 4; ++c) keep_max(r[c], t[c], u0 + c * kConvWarps < units);
                }
            }
            if constexpr (M == Mode::Down) {
                for (int i = w * 32 + (int)lane; i < kMaxSlots * kMaxTokens; i += 32 * kConvWarps)
                    (&sm.dirty[0][0])[i] = 1;
            }
            named_sync(1, 32 * kConvWarps);
            Cursor c, b;
            for (int i = 0; i < nst; ++i) {
                // Every warp waits for every slot, whether or not it has a token
                // in it: a barrier's parity tells one phase from the next only.
                const int slot0 = c.slot;
                bool ok = mbar_wait(&sm.empty[c.slot], c.phase ^ 1u, &sm.abort, 0x0621);
                c.advance(g.w_slots);
                const int slot1 = c.slot;
                if (nw == 2) {
                    ok = ok && mbar_wait(&sm.empty[c.slot], c.phase ^ 1u, &sm.abort, 0x0622);
                    c.advance(g.w_slots);
                }
                if (!ok) break;
                __syncwarp();
                if (cur.i == i) {
                    uint8_t* b_rows = b_ring + (size_t)b.slot * g.b_slot;
                    uint8_t* sfb = b_rows + (size_t)g.nb * 128;
                    const bool inside = in_k(cur);
                    do {
                        const int t = cur.t;
                        float v[8];
                        widen<XT>(r0, v);
                        const bool on = on0;
                        r0[0] = r1[0];
                        r0[1] = r1[1];
                        on0 = on1;
                        next_unit(cur);
                        next_unit(ahead);
                        if (ahead.i < nst) on1 = load(ahead, r1);
                        if (M != Mode::Down || on) {
                            convert<kPlanes>(v, anchor_of<kPlanes>(sm.amax[t]), t, inside, b_rows, sfb, g.sfb_step,
                                             lane);
                            if (M == Mode::Down && lane == 0) sm.dirty[b.slot][t] = 1;
                        } else if (sm.dirty[b.slot][t]) {
                            convert_zero<kPlanes>(t, b_rows, sfb, g.sfb_step, lane);
                            __syncwarp();
                            if (lane == 0) sm.dirty[b.slot][t] = 0;
                        }
                    } while (cur.i == i);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (!kPerExpert && lane == 0) mbar_arrive(&sm.full[slot0]);
                }
                if (kPerExpert && lane == 0) {
                    mbar_arrive(&sm.full[slot0]);
                    mbar_arrive(&sm.full[slot1]);
                }
                b.advance(g.b_slots);
            }
        }
        }
        __syncwarp();
        // ------------------------------------------------------------ partial sums
        // Warps 2..5: a thread reads its row's columns, adds the planes and
        // leaves the slice's sums in shared memory (over the rings, whose last
        // use the accumulator barrier has seen complete).
        if (w < 4) {
            float* part = reinterpret_cast<float*>(ring);
            const bool direct = M != Mode::GateUp && split == 1;
            const uint32_t quarter = warp & 3u;
            const int row = (int)(quarter * 32 + lane);
            if (nst > 0) {
                mbar_wait(&sm.acc_full, 0, &sm.abort, 0x0631);
                __syncwarp();
                tc_fence_after();
            }
            for (int h = 0; h < nw; ++h, part += ntok * kTileRows) {
                const float alpha = M == Mode::Gemv ? p.alpha0[0]
                                    : M == Mode::GateUp ? (h ? p.alpha1 : p.alpha0)[expert]
                                                        : 1.0f;
                const uint32_t acc = tmem + ((quarter * 32u) << 16) + (uint32_t)h * g.acc_cols;
                constexpr int kAtOnce = 4;  // tokens
                for (int t0 = 0; t0 < ntok; t0 += kAtOnce) {
                    if (nst == 0) {
                        for (int t = t0; t < min(t0 + kAtOnce, ntok); ++t) part[t * kTileRows + row] = 0.0f;
                        continue;
                    }
                    constexpr int kLoads = (kPlanes * kAtOnce + 7) / 8;
                    uint32_t c[kLoads][8];
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) tmem_ld_32x32b_x8(acc + (uint32_t)(kPlanes * t0 + 8 * i), c[i]);
                    // With one slice the sums are final: no other block has a part.
                    const int n = tile * kTileRows + row;
                    float r[kAtOnce];
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        r[i] = 0.0f;
                        if constexpr (M == Mode::Gemv)
                            if (direct && p.R && t0 + i < ntok && n < p.N)
                                r[i] = static_cast<float>(static_cast<const YT*>(p.R)[(size_t)(t0 + i) * p.ldr + n]);
                    }
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        if (t0 + i >= ntok) continue;
                        auto col = [&](int n) { return __uint_as_float(c[n >> 3][n & 7]); };
                        float s = col(kPlanes * i + kPlanes - 1);
#pragma unroll
                        for (int q = kPlanes - 2; q >= 0; --q) s = __fmaf_rn(s, 0.125f, col(kPlanes * i + q));
                        const uint32_t mb = sm.amax[t0 + i];
                        s = s * alpha * __uint_as_float((uint32_t)(anchor_of<kPlanes>(mb) - 8 + 127) << 23);
                        if (mb >= kInfBits) s = __uint_as_float(0x7FC00000u);
                        if (!direct) part[(t0 + i) * kTileRows + row] = s;
                        else if (n < p.N) static_cast<YT*>(p.Y)[(size_t)(t0 + i) * p.ldy + n] = from_f32<YT>(s + r[i]);
                    }
                }
            }
            tc_fence_before();
        }
    }
    __syncwarp();
    cluster_sync();

    // ---------------------------------------------------------------- slices
    // The cluster's blocks share the rows out; slices add in rank order.
    {
        // A thread has four rows of a token at a time.
        const int rows = kTileRows >> p.split_log2;  // 16 to 128
        const uint32_t base = smem_u32(ring);
        const int fours = M != Mode::GateUp && split == 1 ? 0 : (ntok * rows) >> 2;
        if constexpr (M == Mode::GateUp) {
            // sm.amax now gathers h's largest magnitudes.
            __syncthreads();
            if (threadIdx.x < kMaxTokens) sm.amax[threadIdx.x] = 0;
            __syncthreads();
        }
        for (int i = (int)threadIdx.x; i < fours; i += kThreads<IMAGE>) {
            const int j = i << 2, t = j >> (7 - p.split_log2), r = slice * rows + (j & (rows - 1));
            const int n = tile * kTileRows + r;
            if (n >= p.N) continue;
            const uint32_t off = base + (uint32_t)(t * kTileRows + r) * 4u;
            if constexpr (M == Mode::GateUp) {
                const float4 s4 = sum_cluster(off, split);
                const float4 u4 = sum_cluster(off + (uint32_t)(ntok * kTileRows) * 4u, split);
                const int slot = sm.slot[t];
                const float c = p.weights[slot] * p.alpha2[expert];
                const float s[4] = {s4.x, s4.y, s4.z, s4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w};
                float hv[4];
                uint32_t m = 0;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    hv[q] = s[q] / (1.0f + expf(-s[q])) * u[q] * c;
                    m = max(m, __float_as_uint(hv[q]) & 0x7FFFFFFFu);
                }
                // F is a multiple of 64, so the four are all inside.
                *reinterpret_cast<float4*>(static_cast<float*>(p.Y) + (size_t)slot * p.ldy + n) =
                    make_float4(hv[0], hv[1], hv[2], hv[3]);
                if (m) atomicMax(&sm.amax[t], m);
            } else {
                const float4 s4 = sum_cluster(off, split);
                const float s[4] = {s4.x, s4.y, s4.z, s4.w};
                YT* y = static_cast<YT*>(p.Y) + (size_t)t * p.ldy + n;
                float res[4] = {};
                if constexpr (M == Mode::Gemv) {
                    if (p.R) {
                        const YT* rr = static_cast<const YT*>(p.R) + (size_t)t * p.ldr + n;
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            if (n + q < p.N) res[q] = static_cast<float>(rr[q]);
                    }
                }
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (n + q < p.N) y[q] = from_f32<YT>(s[q] + res[q]);
            }
        }
        if constexpr (M == Mode::GateUp) {
            __syncthreads();
            // Maxima: the order of the atomics does not matter.
            if ((int)threadIdx.x < ntok && sm.amax[threadIdx.x])
                atomicMax(&p.amax_out[sm.slot[threadIdx.x] / p.top], sm.amax[threadIdx.x]);
        }
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();  // no block leaves while another may read its sums
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, p.tmem_cols);
    }
}

// ---------------------------------------------------------------- host side

static inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// The shape of a stream_kernel's blocks, see block_shape().
static Shape set_shape(Params& p, int planes, int tokens, bool each, int tiles, Fill fill, int stages) {
    for (int t = 1; t <= kMaxTokens; ++t) p.inverse[t] = 65536u / (uint32_t)t + 1;
    const Shape s = block_shape(p.geo, planes, tokens, each, tiles, fill, stages, sizeof(Control));
    p.ring_bytes = s.ring_bytes;
    p.tmem_cols = s.tmem_cols;
    return s;
}

// Slices of K, as a power of two up to 8 (the cluster's size), for `units` blocks of
// `stages` stages without a split: the fewest stage times, of
//   as long as all blocks are resident, the stages of the SM with most blocks, a
//   tenth more where one block has an SM alone that could hold two (less on its
//   way), two stages' time for start and end, half a one for each doubling of the
//   cluster;
//   else waves of blocks, each with that start and end.
// Measured at one token, us, for 1 / 2 / 4 / 8 slices: 2048 x 2048 6.2 / 4.8 / 4.3 /
// 4.4, 4096 x 4096 8.9 / 6.5 / 5.1 / 5.5, 8192 x 2048 6.3 / 5.0 / 5.1 / 10.0, 8192 x
// 8192 14.5 / 10.3 / 8.9 / 13.3, 28672 x 8192 24.0 / 27.1 / 33.1 / 43.0.
static int choose_split_log2(double units, double stages, int sms, int per_sm) {
    int best = 0;
    double best_cost = 0;
    for (int l = 0, s = 1; l <= 3; ++l, s *= 2) {
        if (l > 0 && stages < s) break;
        const double blocks = units * s, each = ceil(stages / s), resident = (double)sms * per_sm;
        double cost = 0.5 * l;
        if (blocks <= resident) {
            const double on = ceil(blocks / sms);
            cost += on * each * (on < per_sm ? 1.1 : 1.0) + 2.0;
        } else {
            cost += ceil(blocks / resident) * per_sm * (each + 2.0);
        }
        if (l == 0 || cost < best_cost) {
            best = l;
            best_cost = cost;
        }
    }
    return best;
}

// Launches a kernel of this family in clusters of `csize` blocks.
static int launch_clusters(void (*kernel)(CUtensorMap, CUtensorMap, Params), uint64_t* configured, int blocks,
                           int threads, int csize, size_t smem, cudaStream_t stream, const CUtensorMap& tm0,
                           const CUtensorMap& tm1, const Params& p) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return GPLK_STATUS_CUDA_ERROR;
    if (!(*configured & (1ull << dev))) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess)
            return GPLK_STATUS_LAUNCH_FAIL;
        *configured |= 1ull << dev;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)csize;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return launch_status(cudaLaunchKernelEx(&cfg, kernel, tm0, tm1, p));
}

template <Mode M, typename XT, typename YT, bool IMAGE = false>
static int launch_stream(const CUtensorMap& tm0, const CUtensorMap& tm1, const Params& p, size_t smem, int clusters,
                         cudaStream_t stream) {
    static thread_local uint64_t configured = 0;  // bit per device
    return launch_clusters(stream_kernel<M, XT, YT, IMAGE>, &configured, clusters << p.split_log2, kThreads<IMAGE>,
                           1 << p.split_log2, smem, stream, tm0, tm1, p);
}

// Tensor map of `matrices` weight matrices of `rows` rows of K / 2 bytes.
static int encode_weights(CUtensorMap* map, const uint8_t* W, int rows, int matrices, int K) {
    const WeightMap m = weight_map((uint64_t)rows, (uint64_t)matrices, (uint64_t)K);
    return encode_tmap_3d_u8(map, W, m.sizes, m.pitches, m.box);
}

}  // namespace fewtok
}  // namespace gplk
