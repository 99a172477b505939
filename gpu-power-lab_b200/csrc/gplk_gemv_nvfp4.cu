// gplk_gemv_nvfp4.cu - products of a few tokens with NVFP4 weights:
//   y[t][n] = alpha * sum_k x[t][k] * sf[n][k / 16] * w[n][k]  (+ r[t][n])
// with E2M1 weights and UE4M3 scales in the layout gplk_gemm_nvfp4_tn reads,
// 16-bit activations and FP32 sums, rounded once to the activations' type.
// The main loop here (stream_kernel) also runs the experts' products of
// gplk_moe_nvfp4.cu.
//
// What bounds it: every weight is read once for 2 T operations, so HBM. A
// B200 reads 46 weights per SM and clock; decoding them on the CUDA cores
// takes about that many issue slots (one warp per row with FP32 FMAs measured
// 0.56 TB/s at one token, 16384 x 8192). So the weights are not decoded at all:
// they go from HBM through TMA to the block-scaled tensor-core MMA
// (kind::mxf4nvf4), codes and scales as they lie, and the activations are
// brought to its operand format instead, exactly enough to count as 16-bit:
//
//   Within a 16-group of a token, 2^b the power of two at or below its largest
//   magnitude, x is rounded to a multiple of 2^b / 8192 and written in
//   balanced base-8 digits  x = 2^b * sum_p d_p / 2 * 8^-p,  p = 0..4,
//   d_0 in -4..4, the others in -4..3. Every d / 2 is an E2M1 value, so digit p
//   of all of k is one E2M1 row ("plane") of the MMA's B operand, and 2^b,
//   relative to the token's largest magnitude 2^A, is the group's UE4M3 scale.
//   Five planes keep 15 bits: an activation is off by at most 2^-14 of its
//   group's largest magnitude (2^-28 of the token's, in groups 2^14 below
//   it), where BF16 itself is off by 2^-9 of each value. The accumulator
//   column of each (token, plane) is exact products in FP32 sums; the epilogue
//   adds 8^-p times the planes' columns.
//
// So T tokens are an MMA of N = 5 T columns (padded to 8), at most 160 of the
// 256 an instruction takes, whose time at T = 32 is still below the time HBM
// needs for the weights.
//
// Layout of the work. A block owns 128 weight rows (the MMA's M) and a slice
// of K; blocks of a cluster share the rows, split K, and add their partial
// sums in rank order through distributed shared memory, so the bits do not
// depend on timing. Two blocks share an SM: one's start and end hide behind
// the other's stream.
//   warp 0      TMA producer: 128 rows x 128 bytes of codes and up to 2 KiB of
//               scales per stage (256 elements of K) into a ring
//   warp 1      owns TMEM; one thread copies the scales to TMEM and issues
//               one MMA per 64 elements of K
//   warps 2..9  convert the same 256 elements of every token into the stage's
//               B rows and scales (a warp per token and stage); warps 2..5
//               then read the accumulator, and all warps add the slices
// Every mbarrier wait is bounded, as everywhere in this library.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cstring>
#include <type_traits>

#include "gplk_ptx.cuh"

namespace gplk {
namespace fewtok {

constexpr int kMaxTokens = 32;
constexpr int kMaxExperts = 512;
constexpr int kMaxTop = 16;
constexpr int kPlanes = 5;
constexpr int kConvWarps = 8;
constexpr int kTileRows = 128;
constexpr int kStageK = 256;                    // elements of K per stage
constexpr uint32_t kWBytes = kTileRows * 128;   // codes of a stage
constexpr uint32_t kSfaBytes = 4 * 512;         // scales of a stage
constexpr int kMaxStages = 8;
constexpr uint32_t kDigitBias = 4u * (1u + 8u + 64u + 512u + 4096u);

// Gemv: all tokens against one matrix. GateUp: a chosen expert's tokens against
// its gate and up matrices. Down: all tokens against every chosen expert's down
// matrix, accumulated over the experts. DownPart: a chosen expert's tokens
// against its down matrix.
enum class Mode { Gemv, GateUp, Down, DownPart };

template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    return static_cast<T>(v);
}

// ---------------------------------------------------------------- routing tables (MoE)
// Written by the route kernel into the layer's workspace.
struct Route {
    int n_active;
    int head[kMaxExperts];                      // active expert a: its index | its tokens << 16, ascending; then 0
    int16_t list[kMaxExperts][kMaxTokens];      // their slots (token * top + rank), ascending
    int16_t slot[kMaxExperts][kMaxTokens];      // slot of token t with active expert a, or -1
};

struct Params {
    const void* X;       // activations (Gemv, GateUp: 16-bit rows; Down: FP32 h rows by slot)
    const uint8_t* sf0;  // scales: W, gate or down
    const uint8_t* sf1;  // GateUp: up
    const float* alpha0; // Gemv: one; GateUp: gate's, per expert
    const float* alpha1; // GateUp: up's
    const float* alpha2; // GateUp: down's, folded into h
    void* Y;             // Gemv, Down: T rows; GateUp: FP32 h rows by slot
    const void* R;
    const Route* route;
    const float* weights;  // MoE: per slot
    const uint8_t* image;  // Image kernels: the converted activations, by stage
    const uint32_t* amax;  // bits of each token's largest magnitude, or NULL: this kernel finds its slice's
    uint32_t* amax_out;    // GateUp: h's, by token
    int T, N, K, ldx, ldy, ldr;
    int x_vec;           // rows of X are 16-byte aligned
    int top;
    int tiles;           // 128-row tiles of one matrix
    int k_stages;        // stages of one matrix row
    int kblocks;         // K / 64
    int split;           // slices of K
    uint32_t ring_bytes; // shared memory of the ring
    uint32_t tmem_cols;
};

// Ring and TMEM layout for a block's tokens. A stage holds codes | their
// scales | B rows | B scales; TMEM the accumulator, then a slot of scale
// columns per stage.
struct Geometry {
    int nb;      // accumulator columns
    int stages;  // ring depth
    uint32_t stage_bytes, sfb_bytes;
    uint32_t sf_col0, sf_slot;
};

__host__ __device__ __forceinline__ Geometry geometry(int ntok, uint32_t ring_bytes, uint32_t tmem_cols) {
    Geometry g;
    g.nb = (kPlanes * ntok + 7) & ~7;
    const bool wide = g.nb > 128;  // a second 128 rows of B scales
    g.sfb_bytes = wide ? 4096 : 2048;
    g.stage_bytes = kWBytes + kSfaBytes + (uint32_t)g.nb * 128 + g.sfb_bytes;
    g.sf_col0 = ((uint32_t)g.nb + 15) & ~15u;
    g.sf_slot = wide ? 48 : 32;
    const uint32_t fit = ring_bytes / g.stage_bytes, slots = (tmem_cols - g.sf_col0) / g.sf_slot;
    g.stages = (int)(fit < slots ? fit : slots);
    if (g.stages > kMaxStages) g.stages = kMaxStages;
    return g;
}

struct Control {
    uint64_t full[kMaxStages];
    uint64_t empty[kMaxStages];
    uint64_t acc_full;
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
    uint32_t amax[kMaxTokens];  // bits of the largest magnitude in this block's slice
    int16_t slot[kMaxTokens];   // GateUp: slots of the block's tokens
    uint8_t dirty[kMaxStages][kMaxTokens];  // Down: the ring slot holds digits of that token
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

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
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

// Exponent A of a token's largest magnitude. Below 2^-100 the anchor stays
// there: what is then lost is below 2^-127, FP32's own subnormal range.
__device__ __forceinline__ int anchor_of(uint32_t amax_bits) { return max((int)(amax_bits >> 23) - 127, -100); }

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

// One token's 256 elements of a stage, eight per lane: planes 5 t .. 5 t + 4
// of the stage's B rows (128-byte swizzled, K-major) and the 16 groups'
// scales. `on` is false for lanes beyond K, whose blocks no MMA reads.
__device__ __forceinline__ void convert(const float (&v)[8], int anchor, int t, bool on, uint8_t* b_rows,
                                        uint8_t* sfb, uint32_t lane) {
    uint32_t m = max_bits(v);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));  // the other half of the 16-group
    const int b = max((int)(m >> 23) - 127, anchor - 14);
    const float scale = __uint_as_float((uint32_t)(13 - b + 127) << 23);
    // x * scale is at most 2^14 in magnitude; adding 1.5 * 2^23 rounds it to an
    // integer, and the bias makes every digit non-negative.
    constexpr float kMagic = 12582912.0f + (float)kDigitBias;
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(__fmaf_rn(v[i], scale, kMagic));
    uint32_t q[4];  // elements i and i + 4: nibbles i and i + 4 of a word are 16 bits apart
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = __byte_perm(u[i], u[i + 4], 0x5410);
    if (!on) return;
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) {
        const int sh = 3 * (kPlanes - 1 - p);
        const uint32_t mask = p == 0 ? 0x000F000Fu : 0x00070007u;
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= ((q[i] >> sh) & mask) << (4 * i);
        w = p == 0 ? digit_codes<true>(w) : digit_codes<false>(w);
        const uint32_t r = (uint32_t)(kPlanes * t + p);
        *reinterpret_cast<uint32_t*>(b_rows + (r >> 3) * 1024 + (r & 7) * 128 + (((lane >> 2) ^ (r & 7)) << 4) +
                                     (lane & 3) * 4) = w;
        if ((lane & 1) == (uint32_t)(p & 1))
            sfb[(r >> 7) * 2048 + (lane >> 3) * 512 + (r & 31) * 16 + ((r & 127) >> 5) * 4 + ((lane >> 1) & 3)] =
                (uint8_t)((b - anchor + 15) << 3);
    }
}

// A token without a part in the stage's expert: zero digits, scale 1.
__device__ __forceinline__ void convert_zero(int t, uint8_t* b_rows, uint8_t* sfb, uint32_t lane) {
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) {
        const uint32_t r = (uint32_t)(kPlanes * t + p);
        *reinterpret_cast<uint32_t*>(b_rows + (r >> 3) * 1024 + (r & 7) * 128 + lane * 4) = 0u;
        if ((lane & 1) == (uint32_t)(p & 1))
            sfb[(r >> 7) * 2048 + (lane >> 3) * 512 + (r & 31) * 16 + ((r & 127) >> 5) * 4 + ((lane >> 1) & 3)] = 0x38;
    }
}

template <bool IMAGE>
constexpr int kThreads = IMAGE ? 64 + 128 : 64 + 32 * kConvWarps;

template <Mode M, typename XT, typename YT, bool IMAGE>
__global__ void __launch_bounds__(kThreads<IMAGE>, 2)
    stream_kernel(const __grid_constant__ CUtensorMap tm0, const __grid_constant__ CUtensorMap tm1, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    Control& sm = *reinterpret_cast<Control*>(ring + p.ring_bytes);
    const uint32_t warp = warp_id_uniform();
    const uint32_t lane = lane_id();
    const int rank = (int)cluster_ctarank();
    const int csize = (M == Mode::GateUp ? 2 : 1) * p.split;
    const int cid = (int)blockIdx.x / csize;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kMaxStages; ++i) {
            mbar_init(&sm.full[i], IMAGE ? 1 : 1 + kConvWarps);
            mbar_init(&sm.empty[i], 1);
        }
        mbar_init(&sm.acc_full, 1);
        mbar_init(&sm.drain, 1);
        sm.abort = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tm0);
        if (M == Mode::GateUp) tma_prefetch_desc(&tm1);
    }
    if (threadIdx.x < kMaxTokens) sm.amax[threadIdx.x] = 0;
    if (warp == 1) {
        tmem_alloc(&sm.tmem_base, p.tmem_cols);
        tmem_relinquish();
    }
    // The set-up above may overlap the previous kernel's tail. The conversion
    // kernel that an Image kernel follows let it start only once every kernel
    // before the two had completed, so weights may be read at once; what that
    // kernel wrote is read behind its own pdl_wait(). Elsewhere nothing below
    // touches global memory before the previous kernel has completed.
    if constexpr (!IMAGE) pdl_wait();
    pdl_launch_dependents();

    // This block's rows, tokens and stages.
    constexpr bool kPerExpert = M == Mode::GateUp || M == Mode::DownPart;
    int tile = cid, slice = rank, expert = 0, ntok = p.T, total = p.k_stages;
    bool second = false;  // GateUp: the `up` half of the cluster
    if constexpr (kPerExpert) {
        const int a = cid / p.tiles;
        tile = cid % p.tiles;
        second = M == Mode::GateUp && rank >= p.split;
        slice = second ? rank - p.split : rank;
        const int head = p.route->head[a];
        if (threadIdx.x < kMaxTokens) sm.slot[threadIdx.x] = p.route->list[a][threadIdx.x];
        expert = head & 0xFFFF;
        ntok = head >> 16;
        if (ntok == 0) total = 0;
    } else if constexpr (M == Mode::Down) {
        total = p.route->n_active * p.k_stages;
    }
    const int first = (int)((long long)total * slice / p.split);
    const int nst = (int)((long long)total * (slice + 1) / p.split) - first;
    const Geometry g = geometry(ntok, p.ring_bytes, p.tmem_cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0, issued_mask = 0, issued_parity = 0;
            bool ok = true;
            const CUtensorMap* tm = second ? &tm1 : &tm0;
            const size_t sf_matrix = (size_t)p.tiles * (size_t)p.kblocks * 512;
            const uint32_t image_bytes = IMAGE ? (uint32_t)g.nb * 128 + g.sfb_bytes : 0u;
            auto load_weights = [&](int i) {
                int kb = first + i;
                if constexpr (M == Mode::Down) {
                    expert = p.route->head[kb / p.k_stages] & 0xFFFF;
                    kb %= p.k_stages;
                }
                const uint32_t sf_bytes = 512u * (uint32_t)min(4, p.kblocks - 4 * kb);
                uint8_t* st = ring + (size_t)stage * g.stage_bytes;
                const uint8_t* sf = (second ? p.sf1 : p.sf0) + (size_t)expert * sf_matrix +
                                    ((size_t)tile * p.kblocks + (size_t)kb * 4) * 512;
                mbar_arrive_expect_tx(&sm.full[stage], kWBytes + sf_bytes + image_bytes);
                tma_load_2d(st, tm, &sm.full[stage], kb * 128, expert * p.N + tile * kTileRows);
                bulk_load(st + kWBytes, sf, sf_bytes, &sm.full[stage]);
                issued_mask |= 1u << stage;
                issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
            };
            auto load_image = [&](int i) {
                bulk_load(ring + (size_t)stage * g.stage_bytes + kWBytes + kSfaBytes,
                          p.image + (size_t)(first + i) * image_bytes, image_bytes, &sm.full[stage]);
            };
            auto advance = [&]() {
                if (++stage == g.stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            };
            // An Image kernel fills the ring with weights before it waits for
            // the conversion.
            int head = 0;
            if constexpr (IMAGE) {
                head = min(nst, g.stages);
                for (int i = 0; i < head; ++i, ++stage) load_weights(i);
                stage = 0;
                pdl_wait();
                for (int i = 0; i < head; ++i) {
                    load_image(i);
                    advance();
                }
            }
            for (int i = head; i < nst; ++i) {
                if (!mbar_wait(&sm.empty[stage], phase ^ 1u, &sm.abort, 0x0601)) {
                    ok = false;
                    break;
                }
                load_weights(i);
                if constexpr (IMAGE) load_image(i);
                advance();
            }
            if (!ok || *(volatile int*)&sm.abort) {
                // Drain: every issued copy must land before the block exits.
                int dummy = 0;
                for (int s2 = 0; s2 < g.stages; ++s2)
                    if (issued_mask & (1u << s2))
                        mbar_wait(&sm.full[s2], (issued_parity >> s2) & 1u, &dummy, 0x0602, 100000000ull);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        // The whole warp runs the loop, so addresses and descriptors stay in
        // uniform registers, and one elected lane issues.
        if (nst > 0) {
            const uint32_t idesc = idesc_nvf4(kTileRows, g.nb);
            const uint32_t bstep = g.sf_slot > 32 ? 8u : 4u;
            const uint64_t op_desc = desc_kmajor_sw128(0), sf_desc = smem_desc(0, 0, 128, 0);
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int i = 0; i < nst; ++i) {
                if (!mbar_wait(&sm.full[stage], phase, &sm.abort, 0x0611)) {
                    ok = false;
                    break;
                }
                __syncwarp();
                tc_fence_after();
                const int kb = M == Mode::Down ? (first + i) % p.k_stages : first + i;
                const int nblk = min(4, p.kblocks - 4 * kb);
                const uint32_t a_addr = smem_u32(ring) + (uint32_t)stage * g.stage_bytes;
                const uint64_t a_desc = op_desc + (a_addr >> 4), b_desc = a_desc + ((kWBytes + kSfaBytes) >> 4);
                const uint64_t sfa_desc = sf_desc + ((a_addr + kWBytes) >> 4);
                const uint64_t sfb_desc = sfa_desc + ((kSfaBytes + (uint32_t)g.nb * 128) >> 4);
                const uint32_t sf_col = tmem + g.sf_col0 + (uint32_t)stage * g.sf_slot;
                // A: K-block j at sf_col + 4 j. B: K-block j, 128-row half h at
                // sf_col + 16 + 8 j + 4 h (two halves), or sf_col + 16 + 4 j.
                auto scales = [&](int j) {
                    tmem_cp_32x128b_warpx4(sf_col + 4 * j, sfa_desc + 32 * j);
                    tmem_cp_32x128b_warpx4(sf_col + 16 + bstep * j, sfb_desc + 32 * j);
                    if (bstep == 8u) tmem_cp_32x128b_warpx4(sf_col + 20 + 8 * j, sfb_desc + 128 + 32 * j);
                };
                auto product = [&](int j) {
                    mma_nvf4(tmem, a_desc + 2 * j, b_desc + 2 * j, idesc, sf_col + 4 * j, sf_col + 16 + bstep * j,
                             (i | j) != 0);
                };
                if (elect_one()) {
                    if (nblk == 4) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) scales(j);
#pragma unroll
                        for (int j = 0; j < 4; ++j) product(j);
                    } else {
                        for (int j = 0; j < nblk; ++j) scales(j);
                        for (int j = 0; j < nblk; ++j) product(j);
                    }
                    tc_commit(&sm.empty[stage]);
                }
                __syncwarp();
                if (++stage == g.stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (elect_one()) {
                if (ok) tc_commit(&sm.acc_full);
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
        auto load = [&](int i, int t, uint4 (&r)[2]) -> bool {
            int kb = first + i, row = t;
            if constexpr (M == Mode::Down) {
                row = p.route->slot[kb / p.k_stages][t];
                kb %= p.k_stages;
            } else if constexpr (M == Mode::GateUp) {
                row = sm.slot[t] / p.top;
            } else if constexpr (M == Mode::DownPart) {
                row = sm.slot[t];
            }
            const int k = kb * kStageK + (int)lane * 8;
            r[0] = r[1] = make_uint4(0, 0, 0, 0);
            if (row < 0) return false;
            if (k < p.K) load_raw(static_cast<const XT*>(p.X) + (size_t)row * p.ldx + k, p.x_vec != 0, r);
            return true;
        };
        struct Unit {
            int i, t;
        };
        const int step_i = ntok > 0 ? kConvWarps / ntok : 0, step_t = ntok > 0 ? kConvWarps % ntok : 0;
        auto next_unit = [&](Unit& u) {
            u.i += step_i;
            u.t += step_t;
            if (u.t >= ntok) {
                u.t -= ntok;
                ++u.i;
            }
        };
        const Unit first_unit = {ntok > 0 ? w / ntok : 0, ntok > 0 ? w % ntok : 0};
        const int units = nst * ntok;
        auto b_rows_of = [&](int st) { return ring + (size_t)st * g.stage_bytes + kWBytes + kSfaBytes; };
        auto in_k = [&](int i) {
            const int kb = M == Mode::Down ? (first + i) % p.k_stages : first + i;
            return kb * kStageK + (int)lane * 8 < p.K;
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
            if (nst <= g.stages && units <= kHeld * kConvWarps) {
                uint4 r[kHeld][2];
                Unit u = first_unit;
#pragma unroll
                for (int c = 0; c < kHeld; ++c, next_unit(u))
                    if (u.i < nst) load(u.i, u.t, r[c]);
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
                    uint8_t* b_rows = b_rows_of(u.i);
                    convert(v, anchor_of(sm.amax[u.t]), u.t, in_k(u.i), b_rows, b_rows + (size_t)g.nb * 128, lane);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0)
                    for (int i = 0; i < nst; ++i) mbar_arrive(&sm.full[i]);
                done = true;
            }
        }
        if (!done) {
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
                        if (u.i < nst) load(u.i, u.t, r[c]);
                    }
#pragma unroll
                    for (int c = 0; c < 4; ++c) keep_max(r[c], t[c], u0 + c * kConvWarps < units);
                }
            }
            if constexpr (M == Mode::Down) {
                for (int i = w * 32 + (int)lane; i < kMaxStages * kMaxTokens; i += 32 * kConvWarps)
                    (&sm.dirty[0][0])[i] = 1;
            }
            named_sync(1, 32 * kConvWarps);
            // Two units' elements are on their way while one is converted.
            Unit cur = first_unit, ahead = first_unit;
            uint4 r0[2], r1[2];
            bool on0 = false, on1 = false;
            if (ahead.i < nst) on0 = load(ahead.i, ahead.t, r0);
            next_unit(ahead);
            if (ahead.i < nst) on1 = load(ahead.i, ahead.t, r1);
            int stage = 0;
            uint32_t phase = 0;
            for (int i = 0; i < nst; ++i) {
                if (!mbar_wait(&sm.empty[stage], phase ^ 1u, &sm.abort, 0x0621)) break;
                __syncwarp();
                uint8_t* b_rows = b_rows_of(stage);
                uint8_t* sfb = b_rows + (size_t)g.nb * 128;
                const bool inside = in_k(i);
                while (cur.i == i) {
                    const int t = cur.t;
                    float v[8];
                    widen<XT>(r0, v);
                    const bool on = on0;
                    r0[0] = r1[0];
                    r0[1] = r1[1];
                    on0 = on1;
                    next_unit(cur);
                    next_unit(ahead);
                    if (ahead.i < nst) on1 = load(ahead.i, ahead.t, r1);
                    if (M != Mode::Down || on) {
                        convert(v, anchor_of(sm.amax[t]), t, inside, b_rows, sfb, lane);
                        if (M == Mode::Down && lane == 0) sm.dirty[stage][t] = 1;
                    } else if (sm.dirty[stage][t]) {
                        convert_zero(t, b_rows, sfb, lane);
                        __syncwarp();
                        if (lane == 0) sm.dirty[stage][t] = 0;
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.full[stage]);
                if (++stage == g.stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        }
        __syncwarp();
        // ------------------------------------------------------------ partial sums
        // Warps 2..5: a thread reads its row's columns, adds the planes and
        // leaves the slice's sum in shared memory (the ring's first stage, whose
        // last use the accumulator barrier has seen complete).
        if (w < 4) {
            float* part = reinterpret_cast<float*>(ring);
            const uint32_t quarter = warp & 3u;
            const int row = (int)(quarter * 32 + lane);
            const float alpha = M == Mode::Gemv ? __ldg(p.alpha0)
                                : M == Mode::GateUp ? __ldg((second ? p.alpha1 : p.alpha0) + expert)
                                                    : 1.0f;
            if (nst > 0) {
                mbar_wait(&sm.acc_full, 0, &sm.abort, 0x0631);
                __syncwarp();
                tc_fence_after();
                for (int t0 = 0; t0 < ntok; t0 += 8) {
                    uint32_t c[5][8];
#pragma unroll
                    for (int i = 0; i < 5; ++i)
                        tmem_ld_32x32b_x8(tmem + ((quarter * 32u) << 16) + (uint32_t)(kPlanes * t0 + 8 * i), c[i]);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (t0 + i >= ntok) continue;
                        auto col = [&](int n) { return __uint_as_float(c[n >> 3][n & 7]); };
                        float s = col(5 * i + 4);
#pragma unroll
                        for (int q = 3; q >= 0; --q) s = __fmaf_rn(s, 0.125f, col(5 * i + q));
                        const uint32_t mb = sm.amax[t0 + i];
                        s = s * alpha * __uint_as_float((uint32_t)(anchor_of(mb) - 8 + 127) << 23);
                        if (mb >= kInfBits) s = __uint_as_float(0x7FC00000u);
                        part[(t0 + i) * kTileRows + row] = s;
                    }
                }
                tc_fence_before();
            } else {
                for (int t = 0; t < ntok; ++t) part[t * kTileRows + row] = 0.0f;
            }
        }
    }
    __syncwarp();
    cluster_sync();

    // ---------------------------------------------------------------- slices
    // The cluster's blocks share the rows out; slices add in rank order.
    {
        const int rows = kTileRows / csize;  // 16 to 128
        const uint32_t base = smem_u32(ring);
        if constexpr (M == Mode::GateUp) {
            // sm.amax now gathers h's largest magnitudes.
            __syncthreads();
            if (threadIdx.x < kMaxTokens) sm.amax[threadIdx.x] = 0;
            __syncthreads();
        }
        for (int i0 = (int)(warp * 32); i0 < ntok * rows; i0 += kThreads<IMAGE>) {
            const int i = i0 + (int)lane;
            const int t = i / rows, r = rank * rows + i % rows;
            const int n = tile * kTileRows + r;
            const bool valid = i < ntok * rows && n < p.N;
            float s = 0.0f, u = 0.0f;
            if (valid) {
                const uint32_t off = base + (uint32_t)(t * kTileRows + r) * 4u;
                for (int c = 0; c < p.split; ++c) s += ld_cluster_f32(mapa_shared(off, (uint32_t)c));
                if constexpr (M == Mode::GateUp)
                    for (int c = 0; c < p.split; ++c) u += ld_cluster_f32(mapa_shared(off, (uint32_t)(p.split + c)));
            }
            if constexpr (M == Mode::GateUp) {
                uint32_t m = 0;
                if (valid) {
                    const int slot = sm.slot[t];
                    const float h = s / (1.0f + expf(-s)) * u * (p.weights[slot] * __ldg(p.alpha2 + expert));
                    static_cast<float*>(p.Y)[(size_t)slot * p.ldy + n] = h;
                    m = __float_as_uint(h) & 0x7FFFFFFFu;
                }
                // 16 neighbouring lanes have one token.
#pragma unroll
                for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                if ((lane & 15) == 0 && m) atomicMax(&sm.amax[t], m);
            } else if (valid) {
                if constexpr (M == Mode::Gemv)
                    if (p.R) s += static_cast<float>(static_cast<const YT*>(p.R)[(size_t)t * p.ldr + n]);
                const size_t row = M == Mode::DownPart ? sm.slot[t] : t;
                static_cast<YT*>(p.Y)[row * p.ldy + n] = from_f32<YT>(s);
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

// ---------------------------------------------------------------- conversion ahead of the products
// Writes the B rows and scales of every stage as the ring holds them, a block
// per token, so that the blocks of an Image kernel fetch them with one bulk
// copy per stage instead of each converting all of the tokens again.
constexpr int kImageThreads = 512;

template <typename XT>
__global__ void __launch_bounds__(kImageThreads)
    image_kernel(const XT* X, uint8_t* image, uint32_t* amax, int K, int ldx, int x_vec, int nb, uint32_t sfb_bytes) {
    __shared__ uint32_t top[kImageThreads / 32];
    constexpr int kWarps = kImageThreads / 32, kHeld = 4;
    const int t = blockIdx.x, warp = (int)warp_id_uniform();
    const uint32_t lane = lane_id();
    const int stages = (K + kStageK - 1) / kStageK;
    // Only now may the products start, whose weight loads wait for no one:
    // every earlier kernel has completed.
    pdl_wait();
    pdl_launch_dependents();
    const XT* x = X + (size_t)t * ldx;
    auto load = [&](int i, uint4 (&r)[2]) {
        const int k = i * kStageK + (int)lane * 8;
        r[0] = r[1] = make_uint4(0, 0, 0, 0);
        if (k < K) load_raw(x + k, x_vec != 0, r);
    };
    uint4 held[kHeld][2];  // the first stages stay in registers
    uint32_t m = 0;
    for (int i0 = warp; i0 < stages; i0 += kHeld * kWarps) {
        uint4 r[kHeld][2];
#pragma unroll
        for (int c = 0; c < kHeld; ++c) {
            r[c][0] = r[c][1] = make_uint4(0, 0, 0, 0);
            if (i0 + c * kWarps < stages) load(i0 + c * kWarps, r[c]);
        }
#pragma unroll
        for (int c = 0; c < kHeld; ++c) {
            float v[8];
            widen<XT>(r[c], v);
            m = max(m, max_bits(v));
            if (i0 == warp) {
                held[c][0] = r[c][0];
                held[c][1] = r[c][1];
            }
        }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) top[warp] = m;
    __syncthreads();
    m = __reduce_max_sync(0xffffffffu, lane < kWarps ? top[lane] : 0u);
    if (threadIdx.x == 0) amax[t] = m;
    const int anchor = anchor_of(m);
    const size_t bytes = (size_t)nb * 128 + sfb_bytes;
    auto emit = [&](int i, const uint4 (&r)[2]) {
        float v[8];
        widen<XT>(r, v);
        uint8_t* b_rows = image + (size_t)i * bytes;
        convert(v, anchor, t, i * kStageK + (int)lane * 8 < K, b_rows, b_rows + (size_t)nb * 128, lane);
    };
#pragma unroll
    for (int c = 0; c < kHeld; ++c)
        if (warp + c * kWarps < stages) emit(warp + c * kWarps, held[c]);
    for (int i = warp + kHeld * kWarps; i < stages; i += kWarps) {
        uint4 r[2];
        load(i, r);
        emit(i, r);
    }
}

// ---------------------------------------------------------------- host side

static inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Shared memory and TMEM of a block. Two blocks share an SM, each with half of
// its shared memory and 256 TMEM columns, unless one token count asks for more
// than 128 accumulator columns in every block.
struct Shape {
    int per_sm;
    size_t smem;
};

static Shape set_shape(Params& p, bool wide) {
    const size_t overhead = 1024 + ((sizeof(Control) + 127) & ~(size_t)127);
    // 228 KiB per SM, 1 KiB of it reserved per block.
    const size_t room = (wide ? 227 * 1024 : (228 * 1024 - 2 * 1024) / 2) - overhead;
    p.ring_bytes = (uint32_t)(room & ~(size_t)1023);
    p.tmem_cols = wide ? 512 : 256;
    return {wide ? 1 : 2, p.ring_bytes + overhead};
}

static bool is_wide(int T) { return kPlanes * T > 128; }

// Slices of K: the split whose waves of blocks, each as long as its stages and
// about two more for its start and end, take the fewest stage times. `units`
// blocks would run without a split, each of `stages` stages.
static int choose_split(double units, double stages, int max_split, int slots) {
    int best = 1;
    double best_cost = 0;
    for (int s = 1; s <= max_split; s *= 2) {
        if (s > 1 && stages < s) break;
        const double waves = (double)(long long)((units * s + slots - 1) / slots);
        const double cost = waves * ((stages + s - 1) / s + 2.0);
        if (s == 1 || cost < best_cost) {
            best = s;
            best_cost = cost;
        }
    }
    return best;
}

template <Mode M, typename XT, typename YT, bool IMAGE = false>
static int launch_stream(const CUtensorMap& tm0, const CUtensorMap& tm1, const Params& p, size_t smem, int clusters,
                         cudaStream_t stream) {
    auto kernel = stream_kernel<M, XT, YT, IMAGE>;
    static thread_local uint64_t configured = 0;  // bit per device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return GPLK_STATUS_CUDA_ERROR;
    if (!(configured & (1ull << dev))) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess)
            return GPLK_STATUS_LAUNCH_FAIL;
        configured |= 1ull << dev;
    }
    const int csize = (M == Mode::GateUp ? 2 : 1) * p.split;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(clusters * csize));
    cfg.blockDim = dim3(kThreads<IMAGE>);
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

// Tensor map of `rows` weight rows of K / 2 bytes, boxes of 128 rows x 128 bytes.
static int encode_weights(CUtensorMap* map, const uint8_t* W, uint64_t rows, int K) {
    return encode_tmap_2d_u8(map, W, (uint64_t)K / 2, rows, (uint64_t)K / 2, 128, kTileRows);
}

// Whether the activations are converted once, by a kernel of their own, or by
// every block for itself.
static bool use_image(int T, int K) { return (long long)T * K > 32768; }

// Workspace of the converted activations: the stages' images, then the
// tokens' largest magnitudes.
static size_t image_bytes(int k_stages, const Geometry& g) { return (size_t)k_stages * ((size_t)g.nb * 128 + g.sfb_bytes); }

template <typename XT>
static int launch_gemv(Params& p, const Shape& s, const CUtensorMap& tm, void* workspace, cudaStream_t stream) {
    if (!workspace) return launch_stream<Mode::Gemv, XT, XT>(tm, tm, p, s.smem, p.tiles, stream);
    uint8_t* image = static_cast<uint8_t*>(workspace);
    const Geometry g = geometry(p.T, p.ring_bytes, p.tmem_cols);
    uint32_t* amax = reinterpret_cast<uint32_t*>(image + image_bytes(p.k_stages, g));
    const int st = launch_status(launch_pdl(image_kernel<XT>, dim3((unsigned)p.T), dim3(kImageThreads), 0, stream,
                                            static_cast<const XT*>(p.X), image, amax, p.K, p.ldx, p.x_vec, g.nb,
                                            g.sfb_bytes));
    if (st != GPLK_STATUS_OK) return st;
    p.image = image;
    p.amax = amax;
    return launch_stream<Mode::Gemv, XT, XT, true>(tm, tm, p, s.smem, p.tiles, stream);
}

}  // namespace fewtok
}  // namespace gplk

extern "C" size_t gplk_gemv_nvfp4_workspace_bytes(int T, int N, int K) {
    using namespace gplk::fewtok;
    if (T <= 0 || T > kMaxTokens || N <= 0 || K <= 0 || K % 64 != 0 || !use_image(T, K)) return 0;
    return image_bytes((K + kStageK - 1) / kStageK, geometry(T, 0, 512)) + sizeof(uint32_t) * kMaxTokens;
}

extern "C" int gplk_gemv_nvfp4(const void* X, const uint8_t* W, const uint8_t* SF, void* Y, const void* R, int T,
                               int N, int K, int ldx, int ldy, int ldr, const float* alpha, int dtype,
                               void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    using namespace gplk;
    using namespace gplk::fewtok;
    if (T < 0 || N < 0 || K < 0 || T > kMaxTokens) return GPLK_STATUS_BAD_ARG;
    if (dtype != GPLK_DTYPE_BF16 && dtype != GPLK_DTYPE_F16) return GPLK_STATUS_BAD_ARG;
    if (T == 0 || N == 0) return GPLK_STATUS_OK;
    if (K == 0 || K % 64 != 0 || ldx < K || ldy < N || (R && ldr < N)) return GPLK_STATUS_BAD_ARG;
    if (N > INT_MAX / 8) return GPLK_STATUS_BAD_ARG;  // N / 128 tiles of 8 slices fit a grid
    if (!X || !W || !SF || !Y || !alpha) return GPLK_STATUS_BAD_ARG;
    if (!aligned16(W) || !aligned16(SF) || !aligned(X, 2) || !aligned(Y, 2) || !aligned(R, 2) || !aligned(alpha, 4) ||
        !aligned16(workspace))
        return GPLK_STATUS_BAD_ARG;
    DeviceInfo d;
    int st = require_sm100(&d);
    if (st != GPLK_STATUS_OK) return st;
    Params p;
    memset(&p, 0, sizeof(p));
    p.X = X;
    p.sf0 = SF;
    p.alpha0 = alpha;
    p.Y = Y;
    p.R = R;
    p.T = T;
    p.N = N;
    p.K = K;
    p.ldx = ldx;
    p.ldy = ldy;
    p.ldr = ldr;
    p.x_vec = aligned16(X) && (T == 1 || ldx % 8 == 0);
    p.tiles = (N + kTileRows - 1) / kTileRows;
    p.k_stages = (K + kStageK - 1) / kStageK;
    p.kblocks = K / 64;
    const Shape s = set_shape(p, is_wide(T));
    if (s.smem > (size_t)d.max_smem_optin) return GPLK_STATUS_UNSUPPORTED;
    p.split = choose_split(p.tiles, p.k_stages, 8, s.per_sm * d.sm_count);
    CUtensorMap tm;
    st = encode_weights(&tm, W, (uint64_t)N, K);
    if (st != GPLK_STATUS_OK) return st;
    const size_t need = gplk_gemv_nvfp4_workspace_bytes(T, N, K);
    void* ws = need > 0 && workspace_bytes >= need ? workspace : nullptr;
    return dtype == GPLK_DTYPE_BF16 ? launch_gemv<__nv_bfloat16>(p, s, tm, ws, stream)
                                    : launch_gemv<__half>(p, s, tm, ws, stream);
}
