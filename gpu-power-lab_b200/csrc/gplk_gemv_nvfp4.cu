// gplk_gemv_nvfp4.cu - products of a few tokens with NVFP4 weights:
//   y[t][n] = alpha * sum_k x[t][k] * sf[n][k / 16] * w[n][k]  (+ r[t][n])
// on the main loop of gplk_nvfp4_stream.cu: the conversion of the activations
// ahead of it, the choice of its shape, and the entry point.
#include "gplk_ptx.cuh"

namespace gplk {
namespace fewtok {

// ---------------------------------------------------------------- conversion ahead of the products
// Writes the B rows and scales of every stage as the ring holds them, a block
// per token, so that the blocks of an Image kernel fetch them with one bulk
// copy per stage instead of each converting all of the tokens again.
// (512 / 1024 threads, us of the product: 32x8192x4096 12.2 / 12.6, 4x8192x8192 10.9 /
// 11.1, 16x8192x8192 13.8 / 13.5, 32x8192x8192 17.5 / 16.9, 4x8192x12288 15.0 / 14.6,
// 32x8192x12288 22.5 / 20.6, 32x16384x16384 43.6 / 39.6: 512 up to K = 8192.)
static int image_threads(int K) { return K <= 8192 ? 512 : 1024; }

template <typename XT>
__global__ void __launch_bounds__(1024)
    image_kernel(const XT* X, uint8_t* image, uint32_t* amax, int K, int ldx, int x_vec, const Geometry g) {
    __shared__ uint32_t top[32];
    constexpr int kHeld = 4;
    const int warps = (int)blockDim.x / 32;
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
    for (int i0 = warp; i0 < stages; i0 += kHeld * warps) {
        uint4 r[kHeld][2];
#pragma unroll
        for (int c = 0; c < kHeld; ++c) {
            r[c][0] = r[c][1] = make_uint4(0, 0, 0, 0);
            if (i0 + c * warps < stages) load(i0 + c * warps, r[c]);
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
    m = __reduce_max_sync(0xffffffffu, (int)lane < warps ? top[lane] : 0u);
    if (threadIdx.x == 0) amax[t] = m;
    constexpr int kPlanes = kPlanesOf<XT>;
    const int anchor = anchor_of<kPlanes>(m);
    auto emit = [&](int i, const uint4 (&r)[2]) {
        float v[8];
        widen<XT>(r, v);
        uint8_t* b_rows = image + (size_t)i * g.image;
        const bool inside = i * kStageK + (int)lane * 8 < K;
        convert<kPlanes>(v, anchor, t, inside, b_rows, b_rows + (size_t)g.nb * 128, g.sfb_step, lane);
    };
#pragma unroll
    for (int c = 0; c < kHeld; ++c)
        if (warp + c * warps < stages) emit(warp + c * warps, held[c]);
    for (int i = warp + kHeld * warps; i < stages; i += warps) {
        uint4 r[2];
        load(i, r);
        emit(i, r);
    }
}

constexpr int kSms = 148;

// Sizes and slices of a product of T tokens.
static void plan(Params& p, int planes, int T, int N, int K) {
    p.T = T;
    p.N = N;
    p.K = K;
    p.tiles = (N + kTileRows - 1) / kTileRows;
    p.k_stages = (K + kStageK - 1) / kStageK;
    p.kblocks = K / 64;
    const int per_sm = planes * T > 128 ? 1 : 2;
    p.split_log2 = choose_split_log2(p.tiles, p.k_stages, kSms, per_sm);
}
static int block_stages(const Params& p) { return ((p.k_stages - 1) >> p.split_log2) + 1; }

// Whether the activations are converted once, by a kernel of their own, or by
// every block for itself: that keeps up with the weights up to about four tokens
// a stage, and a launch costs as much as some 20 units (a token's stage) of it.
// Measured, fused / image, us: 2x16384x16384 29.2 / 29.8, 3x16384x16384 29.4 / 30.0
// (192 units in a block), 3x16384x4096 10.8 / 10.8, 4x16384x16384 33.5 / 30.1 (256),
// 4x16384x8192 19.6 / 18.4 (128), 4x4096x4096 6.2 / 6.7 (16), 6x4096x4096 7.2 / 7.0
// (24), 8x8192x2048 8.1 / 6.8, 8x16384x8192 30.6 / 18.6.
static bool use_image(const Params& p) { return p.T >= 4 && p.T * block_stages(p) >= 24; }

// Workspace of the converted activations: the stages' images, then the
// tokens' largest magnitudes. One size for both types.
static size_t image_bytes(int T, int k_stages) {
    return (size_t)k_stages * geometry(kMaxPlanes, T, 1, Fill::Image, 0, 0).image;
}

template <typename XT>
static int launch_gemv(Params& p, const Shape& s, const CUtensorMap& tm, void* workspace, cudaStream_t stream) {
    if (!workspace) return launch_stream<Mode::Gemv, XT, XT>(tm, tm, p, s.smem, p.tiles, stream);
    uint8_t* image = static_cast<uint8_t*>(workspace);
    uint32_t* amax = reinterpret_cast<uint32_t*>(image + image_bytes(p.T, p.k_stages));
    const int st = launch_status(launch_pdl(image_kernel<XT>, dim3((unsigned)p.T), dim3(image_threads(p.K)), 0, stream,
                                            static_cast<const XT*>(p.X), image, amax, p.K, p.ldx, p.x_vec,
                                            p.geo[0]));
    if (st != GPLK_STATUS_OK) return st;
    p.image = image;
    p.amax = amax;
    return launch_stream<Mode::Gemv, XT, XT, true>(tm, tm, p, s.smem, p.tiles, stream);
}

}  // namespace fewtok
}  // namespace gplk

extern "C" size_t gplk_gemv_nvfp4_workspace_bytes(int T, int N, int K) {
    using namespace gplk::fewtok;
    if (T <= 0 || T > kMaxTokens || N <= 0 || K <= 0 || K % 64 != 0 || N > INT_MAX / 8 ||
        K > INT_MAX / 8)
        return 0;
    Params p;
    memset(&p, 0, sizeof(p));
    bool any = false;
    for (int planes : {kPlanesBF16, kPlanesF16}) {
        plan(p, planes, T, N, K);
        any = any || use_image(p);
    }
    if (!any) return 0;
    return image_bytes(T, (K + kStageK - 1) / kStageK) + sizeof(uint32_t) * kMaxTokens;
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
    if (N > INT_MAX / 8 || K > INT_MAX / 8) return GPLK_STATUS_BAD_ARG;  // grids, sums of stages
    if (!X || !W || !SF || !Y || !alpha || X == Y) return GPLK_STATUS_BAD_ARG;
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
    p.ldx = ldx;
    p.ldy = ldy;
    p.ldr = ldr;
    p.x_vec = aligned16(X) && (T == 1 || ldx % 8 == 0);
    const int planes = dtype == GPLK_DTYPE_BF16 ? kPlanesBF16 : kPlanesF16;
    plan(p, planes, T, N, K);
    const size_t need = use_image(p) ? image_bytes(T, p.k_stages) + sizeof(uint32_t) * kMaxTokens : 0;
    void* ws = need > 0 && workspace_bytes >= need ? workspace : nullptr;
    const Shape s = set_shape(p, planes, T, false, 1, ws ? Fill::Image : Fill::Convert, block_stages(p));
    if (s.smem > (size_t)d.max_smem_optin) return GPLK_STATUS_UNSUPPORTED;
    CUtensorMap tm;
    st = encode_weights(&tm, W, N, 1, K);
    if (st != GPLK_STATUS_OK) return st;
    return dtype == GPLK_DTYPE_BF16 ? launch_gemv<__nv_bfloat16>(p, s, tm, ws, stream)
                                    : launch_gemv<__half>(p, s, tm, ws, stream);
}
