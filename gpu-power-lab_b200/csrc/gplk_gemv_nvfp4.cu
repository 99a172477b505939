// gplk_gemv_nvfp4.cu - products of a few tokens with NVFP4 weights:
//   y[t][n] = alpha * sum_k x[t][k] * sf[n][k / 16] * w[n][k]  (+ r[t][n])
// with E2M1 weights and UE4M3 scales in the layout gplk_gemm_nvfp4_tn reads,
// 16-bit activations and FP32 sums, rounded once to the activations' type.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include <climits>

#include "gplk_ptx.cuh"

namespace gplk {
namespace fewtok {

constexpr int kMaxTokens = 32;

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (sizeof(T) == 4) return (float)v;
    else return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    return static_cast<T>(v);
}

// Byte offset of the scale of 16-group g of row r (see gplk_nvfp4_sf_bytes).
__device__ __forceinline__ size_t sf_offset(size_t r, int g, int kblocks4) {
    return ((r >> 7) * (size_t)kblocks4 + (size_t)(g >> 2)) * 512 + (r & 31) * 16 + ((r & 127) >> 5) * 4 + (g & 3);
}

__device__ __forceinline__ float sf_value(uint8_t b) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}

// Dot products of one weight row with up to 8 activation rows, over the
// 16-groups of one warp's lanes; the warp's sums end in every lane.
template <typename XT>
__device__ __forceinline__ void row_dots(const uint8_t* w, const uint8_t* sf, size_t row, int K, const XT* const* x,
                                         int nx, float (&acc)[8]) {
    const int kb4 = (K + 63) / 64;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
    for (int g = (int)lane_id(); g < K / 16; g += 32) {
        const uint2 c = *reinterpret_cast<const uint2*>(w + row * (size_t)(K / 2) + (size_t)g * 8);
        const float s = sf_value(sf[sf_offset(row, g, kb4)]);
        float v[16];
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const uint8_t byte = (uint8_t)((b < 4 ? c.x : c.y) >> (8 * (b & 3)));
            const __half2 h = __half2(__nv_cvt_fp4x2_to_halfraw2(byte, __NV_E2M1));
            v[2 * b] = __low2float(h) * s;
            v[2 * b + 1] = __high2float(h) * s;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < nx) {
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[i] = fmaf(v[j], to_f32(x[i][g * 16 + j]), acc[i]);
            }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int o = 16; o; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
}

struct GemvParams {
    const void* X;
    const uint8_t* W;
    const uint8_t* SF;
    void* Y;
    const void* R;
    const float* alpha;
    int T, N, K, ldx, ldy, ldr;
};

template <typename XT>
__global__ void __launch_bounds__(256) gemv_simple_kernel(const GemvParams p) {
    const int n = blockIdx.x * 8 + (int)warp_id_uniform();
    const int t0 = blockIdx.y * 8;
    if (n >= p.N) return;
    const int nx = min(8, p.T - t0);
    const XT* x[8];
    for (int i = 0; i < 8; ++i) x[i] = static_cast<const XT*>(p.X) + (size_t)(t0 + min(i, nx - 1)) * p.ldx;
    float acc[8];
    row_dots<XT>(p.W, p.SF, (size_t)n, p.K, x, nx, acc);
    const float alpha = *p.alpha;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < nx && lane_id() == (uint32_t)i) {
            float v = acc[i] * alpha;
            if (p.R) v += to_f32(static_cast<const XT*>(p.R)[(size_t)(t0 + i) * p.ldr + n]);
            static_cast<XT*>(p.Y)[(size_t)(t0 + i) * p.ldy + n] = from_f32<XT>(v);
        }
}

static inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace fewtok
}  // namespace gplk

extern "C" int gplk_gemv_nvfp4(const void* X, const uint8_t* W, const uint8_t* SF, void* Y, const void* R, int T,
                               int N, int K, int ldx, int ldy, int ldr, const float* alpha, int dtype,
                               cudaStream_t stream) {
    using namespace gplk;
    using namespace gplk::fewtok;
    if (T < 0 || N < 0 || K < 0 || T > kMaxTokens) return GPLK_STATUS_BAD_ARG;
    if (dtype != GPLK_DTYPE_BF16 && dtype != GPLK_DTYPE_F16) return GPLK_STATUS_BAD_ARG;
    if (T == 0 || N == 0) return GPLK_STATUS_OK;
    if (K == 0 || K % 64 != 0 || ldx < K || ldy < N || (R && ldr < N)) return GPLK_STATUS_BAD_ARG;
    if (!X || !W || !SF || !Y || !alpha) return GPLK_STATUS_BAD_ARG;
    if (!aligned16(W) || !aligned16(SF) || !aligned(X, 2) || !aligned(Y, 2) || !aligned(R, 2) || !aligned(alpha, 4))
        return GPLK_STATUS_BAD_ARG;
    DeviceInfo d;
    const int st = require_sm100(&d);
    if (st != GPLK_STATUS_OK) return st;
    const GemvParams p{X, W, SF, Y, R, alpha, T, N, K, ldx, ldy, ldr};
    const dim3 grid((unsigned)(((long)N + 7) / 8), (unsigned)((T + 7) / 8));
    if (dtype == GPLK_DTYPE_BF16) gemv_simple_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(p);
    else gemv_simple_kernel<__half><<<grid, 256, 0, stream>>>(p);
    return launch_status(cudaGetLastError());
}
