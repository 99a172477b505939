// gplk_unity.cu - the single translation unit of libgplk.so. Kernels share
// the device status word in gplk_core.cu, so they are compiled together.
#include "gplk_core.cu"
#include "gplk_memstream.cu"
#include "gplk_sgemm.cu"
#include "gplk_gemm_pair.cu"
#include "gplk_gemm_tc.cu"
#include "gplk_nvfp4_stream.cu"
#include "gplk_gemv_nvfp4.cu"
#include "gplk_moe_nvfp4.cu"
#include "gplk_powervirus.cu"
#include "gplk_powervirus_noalloc.cu"
#include "gplk_gemm_lt.cu"
#include "gplk_fabric.cu"

// The other kernels that allocate TMEM share no SM with a few-token block
// (gplk_nvfp4_shape.cuh says why none may).
namespace gplk {
static_assert(fewtok::leaves_no_half(sizeof(gemm_tc::Smem<true, 256>)), "");
static_assert(fewtok::leaves_no_half(sizeof(gemm_tc::Smem<false, 256>)), "");
static_assert(fewtok::leaves_no_half(sizeof(gemm_tc::Smem<false, 128>)), "");
static_assert(fewtok::leaves_no_half(sizeof(gemm_tc::Smem<false, 64>)), "");
static_assert(fewtok::leaves_no_half(sizeof(pair::Smem<256>)), "");
static_assert(fewtok::leaves_no_half(sizeof(pair::Smem<128>)), "");
static_assert(fewtok::leaves_no_half(sizeof(pv::Smem)), "");
}  // namespace gplk
