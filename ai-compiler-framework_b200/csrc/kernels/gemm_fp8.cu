// Products of block-scaled 8-bit matrices: the fp8 variants of OpKind::Gemm, OpKind::GemmEpilogue and
// OpKind::GemmReluBwd.
//
//   inputs [A, B, SA, SB]  /  [A, B, bias, SA, SB]  /  [dY, W, Y, SA, SB],  output C (f32 | bf16 | f16)
//
// A and B are f8e4m3 or f8e5m2 (each its own), shaped and transposed like the 16-bit variants' operands. Each has an fp32
// scale matrix whose shape is the STORED operand's with the extent summed over divided by 128 and the other one divided
// by 1 or by 128, which is what quant_fp8 writes (rows, columns or tiles). With K cut into blocks of 128,
//
//   C[m,n] = epilogue( sum over blocks kb of SA[m,kb] * SB[kb,n] * sum over k in kb of A[m,k] * B[k,n] )
#include <cuda_fp8.h>

#include "gemm_common.cuh"

namespace aicf::cuda {

namespace {

constexpr int kScaleBlk = 128;

// Scale of one operand: element (mn, kb) of the logical [MN, K/128] matrix is data[(mn / per) * smn + kb * sk].
struct ScaleView {
  const float* data = nullptr;
  int64_t smn = 0, sk = 0;
  int per = 1;  // rows (columns for B) that share a scale: 1 or 128
};

struct Fp8Problem {
  GemmProblem g;
  ScaleView sa, sb;
};

enum class Epi { None, BiasRelu, ReluBwdMask };

int64_t blocks_of(int64_t n) { return (n + kScaleBlk - 1) / kScaleBlk; }

bool scale_view(const TensorDesc& s, bool k_first, int64_t mn, int64_t k, ScaleView* v) {
  if (s.dtype != DType::kF32 || s.rank() != 2 || s.stride[0] <= 0 || s.stride[1] <= 0) return false;
  const int dk = k_first ? 0 : 1, dmn = 1 - dk;
  if (s.shape[dk] != blocks_of(k)) return false;
  if (s.shape[dmn] == mn) v->per = 1;
  else if (s.shape[dmn] == blocks_of(mn)) v->per = kScaleBlk;
  else return false;
  v->data = static_cast<const float*>(s.data);
  v->smn = s.stride[dmn];
  v->sk = s.stride[dk];
  return true;
}

bool check(DType c_dtype, Epi epi, const TensorDesc* in, int ni, const TensorDesc* out, int no, const void* attr, Fp8Problem* prob) {
  const int first = epi == Epi::None ? 2 : 3;  // operands before the scales
  if (!in || !out || ni != first + 2 || no != 1) return false;
  if (!dtype_is_fp8(in[0].dtype) || !dtype_is_fp8(in[1].dtype) || out[0].dtype != c_dtype) return false;
  bool ta = false, tb = false, relu = false;
  if (epi == Epi::BiasRelu) read_gemm_epilogue_attr(attr, &ta, &tb, &relu);
  else read_gemm_attr(attr, &ta, &tb);
  Fp8Problem p;
  if (!build_problem(in, epi == Epi::BiasRelu ? 3 : 2, out, no, epi == Epi::BiasRelu, ta, tb, relu, &p.g)) return false;
  if (p.g.M > 0x7fffff00 || p.g.N > 0x7fffff00 || p.g.K > 0x7fffff00) return false;
  if (p.g.N > 1 && p.g.C.cs != 1) return false;
  if (p.g.M > 1 && p.g.C.rs < p.g.N) return false;
  if (epi == Epi::BiasRelu && !dtype_is_float(in[2].dtype)) return false;
  if (epi == Epi::ReluBwdMask) {
    const TensorDesc& Y = in[2];
    if (Y.dtype != c_dtype || Y.rank() != 2 || Y.shape[0] != p.g.M || Y.shape[1] != p.g.N) return false;
    if ((p.g.N > 1 && Y.stride[1] != 1) || (p.g.M > 1 && Y.stride[0] < p.g.N)) return false;
    p.g.mask = Y.data;
    p.g.mask_ld = Y.stride[0];
  }
  if (!scale_view(in[first], ta, p.g.M, p.g.K, &p.sa) || !scale_view(in[first + 1], !tb, p.g.N, p.g.K, &p.sb)) return false;
  if (prob) *prob = p;
  return true;
}

struct Fp8Params {
  const uint8_t *A, *B;
  int64_t ars, acs, brs, bcs;
  int a_e5m2, b_e5m2;
  ScaleView sa, sb;
  void* C;
  int64_t ldc;
  int c_dtype;
  const void* bias;
  int64_t bias_stride;
  int bias_dtype, relu;
  const void* mask;
  int64_t mask_ld;
  int M, N, K;
};

__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int dtype) {
  if (dtype == static_cast<int>(DType::kF32)) return static_cast<const float*>(p)[i];
  if (dtype == static_cast<int>(DType::kBF16)) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_from_f32(void* p, int64_t i, int dtype, float v) {
  if (dtype == static_cast<int>(DType::kF32)) static_cast<float*>(p)[i] = v;
  else if (dtype == static_cast<int>(DType::kBF16)) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}
__device__ __forceinline__ float fp8_value(uint8_t b, int e5m2) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, e5m2 ? __NV_E5M2 : __NV_E4M3)));
}

// 64 x 64 outputs per block, 4 x 4 per thread, operands converted while they are staged; any strides.
__global__ void __launch_bounds__(256) gemm_fp8_tile_kernel(const Fp8Params p, int tiles_n) {
  __shared__ float As[16][64 + 1], Bs[16][64 + 1];
  const int m0 = static_cast<int>(blockIdx.x / tiles_n) * 64, n0 = static_cast<int>(blockIdx.x % tiles_n) * 64;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[4][4] = {}, part[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += 16) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int r = i / 16, c = i % 16;
      const int64_t m = m0 + r, n = n0 + r, k = k0 + c;
      As[c][r] = m < p.M && k < p.K ? fp8_value(p.A[m * p.ars + k * p.acs], p.a_e5m2) : 0.0f;
      Bs[c][r] = n < p.N && k < p.K ? fp8_value(p.B[k * p.brs + n * p.bcs], p.b_e5m2) : 0.0f;
    }
    __syncthreads();
    for (int k = 0; k < 16; ++k)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) part[i][j] = fmaf(As[k][ty + 16 * i], Bs[k][tx + 16 * j], part[i][j]);
    __syncthreads();
    if ((k0 + 16) % kScaleBlk == 0 || k0 + 16 >= p.K) {
      const int64_t kb = k0 / kScaleBlk;
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
          const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
          if (m < p.M && n < p.N)
            // one factor after the other: the product of the scales may leave fp32 where the result does not
            acc[i][j] += part[i][j] * p.sb.data[(n / p.sb.per) * p.sb.smn + kb * p.sb.sk] * p.sa.data[(m / p.sa.per) * p.sa.smn + kb * p.sa.sk];
          part[i][j] = 0.0f;
        }
    }
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m >= p.M || n >= p.N) continue;
      float v = acc[i][j];
      if (p.bias) v += load_as_f32(p.bias, n * p.bias_stride, p.bias_dtype);
      if (p.relu) v = fmaxf(v, 0.0f);
      if (p.mask && !(load_as_f32(p.mask, m * p.mask_ld + n, p.c_dtype) > 0.0f)) v = 0.0f;
      store_from_f32(p.C, m * p.ldc + n, p.c_dtype, v);
    }
}

Status run(const Fp8Problem& q, void*, size_t, cudaStream_t stream) {
  const GemmProblem& g = q.g;
  Fp8Params p{};
  p.A = static_cast<const uint8_t*>(g.A.data);
  p.B = static_cast<const uint8_t*>(g.B.data);
  p.ars = g.A.rs, p.acs = g.A.cs, p.brs = g.B.rs, p.bcs = g.B.cs;
  p.a_e5m2 = g.A.dtype == DType::kF8E5M2, p.b_e5m2 = g.B.dtype == DType::kF8E5M2;
  p.sa = q.sa, p.sb = q.sb;
  p.C = const_cast<void*>(g.C.data), p.ldc = g.C.rs, p.c_dtype = static_cast<int>(g.C.dtype);
  p.bias = g.bias, p.bias_stride = g.bias_stride, p.bias_dtype = static_cast<int>(g.bias_dtype), p.relu = g.relu;
  p.mask = g.mask, p.mask_ld = g.mask_ld;
  p.M = static_cast<int>(g.M), p.N = static_cast<int>(g.N), p.K = static_cast<int>(g.K);
  const int64_t tiles_m = (g.M + 63) / 64, tiles_n = (g.N + 63) / 64;
  if (tiles_m > 0x7fffffff / tiles_n) return Status::InvalidArgument;
  cudaGetLastError();
  gemm_fp8_tile_kernel<<<static_cast<unsigned>(tiles_m * tiles_n), 256, 0, stream>>>(p, static_cast<int>(tiles_n));
  return launch_status();
}

size_t no_workspace(const TensorDesc*, int, const void*) { return 0; }

template <DType kC, Epi kEpi>
bool supported(const TensorDesc* in, int ni, const TensorDesc* out, int no, const void* attr) {
  return check(kC, kEpi, in, ni, out, no, attr, nullptr);
}
template <DType kC, Epi kEpi>
Status launch(const TensorDesc* in, int ni, TensorDesc* out, int no, const void* attr, void* ws, size_t ws_bytes, cudaStream_t stream) {
  Fp8Problem p;
  if (!check(kC, kEpi, in, ni, out, no, attr, &p)) return Status::InvalidArgument;
  return run(p, ws, ws_bytes, stream);
}
template <DType kC, Epi kEpi>
KernelVariant variant(const char* name) {
  KernelVariant v{};
  v.name = name;
  v.flags = kKV_CaptureSafe;
  v.launch = launch<kC, kEpi>;
  v.supported = supported<kC, kEpi>;
  v.query_workspace = no_workspace;
  return v;
}

}  // namespace

KernelVariant make_gemm_fp8_block128_out_f32_variant() { return variant<DType::kF32, Epi::None>("gemm_fp8_block128_out_f32"); }
KernelVariant make_gemm_fp8_block128_out_bf16_variant() { return variant<DType::kBF16, Epi::None>("gemm_fp8_block128_out_bf16"); }
KernelVariant make_gemm_fp8_block128_out_f16_variant() { return variant<DType::kF16, Epi::None>("gemm_fp8_block128_out_f16"); }
KernelVariant make_gemm_bias_relu_fp8_block128_out_f32_variant() { return variant<DType::kF32, Epi::BiasRelu>("gemm_bias_relu_fp8_block128_out_f32"); }
KernelVariant make_gemm_bias_relu_fp8_block128_out_bf16_variant() { return variant<DType::kBF16, Epi::BiasRelu>("gemm_bias_relu_fp8_block128_out_bf16"); }
KernelVariant make_gemm_bias_relu_fp8_block128_out_f16_variant() { return variant<DType::kF16, Epi::BiasRelu>("gemm_bias_relu_fp8_block128_out_f16"); }
KernelVariant make_gemm_relu_bwd_fp8_block128_out_f32_variant() { return variant<DType::kF32, Epi::ReluBwdMask>("gemm_relu_bwd_fp8_block128_out_f32"); }
KernelVariant make_gemm_relu_bwd_fp8_block128_out_bf16_variant() { return variant<DType::kBF16, Epi::ReluBwdMask>("gemm_relu_bwd_fp8_block128_out_bf16"); }
KernelVariant make_gemm_relu_bwd_fp8_block128_out_f16_variant() { return variant<DType::kF16, Epi::ReluBwdMask>("gemm_relu_bwd_fp8_block128_out_f16"); }

}  // namespace aicf::cuda
