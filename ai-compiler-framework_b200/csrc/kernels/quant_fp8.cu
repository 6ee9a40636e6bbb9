// OpKind::QuantFp8: a matrix to 8-bit floating point with one fp32 scale per block of 128 values.
//
//   input   x [M,N] f32 | f16 | bf16, unit column stride
//   outputs [q, s]           q [M,N] f8e4m3 | f8e5m2, unit column stride; the shape of s says which blocks share a scale:
//             s [M, ceil(N/128)]               1 x 128 along each row
//             s [ceil(M/128), N]               128 x 1 along each column
//             s [ceil(M/128), ceil(N/128)]     128 x 128 tiles
//           [q, s, q', s']   the row form and the column form of the same matrix, x read once
//
// With F the format's largest value (448, 57344) and amax the block's largest magnitude, but at least 2^-100:
//   s = amax / F,   q = round_to_nearest_even(x * (F / amax)),   x ~ q * s
// (both quotients and the product in fp32, one rounding each; the lower limit keeps F / amax finite, and a block of
// zeros gets zeros). A NaN or an infinity in a block makes its scale NaN or infinite and its own value NaN.
//
// A block of 256 threads owns one 128 x 128 tile and keeps it in registers (8 rows of 8 columns per thread), so all
// three forms come from one read.
#include <cuda_fp8.h>

#include "common.cuh"

namespace aicf::cuda {

namespace {

constexpr int kBlk = 128;
constexpr int kQThreads = 256;
constexpr int kColsPerThread = 8;
constexpr int kLanesPerRow = kBlk / kColsPerThread;        // 16 threads cover a row of the tile
constexpr int kRowsPerPass = kQThreads / kLanesPerRow;     // 16
constexpr int kPasses = kBlk / kRowsPerPass;               // 8
constexpr float kTiny = 7.888609052210118e-31f;            // 2^-100

enum QuantForms : int { kRowForm = 1, kColForm = 2, kTileForm = 4 };

struct QuantOut {
  uint8_t* q = nullptr;
  float* s = nullptr;
  int64_t ld = 0;        // row pitch of q, elements
  int64_t s0 = 0, s1 = 0;  // strides of s
  int e5m2 = 0;
  int vec = 0;           // 8-byte stores allowed
};
struct QuantParams {
  const void* x;
  int64_t ldx, M, N;
  int64_t tiles_n;
  int vec_in;
  QuantOut row, col;     // the tile form uses `row`
};

// |a| and b, NaN wins
__device__ __forceinline__ float amax_of(float b, float a) {
  float r;
  asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %1;\n\tmax.NaN.f32 %0, t, %2;\n\t}" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t to_fp8x2(float a, float b, int e5m2) {
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, e5m2 ? __NV_E5M2 : __NV_E4M3));
}
__device__ __forceinline__ float top_of(int e5m2) { return e5m2 ? 57344.0f : 448.0f; }

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, int valid, float (&f)[8]) {
  if (vec && valid >= 8) {
    if constexpr (sizeof(T) == 4) {
      float a[4], b[4];
      unpack16(ld_stream(reinterpret_cast<const Pack16<T>*>(p)), a);
      unpack16(ld_stream(reinterpret_cast<const Pack16<T>*>(p) + 1), b);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = a[e], f[4 + e] = b[e];
    } else {
      unpack16(ld_stream(reinterpret_cast<const Pack16<T>*>(p)), f);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < valid ? Cvt<T>::to_f(p[e]) : 0.0f;
  }
}

__device__ __forceinline__ void store8(const QuantOut& o, int64_t row, int64_t col, int valid, const float (&f)[8], const float (&inv)[8]) {
  if (valid <= 0) return;
  uint32_t h[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = to_fp8x2(f[2 * e] * inv[2 * e], f[2 * e + 1] * inv[2 * e + 1], o.e5m2);
  uint8_t* dst = o.q + row * o.ld + col;
  if (o.vec && valid >= 8) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid) dst[e] = static_cast<uint8_t>(h[e >> 1] >> (8 * (e & 1)));
  }
}

template <typename T, int kForms>
__global__ void __launch_bounds__(kQThreads) quant_fp8_kernel(const QuantParams p) {
  __shared__ float part[kQThreads / 32][kBlk];
  const int cg = threadIdx.x % kLanesPerRow, rl = threadIdx.x / kLanesPerRow;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t tm = blockIdx.x / p.tiles_n, tn = blockIdx.x % p.tiles_n;
  const int64_t row0 = tm * kBlk + rl, col = tn * kBlk + cg * kColsPerThread;
  const int valid = p.N - col >= 8 ? 8 : static_cast<int>(p.N - col);  // columns of this thread inside the matrix
  float v[kPasses][8];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int64_t row = row0 + i * kRowsPerPass;
    load8(static_cast<const T*>(p.x) + row * p.ldx + col, p.vec_in != 0, row < p.M ? valid : 0, v[i]);
  }
  if constexpr ((kForms & kRowForm) != 0) {
    const float top = top_of(p.row.e5m2);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int64_t row = row0 + i * kRowsPerPass;
      float a = kTiny;
#pragma unroll
      for (int e = 0; e < 8; ++e) a = amax_of(a, v[i][e]);
#pragma unroll
      for (int o = kLanesPerRow / 2; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
      const float k = top / a;
      const float inv[8] = {k, k, k, k, k, k, k, k};
      if (row < p.M) {
        store8(p.row, row, col, valid, v[i], inv);
        if (cg == 0) p.row.s[row * p.row.s0 + tn * p.row.s1] = a / top;
      }
    }
  }
  if constexpr ((kForms & kColForm) != 0) {
    const float top = top_of(p.col.e5m2);
    float a[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e] = kTiny;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) a[e] = amax_of(a[e], v[i][e]);
      a[e] = max_nan(a[e], __shfl_xor_sync(0xffffffffu, a[e], 16));
      if (lane < 16) part[warp][cg * 8 + e] = a[e];
    }
    __syncthreads();
    float inv[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e] = part[0][cg * 8 + e];
#pragma unroll
      for (int w = 1; w < kQThreads / 32; ++w) a[e] = max_nan(a[e], part[w][cg * 8 + e]);
      inv[e] = top / a[e];
      if (rl == 0 && e < valid) p.col.s[tm * p.col.s0 + (col + e) * p.col.s1] = a[e] / top;
    }
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int64_t row = row0 + i * kRowsPerPass;
      if (row < p.M) store8(p.col, row, col, valid, v[i], inv);
    }
  }
  if constexpr (kForms == kTileForm) {
    const float top = top_of(p.row.e5m2);
    float a = kTiny;
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) a = amax_of(a, v[i][e]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
    if (lane == 0) part[0][warp] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQThreads / 32; ++w) a = max_nan(a, part[0][w]);
    const float k = top / a;
    const float inv[8] = {k, k, k, k, k, k, k, k};
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int64_t row = row0 + i * kRowsPerPass;
      if (row < p.M) store8(p.row, row, col, valid, v[i], inv);
    }
    if (threadIdx.x == 0) p.row.s[tm * p.row.s0 + tn * p.row.s1] = a / top;
  }
}

int64_t blocks_of(int64_t n) { return (n + kBlk - 1) / kBlk; }

// Which form a scale matrix describes for an M x N input; 0 = none. Where two readings of the shape agree (M = 1, say)
// the blocks agree, too.
int form_of(const TensorDesc& s, int64_t M, int64_t N) {
  if (s.dtype != DType::kF32 || s.rank() != 2 || s.stride[0] <= 0 || s.stride[1] <= 0) return 0;
  if (s.shape[0] == M && s.shape[1] == blocks_of(N)) return kRowForm;
  if (s.shape[0] == blocks_of(M) && s.shape[1] == N) return kColForm;
  if (s.shape[0] == blocks_of(M) && s.shape[1] == blocks_of(N)) return kTileForm;
  return 0;
}
bool rows_ok(const TensorDesc& t, int64_t M, int64_t N) {
  return t.rank() == 2 && t.shape[0] == M && t.shape[1] == N && (N == 1 || t.stride[1] == 1) && (M == 1 || t.stride[0] >= N);
}
int64_t pitch_of(const TensorDesc& t) { return t.shape[0] == 1 ? t.shape[1] : t.stride[0]; }

bool quant_check(const TensorDesc* in, int ni, const TensorDesc* out, int no, int* forms) {
  if (!in || !out || ni != 1 || (no != 2 && no != 4)) return false;
  const TensorDesc& x = in[0];
  if (x.rank() != 2 || x.shape[0] <= 0 || x.shape[1] <= 0 || !dtype_is_float(x.dtype)) return false;
  const int64_t M = x.shape[0], N = x.shape[1];
  if (!rows_ok(x, M, N) || blocks_of(M) > 0x7fffffff / blocks_of(N)) return false;
  for (int i = 0; i < no; i += 2)
    if (!dtype_is_fp8(out[i].dtype) || !rows_ok(out[i], M, N)) return false;
  *forms = form_of(out[1], M, N);
  if (*forms == 0) return false;
  if (no == 4) {
    // M = 1 or N = 1 can make a shape fit two forms: what counts is that the pair is (rows, columns)
    const TensorDesc &sr = out[1], &sc = out[3];
    if (form_of(sc, M, N) == 0 || sr.shape[0] != M || sr.shape[1] != blocks_of(N) || sc.shape[0] != blocks_of(M) || sc.shape[1] != N)
      return false;
    *forms = kRowForm | kColForm;
  }
  return true;
}
bool quant_supported(const TensorDesc* in, int ni, const TensorDesc* out, int no, const void*) {
  int forms = 0;
  return quant_check(in, ni, out, no, &forms);
}

QuantOut out_of(const TensorDesc& q, const TensorDesc& s) {
  QuantOut o;
  o.q = static_cast<uint8_t*>(q.data);
  o.s = static_cast<float*>(s.data);
  o.ld = pitch_of(q);
  o.s0 = s.stride[0];
  o.s1 = s.stride[1];
  o.e5m2 = q.dtype == DType::kF8E5M2 ? 1 : 0;
  o.vec = aligned_to(q.data, 8) && o.ld % 8 == 0;
  return o;
}

template <typename T>
Status quant_run(const QuantParams& p, int forms, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>(blocks_of(p.M) * p.tiles_n);
  cudaGetLastError();
  switch (forms) {
    case kRowForm: quant_fp8_kernel<T, kRowForm><<<grid, kQThreads, 0, stream>>>(p); break;
    case kColForm: quant_fp8_kernel<T, kColForm><<<grid, kQThreads, 0, stream>>>(p); break;
    case kTileForm: quant_fp8_kernel<T, kTileForm><<<grid, kQThreads, 0, stream>>>(p); break;
    default: quant_fp8_kernel<T, (kRowForm | kColForm)><<<grid, kQThreads, 0, stream>>>(p); break;
  }
  return launch_status();
}

Status quant_launch(const TensorDesc* in, int ni, TensorDesc* out, int no, const void*, void*, size_t, cudaStream_t stream) {
  int forms = 0;
  if (!quant_check(in, ni, out, no, &forms)) return Status::InvalidArgument;
  QuantParams p{};
  p.x = in[0].data;
  p.M = in[0].shape[0];
  p.N = in[0].shape[1];
  p.ldx = pitch_of(in[0]);
  p.tiles_n = blocks_of(p.N);
  p.vec_in = aligned_to(p.x, 16) && (p.ldx * dtype_size_bytes(in[0].dtype)) % 16 == 0;
  if (no == 4) {
    p.row = out_of(out[0], out[1]);
    p.col = out_of(out[2], out[3]);
  } else {
    (forms == kColForm ? p.col : p.row) = out_of(out[0], out[1]);
  }
  if (in[0].dtype == DType::kF32) return quant_run<float>(p, forms, stream);
  if (in[0].dtype == DType::kBF16) return quant_run<__nv_bfloat16>(p, forms, stream);
  return quant_run<__half>(p, forms, stream);
}

size_t no_workspace(const TensorDesc*, int, const void*) { return 0; }

}  // namespace

KernelVariant make_quant_fp8_block128_variant() {
  KernelVariant v{};
  v.name = "quant_fp8_block128_sm100";
  v.flags = kKV_CaptureSafe;
  v.launch = quant_launch;
  v.supported = quant_supported;
  v.query_workspace = no_workspace;
  return v;
}

}  // namespace aicf::cuda
