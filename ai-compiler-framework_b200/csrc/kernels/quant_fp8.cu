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
//   s = amax / F rounded to fp32,   q = the format's value nearest to x F / amax (ties to even),   x ~ q * s
// q is rounded once, from the exact quotient; the lower limit keeps F / amax finite, and a block of zeros gets zeros. A NaN or
// an infinity makes its block's scale NaN or infinite and its values NaN.
//
// A block of threads owns one 128 x 128 tile and keeps it in registers as it was read, eight columns of kRows rows per
// thread, so all forms come from one read. HBM bounds it (4 bytes per bf16 value for both forms), with instruction issue close
// behind: about 17 instructions per value for two forms, hence packed 16-bit maxima, one division per row and column of the
// tile, and the exact rounding below without a branch in the usual case. Measured: 65536 x 8192 bf16, both forms, 485 us (4.5 TB/s),
// the row form alone 287 us (5.7); 8192 x 8192 f32 tiles 78 us (4.3).
//
// Rounding. p = x inv + x inv_lo with inv + inv_lo = F / amax to 2^-48 is x F / amax rounded to fp32. Rounding p to eight bits
// gives the right value unless p is exactly half way between two of them, where the quotient itself may lie to either side:
// such a p (one in 2^20 fp32 values) is held against the quotient by the sign of x F - p amax. With 16-bit inputs it cannot
// happen: x F / amax = X F / A with X and A of at most 11 bits differs from a half-way point of 5 bits by 2^-16 of itself or
// not at all.
#include <cuda_fp8.h>

#include "common.cuh"

namespace aicf::cuda {

namespace {

constexpr int kBlk = 128;
constexpr int kLanesPerRow = 16;                           // eight columns each
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

__device__ __forceinline__ float top_of(int e5m2) { return e5m2 ? 57344.0f : 448.0f; }

// Magnitudes as integers: with the sign bit cleared, the order of the bit patterns is the order of the magnitudes, infinities
// and NaNs above everything. 16-bit types go two to a word.
template <typename T> struct Mag {
  static constexpr int kWords = 8;   // words that hold eight values
  __device__ __forceinline__ static uint32_t clear(uint32_t w) { return w & 0x7FFFFFFFu; }
  __device__ __forceinline__ static uint32_t max(uint32_t a, uint32_t b) { return a > b ? a : b; }
};
template <typename T> struct Mag16 {
  static constexpr int kWords = 4;
  __device__ __forceinline__ static uint32_t clear(uint32_t w) { return w & 0x7FFF7FFFu; }
  __device__ __forceinline__ static uint32_t max(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
};
template <> struct Mag<__half> : Mag16<__half> {};
template <> struct Mag<__nv_bfloat16> : Mag16<__nv_bfloat16> {};
// the value of a magnitude pattern (low half of the word for the 16-bit types)
template <typename T> __device__ __forceinline__ float mag_value(uint32_t w) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(w);
  } else {
    const uint16_t h = static_cast<uint16_t>(w);
    T t;
    memcpy(&t, &h, 2);
    return Cvt<T>::to_f(t);
  }
}

// What a block's largest magnitude comes down to.
struct Factor {
  float amax, inv, lo;  // F / amax = inv + lo
  __device__ __forceinline__ Factor() {}
  __device__ __forceinline__ Factor(float a, float top) {
    amax = a < kTiny ? kTiny : a;  // a NaN stays
    inv = top / amax;
    lo = fmaf(-amax, inv, top) * (inv / top);
  }
};

// Eight values as they lie in memory.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, int valid, uint32_t (&w)[Mag<T>::kWords]) {
  if (vec && valid >= 8) {
    const int4* src = reinterpret_cast<const int4*>(p);
#pragma unroll
    for (int i = 0; i < Mag<T>::kWords / 4; ++i) {
      const int4 t = __ldcs(src + i);
      w[4 * i] = t.x, w[4 * i + 1] = t.y, w[4 * i + 2] = t.z, w[4 * i + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < Mag<T>::kWords; ++i) w[i] = 0u;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < valid) w[e] = reinterpret_cast<const uint32_t*>(p)[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < valid) w[e >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[e]) << (16 * (e & 1));
    }
  }
}
template <typename T>
__device__ __forceinline__ void values8(const uint32_t (&w)[Mag<T>::kWords], float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(w[e]);
  } else {
    Pack16<T> p;
    *reinterpret_cast<uint4*>(&p) = make_uint4(w[0], w[1], w[2], w[3]);
    unpack16(p, f);
  }
}

// A p that lies exactly between two values of the format moves one step towards the exact quotient x F / amax, by the sign of
// x F - p amax: both products are exact in 64 bits (in pairs of fp32 numbers they overflow for blocks above 2^112).
// Not inlined: its registers would cost every value (8192 x 8192 fp32 tiles: 104 against 78 us).
__device__ __noinline__ float off_the_tie(float p, float x, float amax, float top) {
  const double d = fma(static_cast<double>(x), static_cast<double>(top), -static_cast<double>(p) * static_cast<double>(amax));
  const double towards = p < 0.0f ? -d : d;  // > 0: the quotient's magnitude is larger
  const int step = towards > 0.0 ? 1 : towards < 0.0 ? -1 : 0;
  return __int_as_float(__float_as_int(p) + step);
}

// Eight values to eight bytes. `amax(e)` is asked for in the rare case only.
template <typename T, typename Inv, typename Lo, typename Amax>
__device__ __forceinline__ uint2 quant8(const float (&x)[8], int e5m2, Inv inv, Lo lo, Amax amax) {
  float p[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) p[e] = fmaf(x[e], inv(e), x[e] * lo(e));
  if constexpr (sizeof(T) == 4) {
    const float least = e5m2 ? 6.103515625e-05f : 0.015625f;  // smallest normal value
    const uint32_t half = e5m2 ? 0x100000u : 0x80000u, mask = 2u * half - 1u;
    bool tie = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // a value below the normal range is lifted into it, where its half steps have the same bit pattern as everybody's (where
      // the lifting rounds, a tie may be seen that is none: it is looked at again)
      float y = fabsf(p[e]);
      asm("{\n\t.reg .pred q;\n\tsetp.lt.f32 q, %0, %1;\n\t@q add.f32 %0, %0, %1;\n\t}" : "+f"(y) : "f"(least));
      tie |= (__float_as_uint(y) & mask) == half;
    }
    if (__builtin_expect(tie, 0)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = fabsf(p[e]), y = a < least ? __fadd_rn(a, least) : a;
        if ((__float_as_uint(y) & mask) == half && (a >= least || __fadd_rn(y, -least) == a))
          p[e] = off_the_tie(p[e], x[e], amax(e), top_of(e5m2));
      }
    }
  }
  uint32_t h[4];
  if (e5m2) {
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __nv_cvt_float2_to_fp8x2(make_float2(p[2 * e], p[2 * e + 1]), __NV_SATFINITE, __NV_E5M2);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __nv_cvt_float2_to_fp8x2(make_float2(p[2 * e], p[2 * e + 1]), __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}
__device__ __forceinline__ void store8(const QuantOut& o, int64_t row, int64_t col, int valid, uint2 b) {
  uint8_t* dst = o.q + row * o.ld + col;
  if (o.vec && valid >= 8) {
    *reinterpret_cast<uint2*>(dst) = b;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid) dst[e] = static_cast<uint8_t>((e < 4 ? b.x : b.y) >> (8 * (e & 3)));
  }
}

// Rows per thread: 32 registers hold eight rows of a 16-bit type or four of fp32.
template <typename T> struct Shape {
  static constexpr int kRows = sizeof(T) == 4 ? 4 : 8;
  static constexpr int kThreads = kBlk / kRows * kLanesPerRow;  // 512 or 256
  static constexpr int kWarps = kThreads / 32;
  static constexpr int kRowStep = kThreads / kLanesPerRow;      // rows between a thread's rows
};

template <typename T, int kForms>
__global__ void __launch_bounds__(Shape<T>::kThreads, sizeof(T) == 4 ? 2 : kForms == (kRowForm | kColForm) ? 3 : 4) quant_fp8_kernel(const QuantParams p) {
  using G = Mag<T>;
  constexpr int kRows = Shape<T>::kRows, kWarps = Shape<T>::kWarps, kRowStep = Shape<T>::kRowStep, kW = G::kWords;
  __shared__ uint32_t part[kWarps][kLanesPerRow][kW];  // a warp's maxima of each lane's columns
  __shared__ float col_inv[kBlk], col_lo[kBlk], col_amax[kBlk], row_amax[kBlk];
  const int cg = threadIdx.x % kLanesPerRow, rl = threadIdx.x / kLanesPerRow;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t tm = blockIdx.x / p.tiles_n, tn = blockIdx.x % p.tiles_n;
  const int64_t row0 = tm * kBlk + rl, col = tn * kBlk + cg * 8;
  const int valid = p.N - col >= 8 ? 8 : p.N > col ? static_cast<int>(p.N - col) : 0;  // columns of this thread inside
  uint32_t w[kRows][kW];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t row = row0 + i * kRowStep;
    load8<T>(static_cast<const T*>(p.x) + row * p.ldx + col, p.vec_in != 0, row < p.M ? valid : 0, w[i]);
  }
  // ---- columns (and the tile): each lane's eight over its rows, over the two half warps, over the warps
  if constexpr (kForms != kRowForm) {
    uint32_t a[kW];
#pragma unroll
    for (int k = 0; k < kW; ++k) {
      a[k] = G::clear(w[0][k]);
#pragma unroll
      for (int i = 1; i < kRows; ++i) a[k] = G::max(a[k], G::clear(w[i][k]));
      a[k] = G::max(a[k], __shfl_xor_sync(0xffffffffu, a[k], 16));
    }
    if (lane < 16) {
#pragma unroll
      for (int k = 0; k < kW; k += 4) *reinterpret_cast<uint4*>(&part[warp][cg][k]) = make_uint4(a[k], a[k + 1], a[k + 2], a[k + 3]);
    }
  }
  // ---- rows: kRows maxima over the sixteen lanes of a row; 16-bit types two rows to a word
  Factor rf;            // of the row this lane works out: row cg of its kRows
  if constexpr ((kForms & kRowForm) != 0) {
    constexpr int kR = sizeof(T) == 4 ? kRows : kRows / 2;
    uint32_t a[kR];
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      if constexpr (sizeof(T) == 4) {
        a[i] = G::clear(w[i][0]);
#pragma unroll
        for (int k = 1; k < kW; ++k) a[i] = G::max(a[i], G::clear(w[i][k]));
      } else {
        uint32_t b[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          b[h] = G::clear(w[2 * i + h][0]);
#pragma unroll
          for (int k = 1; k < kW; ++k) b[h] = G::max(b[h], G::clear(w[2 * i + h][k]));
        }
        // low halves of both rows side by side, high halves too, then one maximum: row 2i below, row 2i + 1 above
        a[i] = G::max(__byte_perm(b[0], b[1], 0x5410), __byte_perm(b[0], b[1], 0x7632));
      }
#pragma unroll
      for (int o = kLanesPerRow / 2; o > 0; o >>= 1) a[i] = G::max(a[i], __shfl_xor_sync(0xffffffffu, a[i], o));
    }
    uint32_t mine = a[0];
#pragma unroll
    for (int i = 1; i < kR; ++i)
      if ((sizeof(T) == 4 ? cg : cg >> 1) == i) mine = a[i];
    if (sizeof(T) != 4 && (cg & 1)) mine >>= 16;
    rf = Factor(mag_value<T>(sizeof(T) == 4 ? mine : mine & 0xFFFFu), top_of(p.row.e5m2));
    const int64_t row = row0 + cg * kRowStep;
    if (cg < kRows) {
      row_amax[rl + cg * kRowStep] = rf.amax;
      if (row < p.M) p.row.s[row * p.row.s0 + tn * p.row.s1] = rf.amax / top_of(p.row.e5m2);
    }
  }
  Factor tile;
  if constexpr (kForms != kRowForm) {
    __syncthreads();
    if (threadIdx.x < kBlk) {
      const int k = threadIdx.x % 8, l = threadIdx.x / 8;  // column 8 l + k
      uint32_t a = 0u;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) a = G::max(a, sizeof(T) == 4 ? part[v][l][k % kW] : part[v][l][(k >> 1) % kW]);
      if (sizeof(T) != 4) a = (k & 1) ? a >> 16 : a & 0xFFFFu;
      if constexpr (kForms == kTileForm) {
        // the tile: over its columns, which are the first four warps' lanes
        a = __reduce_max_sync(0xffffffffu, a);
        if (lane == 0) col_amax[warp] = mag_value<T>(a);
      } else {
        const Factor f(mag_value<T>(a), top_of(p.col.e5m2));
        col_inv[threadIdx.x] = f.inv, col_lo[threadIdx.x] = f.lo, col_amax[threadIdx.x] = f.amax;
        const int64_t c = tn * kBlk + threadIdx.x;
        if (c < p.N) p.col.s[tm * p.col.s0 + c * p.col.s1] = f.amax / top_of(p.col.e5m2);
      }
    }
    __syncthreads();
    if constexpr (kForms == kTileForm) {
      // the bit patterns again, so that a NaN wins
      uint32_t a = __float_as_uint(col_amax[0]);
#pragma unroll
      for (int v = 1; v < 4; ++v) a = max(a, __float_as_uint(col_amax[v]));
      tile = Factor(__uint_as_float(a), top_of(p.row.e5m2));
      if (threadIdx.x == 0) p.row.s[tm * p.row.s0 + tn * p.row.s1] = tile.amax / top_of(p.row.e5m2);
    }
  } else {
    __syncwarp();  // row_amax: written and read within a row's sixteen lanes
  }
  float ci[8], cl[8];
  if constexpr ((kForms & kColForm) != 0) {
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const float4 a = *reinterpret_cast<const float4*>(&col_inv[cg * 8 + e]), b = *reinterpret_cast<const float4*>(&col_lo[cg * 8 + e]);
      ci[e] = a.x, ci[e + 1] = a.y, ci[e + 2] = a.z, ci[e + 3] = a.w;
      cl[e] = b.x, cl[e + 1] = b.y, cl[e + 2] = b.z, cl[e + 3] = b.w;
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t row = row0 + i * kRowStep;
    float f[8];
    values8<T>(w[i], f);
    float inv = tile.inv, lo = tile.lo;
    if constexpr ((kForms & kRowForm) != 0) {
      inv = __shfl_sync(0xffffffffu, rf.inv, (lane & 16) + i);
      lo = __shfl_sync(0xffffffffu, rf.lo, (lane & 16) + i);
    }
    if (row >= p.M || valid == 0) continue;
    if constexpr ((kForms & (kRowForm | kTileForm)) != 0)
      store8(p.row, row, col, valid, quant8<T>(f, p.row.e5m2, [&](int) { return inv; }, [&](int) { return lo; },
                                            [&](int) { return kForms == kTileForm ? tile.amax : row_amax[rl + i * kRowStep]; }));
    if constexpr ((kForms & kColForm) != 0)
      store8(p.col, row, col, valid, quant8<T>(f, p.col.e5m2, [&](int e) { return ci[e]; }, [&](int e) { return cl[e]; },
                                            [&](int e) { return col_amax[cg * 8 + e]; }));
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
    case kRowForm: quant_fp8_kernel<T, kRowForm><<<grid, Shape<T>::kThreads, 0, stream>>>(p); break;
    case kColForm: quant_fp8_kernel<T, kColForm><<<grid, Shape<T>::kThreads, 0, stream>>>(p); break;
    case kTileForm: quant_fp8_kernel<T, kTileForm><<<grid, Shape<T>::kThreads, 0, stream>>>(p); break;
    default: quant_fp8_kernel<T, (kRowForm | kColForm)><<<grid, Shape<T>::kThreads, 0, stream>>>(p); break;
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
