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
//
// The inner sums are tcgen05.mma.kind::f8f6f4 products (one k block = 128 bytes = one swizzle row = four MMAs of K = 32),
// each accumulated from zero in a tensor-memory buffer of its own; the outer sum is held in fp32 registers by the eight
// epilogue warps, which read a buffer back, scale it and add it while the next block is being multiplied. Roles, ring,
// bounded waits and the CTA pair are those of the 16-bit kernel (gemm_tcgen05.cu): warp 0 TMA producer, warp 1 MMA issuer.
// An operand contiguous along M / N instead of K is described to the MMA as MN-major, so no transposed copy is made.
// Operands that TMA cannot address (rows not 16-byte aligned, or neither stride one) are first copied to aligned rows in
// the workspace by repitch_kernel.
//
// What bounds a long K is the epilogue warps' chain per k block (barrier, tensor-memory load, scale, add): 8192^3 takes 520 us
// (2.1 PFLOP/s), of which the MMAs alone would need about 340 and the epilogue without any MMA takes 370 to 480. With 1000 along
// K it is storing the tiles (65536 x 8192: 710 us, with a mask 1310), with one row reading B (8192 x 8192: 23 us as called).
#include <cstdlib>
#include <type_traits>

#include "gemm_common.cuh"
#include "sm100_tcgen05.cuh"

namespace aicf::cuda {

using namespace sm100;

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

constexpr int kTileM = 128;        // rows of C per CTA
constexpr int kTileK = 128;        // bytes of K per stage: one scale block, one 128-byte swizzle row
constexpr int kUmmaK = 32;         // k extent of one kind::f8f6f4 MMA
constexpr int kChunkBytes = kTileK * 128;   // MN-major operands: 128 k rows of 128 bytes
constexpr int kRingBytes = 192 * 1024;
constexpr int kFirstEpiWarp = 4;   // warps 0-3: TMA, MMA, scales, scales
constexpr int kScaleGroup = 8;     // k blocks whose scales are staged at a time
constexpr int kGroupM = 16;        // tile rasterisation: 16 row tiles share their column tiles in L2
constexpr unsigned long long kWaitBudgetNs = 1000000000ull;

__device__ int g_fp8_status = 0;   // 0 ok; otherwise (role << 8) | reason of the first CTA that gave up

struct Fp8Params {
  void* C;
  const void* bias;
  const void* mask;      // ReLU-backward mask, dtype of C
  int64_t ldc, mask_ld, bias_stride;
  ScaleView sa, sb;
  int M, N, K;
  int c_dtype, bias_dtype;  // DType values, 0 = no bias
  int relu;
  int c_vec, mask_vec;   // rows of C (of the mask) allow 32-byte stores (16-byte loads)
  int bias_vec;          // fp32, unit stride, 16-byte aligned
  int a_mn_major, b_mn_major;
  uint32_t idesc;
  int a_bytes;           // A's bytes per stage: fewer than a whole tile when M is small and A K-major (rows beyond are never stored)
  int splits;            // CTAs of a cluster that share a tile, each with a range of k blocks (single-CTA kernel)
};

// Tile shapes. kCg CTAs work on one tile of kCg * 128 rows and kTn columns; each holds 128 rows of A and kTn / kCg columns of
// B per stage, and a 128 x kTn accumulator.
template <int kCg, int kTn, bool kVecB> struct Cfg {
  static constexpr int kBCols = kTn / kCg;
  static constexpr int kABytes = kTileM * kTileK;
  static constexpr int kStageBytes = kABytes + kBCols * kTileK;
  static constexpr int kStages = kRingBytes / kStageBytes;
  static constexpr int kBufs = kTn == 256 ? 2 : 4;          // accumulator buffers in tensor memory
  static constexpr int kTmem = kBufs * kTn;
  // Epilogue warps: two per 32 rows, half the tile's columns each. For the 256-column tile that is 128 fp32 sums a thread:
  // 384 threads are launched with 168 registers each, the first warpgroup gives up 112 of its own and the epilogue
  // warpgroups take 56 more: 128 * 56 + 256 * 224 = 384 * 168. (Sixteen warps of 64 columns spill at the 112 registers they
  // could have, and were slower: 1657 against 524 us at 8192^3.)
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 32 * (kFirstEpiWarp + kEpiWarps);
  static constexpr bool kRegShift = kTn == 256;
  static constexpr int kRegsLaunch = 168, kRegsRoles = 56, kRegsEpi = 224;
  static_assert(128 * kRegsRoles + 32 * kEpiWarps * kRegsEpi <= kThreads * kRegsLaunch, "the warpgroups' shares come out of the block's registers");
  static constexpr int kCols = kTn / (kEpiWarps / 4);       // columns per epilogue warp
  // columns per TMEM load: two sets of 32 next to 128 sums spill (599 against 480 us at 8192^3); next to 64 they are faster
  // (609 against 637 us), unless the columns' factors want registers, too (937 against 811 us for the weight gradient)
  static constexpr int kCh = kCols == 64 && !kVecB ? 32 : 16;
  // staged scales: two groups of kScaleGroup k blocks, each the rows' and then the columns' factors
  static constexpr int kColScales = kVecB ? kTn : 2;        // one per column, or one per 128-column block of the tile
  static constexpr int kGroupFloats = kScaleGroup * (kTileM + kColScales);
  static constexpr size_t kSmem = 1024 + kRingBytes + 256 + 2 * kGroupFloats * sizeof(float);
  static_assert(kBufs <= kStages, "one parity per block in flight");
  static_assert(16 * kStages + 8 * kBufs + 32 + 8 <= 256, "barriers fit their 256 bytes");
};

// Bounded wait of a whole warp: every lane leaves with the same answer. The clock behind the bound is read only after some
// tries: reading it costs more than a wait usually lasts.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int who) {
  for (int i = 0; i < 32; ++i)
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait_or_abort(bar, parity, abort_flag, &g_fp8_status, who, kWaitBudgetNs));
}
// True in one lane of a converged warp. The producer's and the issuer's loops run in the whole warp, so that addresses and
// descriptors stay in uniform registers, and only the asynchronous instructions are left to this lane: with the loop itself
// behind `lane == 0` every operand is moved to a uniform register first, and issuing one block's four MMAs and two commits
// took 630 cycles, more than executing them.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
template <int kCg>
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  if constexpr (kCg == 1)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle, for 8-bit elements.
//   K-major : rows of 128 B (128 elements of K); 1024 B between 8-row groups
//   MN-major: 128 k rows of 128 B (128 elements of M / N) per chunk; 1024 B between 8-k groups, kChunkBytes between chunks
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, int mn_major) {
  const uint64_t lbo = mn_major ? (kChunkBytes >> 4) : 1;
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (lbo << 16) | (uint64_t(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// kN (32 or 16) consecutive columns of this warp's 32 lanes; the registers may be read after tmem_ld_wait only.
template <int kN>
__device__ __forceinline__ void tmem_ld_start(uint32_t taddr, uint32_t (&r)[kN]) {
  if constexpr (kN == 32)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
// Waits for this warp's loads; naming the registers keeps their uses behind the wait.
template <int kN>
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[kN]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int j = 0; j < kN; ++j) asm volatile("" : "+r"(r[j]));
}

// Packed fp32 pairs: Blackwell's FMA pipe takes two per instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Shared memory by its 32-bit address: a generic pointer would take two of the epilogue's registers.
__device__ __forceinline__ float lds1(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 lds4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
  return v;
}
// Four bytes from global to shared memory, or zeros.
__device__ __forceinline__ void copy4(uint32_t dst, const float* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
// The product of two scales, held inside fp32's range: a block of zeros stays zero whatever its scales. A NaN stays one.
__device__ __forceinline__ float clamp_finite(float v) {
  float r;
  asm("{\n\t.reg .f32 t;\n\tmin.NaN.f32 t, %1, 0f7F7FFFFF;\n\tmax.NaN.f32 %0, t, 0fFF7FFFFF;\n\t}" : "=f"(r) : "f"(v));
  return r;
}

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
// 32 bytes = one whole DRAM sector per store
__device__ __forceinline__ void st_sector(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// 32 consecutive columns of one row of C: bias and ReLU, or the ReLU-backward mask; convert; store.
// `ahead`: the 16-bit mask of these columns, loaded before the columns before them were finished.
__device__ __forceinline__ void load_mask32(const Fp8Params& p, int row, int col0, uint4 (&ahead)[4]) {
  if (p.mask && p.mask_vec && p.c_dtype != static_cast<int>(DType::kF32) && row < p.M && col0 + 32 <= p.N) {
    const uint4* ms = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.mask) + static_cast<int64_t>(row) * p.mask_ld + col0);
#pragma unroll
    for (int q = 0; q < 4; ++q) ahead[q] = __ldcs(ms + q);
  }
}
__device__ __forceinline__ void finish32(const Fp8Params& p, int row, int col0, float (&v)[32], const uint4 (&ahead)[4]) {
  if (p.bias_vec && col0 + 32 <= p.N) {  // the same address in every lane
    const float4* b = reinterpret_cast<const float4*>(static_cast<const float*>(p.bias) + col0);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float4 t = __ldg(b + q);
      v[4 * q] += t.x, v[4 * q + 1] += t.y, v[4 * q + 2] += t.z, v[4 * q + 3] += t.w;
    }
  } else if (p.bias_dtype != 0) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (col0 + j < p.N) v[j] += load_as_f32(p.bias, (col0 + j) * p.bias_stride, p.bias_dtype);
  }
  if (p.relu) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];  // a NaN stays one
  }
  if (row >= p.M) return;
  const bool whole = col0 + 32 <= p.N;
  const bool f32 = p.c_dtype == static_cast<int>(DType::kF32), bf16 = p.c_dtype == static_cast<int>(DType::kBF16);
  if (p.mask) {
    if (whole && p.mask_vec && !f32) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t w[4] = {ahead[q].x, ahead[q].y, ahead[q].z, ahead[q].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float lo, hi;
          if (bf16) {
            lo = __uint_as_float(w[e] << 16), hi = __uint_as_float(w[e] & 0xFFFF0000u);
          } else {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
            lo = t.x, hi = t.y;
          }
          if (!(lo > 0.0f)) v[8 * q + 2 * e] = 0.0f;
          if (!(hi > 0.0f)) v[8 * q + 2 * e + 1] = 0.0f;
        }
      }
    } else {
      const int64_t moff = static_cast<int64_t>(row) * p.mask_ld + col0;
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col0 + j < p.N && !(load_as_f32(p.mask, moff + j, p.c_dtype) > 0.0f)) v[j] = 0.0f;
    }
  }
  const int64_t off = static_cast<int64_t>(row) * p.ldc + col0;
  if (f32) {
    float* dst = static_cast<float*>(p.C) + off;
    if (whole && p.c_vec) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(v[8 * q + e]);
        st_sector(dst + 8 * q, w);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col0 + j < p.N) dst[j] = v[j];
    }
    return;
  }
  uint32_t w[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if (bf16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  uint16_t* dst = static_cast<uint16_t*>(p.C) + off;
  if (whole && p.c_vec) {
    st_sector(dst, w);
    st_sector(dst + 16, w + 8);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (col0 + j < p.N) dst[j] = static_cast<uint16_t>((j & 1) ? (w[j >> 1] >> 16) : (w[j >> 1] & 0xFFFFu));
  }
}

__device__ __forceinline__ void tile_of(int item, int tiles_m, int tiles_n, int group, int* tm, int* tn) {
  const int per_group = group * tiles_n;
  const int g = item / per_group;
  const int first = g * group;
  const int rows = min(group, tiles_m - first);
  const int in_group = item - g * per_group;
  *tm = first + in_group % rows;
  *tn = in_group / rows;
}

// kVecB: the columns of B have a scale each (per = 1); otherwise 128 columns share one.
template <int kCg, int kTn, bool kVecB>
__global__ void __launch_bounds__(Cfg<kCg, kTn, kVecB>::kThreads, 1)
    gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const Fp8Params p) {
  using F = Cfg<kCg, kTn, kVecB>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;  // 128B swizzle atoms repeat every 1024 B
  uint8_t* base_ptr = smem_raw + (base - raw);
  // bar_empty[stage] is the completion of a k block's MMAs: the producer takes it as "stage free" and the epilogue as
  // "accumulator ready". The issuer is at most kBufs < kStages blocks ahead of the epilogue, so a parity names one block.
  const uint32_t bar_full = base + kRingBytes, bar_empty = bar_full + 8 * F::kStages,
                 bar_acc_empty = bar_empty + 8 * F::kStages, bar_sc_full = bar_acc_empty + 8 * F::kBufs, bar_sc_empty = bar_sc_full + 16;
  uint8_t* misc = base_ptr + kRingBytes + 16 * F::kStages + 8 * F::kBufs + 32;
  const uint32_t scales_a = base + kRingBytes + 256;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(misc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = kCg == 2 || p.splits > 1 ? cluster_ctarank() : 0;
  const bool leader = kCg == 1 || rank == 0;
  const int splits = kCg == 1 ? p.splits : 1;
  // work items: tiles, taken round-robin by clusters; CTA `split` of a split cluster takes a range of the tile's k blocks
  const int first_item = kCg == 2 || splits > 1 ? static_cast<int>(cluster_id_x()) : static_cast<int>(blockIdx.x);
  const int item_step = kCg == 2 || splits > 1 ? static_cast<int>(cluster_count_x()) : static_cast<int>(gridDim.x);
  const int split = splits > 1 ? static_cast<int>(rank) : 0;
  const int tiles_m = (p.M + kCg * kTileM - 1) / (kCg * kTileM), tiles_n = (p.N + kTn - 1) / kTn;
  const int items = tiles_m * tiles_n;
  const int k_blocks = (p.K + kTileK - 1) / kTileK;
  const int kb_per = (k_blocks + splits - 1) / splits;
  const int kb_lo = split * kb_per, kb_hi = min(kb_lo + kb_per, k_blocks);

  if (threadIdx.x == 0) {
    for (int s = 0; s < F::kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < F::kBufs; ++b) mbar_init(bar_acc_empty + 8 * b, kCg * F::kEpiWarps);
    for (int g = 0; g < 2; ++g) {
      mbar_init(bar_sc_full + 8 * g, 64);          // the two scale warps' threads, when their copies have landed
      mbar_init(bar_sc_empty + 8 * g, F::kEpiWarps);
    }
    *abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 1) {
    const uint32_t slot = smem_addr(const_cast<uint32_t*>(tmem_slot));
    if constexpr (kCg == 1) tmem_alloc(slot, F::kTmem);
    else tmem_alloc_pair(slot, F::kTmem);
  }
  tc_fence_before();
  if constexpr (kCg == 2) cluster_sync_all();  // both CTAs' barriers exist before anybody signals across the pair
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp < kFirstEpiWarp) {
  if constexpr (F::kRegShift) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::kRegsRoles));
  if (warp == 0) {
    // ---------------- TMA producer: in a pair each CTA loads its own halves, completion lands on the leader's barrier
    {
      int stage = 0;
      uint32_t phase = 0;
      bool alive = true;
      for (int item = first_item; item < items && alive; item += item_step) {
        int tm, tn;
        tile_of(item, tiles_m, tiles_n, max(kGroupM / kCg, 1), &tm, &tn);
        const int m0 = (tm * kCg + (kCg == 2 ? static_cast<int>(rank) : 0)) * kTileM;
        const int n0 = tn * kTn + (kCg == 2 ? static_cast<int>(rank) * F::kBCols : 0);
        for (int kb = kb_lo; kb < kb_hi; ++kb) {
          if (!warp_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, 1)) { alive = false; break; }
          const uint32_t sa = base + stage * F::kStageBytes, sb = sa + F::kABytes;
          const int k0 = kb * kTileK;
          const int ax = p.a_mn_major ? m0 : k0, ay = p.a_mn_major ? k0 : m0;
          const int bx = p.b_mn_major ? n0 : k0, by = p.b_mn_major ? k0 : n0;
          if (elect_one()) {
          if constexpr (kCg == 2) {
            const uint32_t full = map_to_cta(bar_full + 8 * stage, 0);
            if (leader) mbar_expect_tx(bar_full + 8 * stage, 2 * (p.a_bytes + F::kBCols * kTileK));
            tma_load_2d_pair(sa, &tmap_a, ax, ay, full);
            tma_load_2d_pair(sb, &tmap_b, bx, by, full);
          } else {
            const uint32_t full = bar_full + 8 * stage;
            mbar_expect_tx(full, p.a_bytes + F::kBCols * kTileK);
            tma_load_2d(sa, &tmap_a, ax, ay, full);
            tma_load_2d(sb, &tmap_b, bx, by, full);
            if (kTn == 256 && p.b_mn_major) tma_load_2d(sb + kChunkBytes, &tmap_b, bx + 128, by, full);
          }
          }
          __syncwarp();
          if (++stage == F::kStages) { stage = 0; phase ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer: one lane, in a pair the leader's
    if (leader) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      bool alive = true;
      const uint32_t a_step = p.a_mn_major ? (kUmmaK * 128) >> 4 : kUmmaK >> 4;  // descriptor units of 16 B
      const uint32_t b_step = p.b_mn_major ? (kUmmaK * 128) >> 4 : kUmmaK >> 4;
      for (int item = first_item; item < items && alive; item += item_step) {
        for (int kb = kb_lo; kb < kb_hi; ++kb) {
          const uint32_t both = mbar_try_wait(bar_acc_empty + 8 * buf, buf_phase ^ 1u) & mbar_try_wait(bar_full + 8 * stage, phase);
          if (!__all_sync(0xffffffffu, both)) {
            if (!warp_wait(bar_acc_empty + 8 * buf, buf_phase ^ 1u, abort_flag, 2) || !warp_wait(bar_full + 8 * stage, phase, abort_flag, 3)) {
              alive = false;
              break;
            }
          }
          tc_fence_after();
          const uint32_t sa = base + stage * F::kStageBytes, sb = sa + F::kABytes;
          const uint64_t adesc = smem_desc(sa, p.a_mn_major), bdesc = smem_desc(sb, p.b_mn_major);
          if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kTileK / kUmmaK; ++k)
            umma_f8<kCg>(tmem_base + buf * kTn, adesc + k * a_step, bdesc + k * b_step, p.idesc, k != 0 ? 1u : 0u);
          if constexpr (kCg == 2) {
            umma_commit_pair(bar_empty + 8 * stage);
          } else {
            umma_commit(bar_empty + 8 * stage);
          }
          }
          __syncwarp();
          if (++stage == F::kStages) { stage = 0; phase ^= 1u; }
          if (++buf == F::kBufs) { buf = 0; buf_phase ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------- scales: both warps stage the factors of kScaleGroup k blocks at a time, two groups ahead at most.
    // Read where they are used, a row's factor would cost its warp an uncoalesced load (32 rows, 32 sectors) per k block.
    const int t = threadIdx.x - 64;
    int g = 0;
    uint32_t g_phase = 0;
    bool alive = true;
    for (int item = first_item; item < items && alive; item += item_step) {
      int tm, tn;
      tile_of(item, tiles_m, tiles_n, max(kGroupM / kCg, 1), &tm, &tn);
      const int m0 = (tm * kCg + (kCg == 2 ? static_cast<int>(rank) : 0)) * kTileM, n0 = tn * kTn;
      if (p.mask) {
        // the tile of the mask, on its way to L2 while the tile is multiplied: the input gradient of [65536,1000] x
        // [1000,8192] takes 710 us without a mask, 2250 with one read from HBM where it is used, 1310 so. (Turned into bits
        // here, it was 1250..3000 us and slowed the other products, in the epilogue before the tile 1700.)
        const int bytes = p.c_dtype == static_cast<int>(DType::kF32) ? 4 : 2;
        for (int i = t; i < kTileM * (kTn * bytes / 128); i += 64) {
          const int row = m0 + i % kTileM, col = n0 + i / kTileM * (128 / bytes);
          if (row < p.M && col < p.N)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(p.mask) + (static_cast<int64_t>(row) * p.mask_ld + col) * bytes));
        }
      }
      for (int kb0 = kb_lo; kb0 < kb_hi; kb0 += kScaleGroup) {
        if (!warp_wait(bar_sc_empty + 8 * g, g_phase ^ 1u, abort_flag, 5)) { alive = false; break; }
        // 4-byte asynchronous copies: nothing waits for one, and what lies outside the matrix becomes 0. (With loads through
        // registers, eight at a time, staging was what the weight gradient waited for.)
        const uint32_t rows_a = scales_a + 4 * g * F::kGroupFloats, cols_a = rows_a + 4 * kScaleGroup * kTileM;
        const int n = min(kScaleGroup, kb_hi - kb0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = m0 + t + 64 * h;
          const bool in = row < p.M;
          const float* src = p.sa.data + (in ? (row / p.sa.per) * p.sa.smn + kb0 * p.sa.sk : 0);
          for (int q = 0; q < n; ++q, src += in ? p.sa.sk : 0) copy4(rows_a + 4 * (q * kTileM + t + 64 * h), src, in);
        }
        if constexpr (kVecB) {
#pragma unroll 1
          for (int h = 0; h < kTn / 64; ++h) {
            const int col = n0 + t + 64 * h;
            const bool in = col < p.N;
            const float* src = p.sb.data + (in ? col * p.sb.smn + kb0 * p.sb.sk : 0);
            for (int q = 0; q < n; ++q, src += in ? p.sb.sk : 0) copy4(cols_a + 4 * (q * kTn + t + 64 * h), src, in);
          }
        } else if (t < 2 * n) {
          const int q = t >> 1, blk = n0 / kScaleBlk + (t & 1);  // a tile narrower than 128 columns lies in one block
          const bool in = blk * kScaleBlk < p.N;
          copy4(cols_a + 4 * t, p.sb.data + (in ? blk * p.sb.smn + (kb0 + q) * p.sb.sk : 0), in);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar_sc_full + 8 * g) : "memory");
        if (++g == 2) { g = 0; g_phase ^= 1u; }
      }
    }
  }
  } else {
    if constexpr (F::kRegShift) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F::kRegsEpi));
    // ---------------- epilogue warps: 32 lanes (rows) x kCols columns each, the outer sum in registers
    constexpr int kCols = F::kCols;
    const int sub = warp & 3, half = (warp - kFirstEpiWarp) >> 2;
    int buf = 0, stage = 0, g = 0;
    uint32_t phase = 0, g_phase = 0;
    bool alive = true;
    const uint32_t tmem_lane = tmem_base + (static_cast<uint32_t>(sub * 32) << 16) + half * kCols;
    for (int item = first_item; item < items && alive; item += item_step) {
      int tm, tn;
      tile_of(item, tiles_m, tiles_n, max(kGroupM / kCg, 1), &tm, &tn);
      int row = (tm * kCg + (kCg == 2 ? static_cast<int>(rank) : 0)) * kTileM + sub * 32 + lane;
      int col0 = tn * kTn + half * kCols;
      const bool idle = row - lane >= p.M || col0 >= p.N;  // nothing of this warp's part is stored: it only keeps pace
      uint64_t acc[kCols / 2];
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) acc[j] = 0ull;
      // A buffer is read in chunks of kCh columns through two register sets: while a chunk is scaled and added the next one
      // is on its way, and the first one of the next buffer while the last one of this is. The loop is rotated so that
      // every load stands at one place in it: a register set that is loaded at two places costs a copy per register.
      constexpr int kCh = F::kCh, kChunks = kCols / kCh;
      static_assert(kChunks % 2 == 0, "chunk c uses register set c & 1");
      uint32_t r[2][kCh];
      // One chunk scaled and added: by one factor, after the columns' factors at shared-memory address `vec` (kVecB).
      auto add_chunk = [&](int c, float f, uint32_t vec) {
        const uint32_t(&d)[kCh] = r[c & 1];
        const uint64_t f2 = pack2(f, f);
#pragma unroll
        for (int j = 0; j < kCh / 2; j += 2) {
          uint64_t d0 = pack2(__uint_as_float(d[2 * j]), __uint_as_float(d[2 * j + 1]));
          uint64_t d1 = pack2(__uint_as_float(d[2 * j + 2]), __uint_as_float(d[2 * j + 3]));
          if constexpr (kVecB) {
            const float4 b = lds4(vec + 4 * (kCh * c + 2 * j));
            d0 = mul2(d0, pack2(b.x, b.y));
            d1 = mul2(d1, pack2(b.z, b.w));
          }
          acc[kCh / 2 * c + j] = fma2(d0, f2, acc[kCh / 2 * c + j]);
          acc[kCh / 2 * c + j + 1] = fma2(d1, f2, acc[kCh / 2 * c + j + 1]);
        }
      };
      // The k blocks of one scale group at a time. What a block needs before its first load - its barrier, its factors - is
      // asked for while the block before it is still being added: asked for at the loop's top, their latencies alone came to
      // about as much as the block's MMAs take.
#pragma unroll 1
      for (int kb0 = kb_lo; kb0 < kb_hi; kb0 += kScaleGroup) {
        alive = warp_wait(bar_sc_full + 8 * g, g_phase, abort_flag, 6);
        if (!alive) break;
        const int n = min(kScaleGroup, kb_hi - kb0);
        if (idle) {
          for (int q = 0; q < n && alive; ++q) {
            alive = warp_wait(bar_empty + 8 * stage, phase, abort_flag, 4);
            if (lane == 0 && alive) {
              const uint32_t empty = bar_acc_empty + 8 * buf;
              if constexpr (kCg == 2) mbar_arrive_cluster(map_to_cta(empty, 0));
              else mbar_arrive(empty);
            }
            if (++buf == F::kBufs) buf = 0;
            if (++stage == F::kStages) { stage = 0; phase ^= 1u; }
          }
          if (!alive) break;
          if (lane == 0) mbar_arrive(bar_sc_empty + 8 * g);
          if (++g == 2) { g = 0; g_phase ^= 1u; }
          continue;
        }
        const uint32_t rows_a = scales_a + 4 * (g * F::kGroupFloats + sub * 32 + lane);
        const uint32_t cols_a = scales_a + 4 * (g * F::kGroupFloats + kScaleGroup * kTileM + (kVecB ? half * kCols : (half * kCols) / kScaleBlk));
        float f = 0.0f;
        uint32_t vec = cols_a;
#pragma unroll
        for (int j = 0; j < kCh; ++j) r[1][j] = 0u;  // "last chunk" before the group's first block: adds zeros
        float row_f = lds1(rows_a), col_f = kVecB ? 1.0f : lds1(cols_a);
        uint32_t ready = mbar_try_wait(bar_empty + 8 * stage, phase);
#pragma unroll 1
        for (int q = 0; q < n; ++q) {
          // the TMEM loads are warp-collective: the whole warp proceeds or the whole warp leaves
          if (!__all_sync(0xffffffffu, ready)) {
            alive = warp_wait(bar_empty + 8 * stage, phase, abort_flag, 4);
            if (!alive) break;
          }
          tc_fence_after();
          const uint32_t tbuf = tmem_lane + buf * kTn;
          tmem_ld_start<kCh>(tbuf, r[0]);
          add_chunk(kChunks - 1, f, vec);
          f = kVecB ? row_f : clamp_finite(row_f * col_f);
          vec = cols_a + 4 * q * kTn;
          if (++stage == F::kStages) { stage = 0; phase ^= 1u; }
#pragma unroll
          for (int c = 0; c + 1 < kChunks; ++c) {
            tmem_ld_wait<kCh>(r[c & 1]);
            tmem_ld_start<kCh>(tbuf + kCh * (c + 1), r[(c + 1) & 1]);
            if (c + 2 == kChunks) {
              const int next = q + 1 < n ? q + 1 : q;
              row_f = lds1(rows_a + 4 * next * kTileM);
              if (!kVecB) col_f = lds1(cols_a + 8 * next);
              ready = mbar_try_wait(bar_empty + 8 * stage, phase);
            }
            add_chunk(c, f, vec);
          }
          tmem_ld_wait<kCh>(r[1]);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            const uint32_t empty = bar_acc_empty + 8 * buf;
            if constexpr (kCg == 2) mbar_arrive_cluster(map_to_cta(empty, 0));
            else mbar_arrive(empty);
          }
          if (++buf == F::kBufs) buf = 0;
        }
        if (!alive) break;
        add_chunk(kChunks - 1, f, vec);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_sc_empty + 8 * g);
        if (++g == 2) { g = 0; g_phase ^= 1u; }
      }
      if (!alive) break;
      // the tile's place again: carried through the loop above it would cost registers that the sums need
      int again = item;
      asm volatile("" : "+r"(again));
      tile_of(again, tiles_m, tiles_n, max(kGroupM / kCg, 1), &tm, &tn);
      row = (tm * kCg + (kCg == 2 ? static_cast<int>(rank) : 0)) * kTileM + sub * 32 + lane;
      col0 = tn * kTn + half * kCols;
      if (splits > 1) {
        // this CTA's part of the sum, parked where the ring was: its last MMA has read it, and no load is in flight
        float* park = reinterpret_cast<float*>(base_ptr) + (sub * 32 + lane) * (kTn + 4) + half * kCols;
#pragma unroll
        for (int j = 0; j < kCols / 2; j += 2) {
          const float2 a = unpack2(acc[j]), b = unpack2(acc[j + 1]);
          *reinterpret_cast<float4*>(park + 2 * j) = make_float4(a.x, a.y, b.x, b.y);
        }
        break;  // a split cluster has one item
      }
      uint4 ahead[2][4];
      load_mask32(p, row, col0, ahead[0]);
#pragma unroll
      for (int c = 0; c < kCols / 32; ++c) {
        if (c + 1 < kCols / 32) load_mask32(p, row, col0 + 32 * (c + 1), ahead[(c + 1) & 1]);
        if (col0 + 32 * c < p.N) {
          float v[32];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 a = unpack2(acc[16 * c + j]);
            v[2 * j] = a.x, v[2 * j + 1] = a.y;
          }
          finish32(p, row, col0 + 32 * c, v, ahead[c & 1]);
        }
      }
      __syncwarp();
    }
  }

  if constexpr (kCg == 1) {
    if (splits > 1) {
      // Every CTA of the cluster adds the parts of its share of the tile, in split order, and stores it.
      cluster_sync_all();
      if (warp >= kFirstEpiWarp) {
        int tm, tn;
        tile_of(first_item, tiles_m, tiles_n, kGroupM, &tm, &tn);
        const int m0 = tm * kTileM, n0 = tn * kTn;
        const int rows = min(kTileM, p.M - m0);
        for (int i = static_cast<int>(rank) * (32 * F::kEpiWarps) + threadIdx.x - 32 * kFirstEpiWarp; i < rows * (kTn / 4); i += splits * 32 * F::kEpiWarps) {
          const int r = i / (kTn / 4), c = (i % (kTn / 4)) * 4;
          const uint32_t mine = base + (r * (kTn + 4) + c) * 4;
          float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          for (int sp = 0; sp < splits; ++sp) {
            float4 t;
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(t.x), "=f"(t.y), "=f"(t.z), "=f"(t.w) : "r"(map_to_cta(mine, sp)) : "memory");
            v[0] += t.x, v[1] += t.y, v[2] += t.z, v[3] += t.w;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t row = m0 + r, col = n0 + c + e;
            if (col >= p.N) break;
            if (p.bias_dtype != 0) v[e] += load_as_f32(p.bias, col * p.bias_stride, p.bias_dtype);
            if (p.relu && v[e] < 0.0f) v[e] = 0.0f;
            if (p.mask && !(load_as_f32(p.mask, row * p.mask_ld + col, p.c_dtype) > 0.0f)) v[e] = 0.0f;
            store_from_f32(p.C, row * p.ldc + col, p.c_dtype, v[e]);
          }
        }
      }
      cluster_sync_all();  // nobody leaves while a peer may still be reading its shared memory
    }
  }
  if (warp == 2 || warp == 3) asm volatile("cp.async.wait_all;" ::: "memory");
  if (*abort_flag) {
    // error path only: give loads that may still be in flight time to land before shared memory is released
    for (int i = 0; i < 64; ++i) __nanosleep(16384);
  }
  tc_fence_before();
  if constexpr (kCg == 2) cluster_sync_all();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (kCg == 1) tmem_dealloc(tmem_base, F::kTmem);
    else tmem_dealloc_pair(tmem_base, F::kTmem);
  }
}

// Copies an operand to rows that start on 16 bytes. `wide`: source rows allow 4-byte loads.
__global__ void __launch_bounds__(256) repitch_kernel(const uint8_t* __restrict__ src, int64_t rs, int64_t cs, int64_t rows, int64_t cols,
                                                      uint8_t* __restrict__ dst, int64_t ld, int wide) {
  const int64_t words = ld / 4;
  const int64_t total = rows * words, stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += stride) {
    const int64_t r = i / words, c = (i % words) * 4;
    const uint8_t* s = src + r * rs + c * cs;
    uint32_t w = 0;
    if (wide && c + 4 <= cols) {
      w = *reinterpret_cast<const uint32_t*>(s);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < cols) w |= static_cast<uint32_t>(s[e * cs]) << (8 * e);
    }
    *reinterpret_cast<uint32_t*>(dst + r * ld + c) = w;
  }
}

// ------------------------------------------------------------------ host side
// 0 = K-major, 1 = MN-major, -1 = TMA cannot address it as it is
int operand_major(const MatView& v, bool k_is_row) {
  const int64_t mn = k_is_row ? v.cols : v.rows, k = k_is_row ? v.rows : v.cols;
  const int64_t mn_stride = k_is_row ? v.cs : v.rs, k_stride = k_is_row ? v.rs : v.cs;
  if (!aligned_to(v.data, 16)) return -1;
  if ((k == 1 || k_stride == 1) && (mn == 1 || (mn_stride % 16 == 0 && mn_stride >= k))) return 0;
  if ((mn == 1 || mn_stride == 1) && (k == 1 || (k_stride % 16 == 0 && k_stride >= mn))) return 1;
  return -1;
}
// An operand as the kernel reads it: `inner` contiguous elements per line, `outer` lines `ld` bytes apart.
struct Operand {
  const uint8_t* data;
  int major;  // 0: inner = K, 1: inner = M / N
  int64_t inner, outer, ld;
  bool copied;
  size_t copy_bytes;
};
Operand operand_of(const MatView& v, bool k_is_row) {
  const int64_t mn = k_is_row ? v.cols : v.rows, k = k_is_row ? v.rows : v.cols;
  const int64_t mn_stride = k_is_row ? v.cs : v.rs, k_stride = k_is_row ? v.rs : v.cs;
  Operand o{static_cast<const uint8_t*>(v.data), operand_major(v, k_is_row), 0, 0, 0, false, 0};
  o.copied = o.major < 0;
  if (o.copied) o.major = mn_stride == 1 && k_stride != 1 ? 1 : 0;  // keeps the contiguous side contiguous
  o.inner = o.major == 0 ? k : mn;
  o.outer = o.major == 0 ? mn : k;
  o.ld = o.major == 0 ? mn_stride : k_stride;
  if (o.copied || o.outer == 1) o.ld = (o.inner + 15) / 16 * 16;
  if (o.copied) o.copy_bytes = (static_cast<size_t>(o.outer) * o.ld + 255) / 256 * 256;
  return o;
}
void repitch(const Operand& o, const MatView& v, bool k_is_row, uint8_t* dst, cudaStream_t stream) {
  const int64_t mn_stride = k_is_row ? v.cs : v.rs, k_stride = k_is_row ? v.rs : v.cs;
  const int64_t rs = o.major == 0 ? mn_stride : k_stride, cs = o.major == 0 ? k_stride : mn_stride;
  const int wide = cs == 1 && rs % 4 == 0 && aligned_to(v.data, 4);
  repitch_kernel<<<streaming_grid(o.outer * (o.ld / 4), 256, kStreamBlocksPerSm), 256, 0, stream>>>(
      static_cast<const uint8_t*>(v.data), rs, cs, o.outer, o.inner, dst, o.ld, wide);
}
bool encode(CUtensorMap* map, const uint8_t* data, const Operand& o, uint32_t mn_box) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(o.inner), static_cast<cuuint64_t>(o.outer)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(o.ld)};
  const cuuint32_t box[2] = {128, o.major == 0 ? mn_box : static_cast<cuuint32_t>(kTileK)};
  const cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(data), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Choice {
  int cg = 1, tn = 128, splits = 1;
};
// Tile shape by a cost model: rounds of tiles over the SMs (or SM pairs), each round the time of a tile's k blocks and of
// storing it. The times are those of one round, measured at K = 8192 and K = 1000 (microseconds per k block / per tile stored):
//                           k block, with a factor per column of B   stored, with a mask
//   256 x 256, CTA pair     0.54       0.72                            2.1     9.2
//   128 x 256               0.56       0.74                            2.0     7.3
//   128 x 128               0.34       0.45                            1.0     4.0
//   128 x 64                0.27       0.30                            0.6     2.2
// The narrow tiles may share K among the CTAs of a cluster (which costs about 3 us for the exchange): that is for few rows,
// where one round of unsplit tiles leaves each CTA a long serial walk along K (M = 1, 8192 x 8192: 33.7 us unsplit on 128 x 64
// tiles, 28.9 as two halves of 128 x 128).
// AICF_FP8_TILE=<ctas><columns> (2256, 1256, 1128, 164) and AICF_FP8_SPLITK=n override it (tuning and tests).
Choice choose(const Fp8Problem& q, bool b_n_major) {
  const GemmProblem& g = q.g;
  const int64_t sms = sm_count(), kb = blocks_of(g.K);
  const bool vec = q.sb.per == 1;
  struct Shape { int cg, tn; double block, store; };
  const bool mask = g.mask != nullptr;
  const Shape shapes[4] = {{2, 256, vec ? 0.72 : 0.54, mask ? 9.2 : 2.1}, {1, 256, vec ? 0.74 : 0.56, mask ? 7.3 : 2.0},
                           {1, 128, vec ? 0.45 : 0.34, mask ? 4.0 : 1.0}, {1, 64, vec ? 0.30 : 0.27, mask ? 2.2 : 0.6}};
  Choice best;
  double best_cost = 1e300;
  for (const Shape& s : shapes) {
    if (s.cg == 2 && g.M <= kTileM) continue;
    if (s.tn == 64 && b_n_major) continue;  // an N-major box is 128 columns wide
    const int64_t tiles = ((g.M + s.cg * kTileM - 1) / (s.cg * kTileM)) * ((g.N + s.tn - 1) / s.tn), slots = sms / s.cg > 0 ? sms / s.cg : 1;
    for (int splits = 1; splits <= (s.tn <= 128 ? 8 : 1); splits *= 2) {
      if (splits > 1 && (tiles * splits > slots || kb < 8 * splits)) break;
      const double rounds = static_cast<double>((tiles * splits + slots - 1) / slots);
      const double cost = rounds * (static_cast<double>((kb + splits - 1) / splits) * s.block + s.store) + (splits > 1 ? 3.0 : 0.0);
      if (cost < best_cost) best_cost = cost, best = Choice{s.cg, s.tn, splits};
    }
  }
  if (const char* e = std::getenv("AICF_FP8_TILE")) {
    const int v = std::atoi(e);
    if (v == 2256) best = Choice{2, 256, 1};
    if (v == 1256) best = Choice{1, 256, 1};
    if (v == 1128) best = Choice{1, 128, 1};
    if (v == 164) best = Choice{1, b_n_major ? 128 : 64, 1};
  }
  if (const char* e = std::getenv("AICF_FP8_SPLITK")) best.splits = std::atoi(e) < 8 ? std::atoi(e) : 8;
  if (best.cg == 2 || best.tn == 256 || best.splits < 1) best.splits = 1;
  while (best.splits > 1 && (best.splits > kb || (kb + best.splits - 1) / best.splits * (best.splits - 1) >= kb)) --best.splits;  // no empty part
  return best;
}

template <int kCg, int kTn, bool kVecB>
Status launch_tiles(const CUtensorMap& ta, const CUtensorMap& tb, const Fp8Params& p, cudaStream_t stream) {
  using F = Cfg<kCg, kTn, kVecB>;
  auto kernel = gemm_fp8_kernel<kCg, kTn, kVecB>;
  static PerDeviceOnce opt_in;
  if (!opt_in.run([&] {
        // a register hand-over that does not come out even would wait forever: refuse a build that has another count
        cudaFuncAttributes a{};
        return cudaFuncGetAttributes(&a, kernel) == cudaSuccess && (!F::kRegShift || a.numRegs == F::kRegsLaunch) &&
               cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(F::kSmem)) == cudaSuccess;
      })) {
    cudaGetLastError();
    return Status::Internal;
  }
  const int64_t items = ((static_cast<int64_t>(p.M) + kCg * kTileM - 1) / (kCg * kTileM)) * ((static_cast<int64_t>(p.N) + kTn - 1) / kTn);
  if (items > 0x7fffffff / 8) return Status::InvalidArgument;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(kCg == 2 ? 2 : p.splits);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(F::kThreads);
  cfg.dynamicSmemBytes = F::kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = kCg == 2 || p.splits > 1 ? 1 : 0;
  if (kCg == 2) {
    const int64_t pairs = sm_count() / 2 > 0 ? sm_count() / 2 : 1;
    cfg.gridDim = dim3(static_cast<unsigned>(2 * (items < pairs ? items : pairs)));
  } else if (p.splits > 1) {
    cfg.gridDim = dim3(static_cast<unsigned>(items * p.splits));
  } else {
    cfg.gridDim = dim3(static_cast<unsigned>(items < sm_count() ? items : sm_count()));
  }
  if (cudaLaunchKernelEx(&cfg, kernel, ta, tb, p) != cudaSuccess) {
    cudaGetLastError();
    return Status::Internal;
  }
  return launch_status();
}

Status run(const Fp8Problem& q, void* ws, size_t ws_bytes, cudaStream_t stream) {
  const GemmProblem& g = q.g;
  if (!encode_fn()) return Status::NotImplemented;
  // A is [M,K], B is [K,N]
  const Operand a = operand_of(g.A, false), b = operand_of(g.B, true);
  uint8_t* w = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ws) + 255) & ~uintptr_t(255));
  if (a.copied || b.copied) {
    if (!ws || ws_bytes < a.copy_bytes + b.copy_bytes + 256) return Status::InvalidArgument;
  }
  cudaGetLastError();
  if (a.copied) repitch(a, g.A, false, w, stream);
  if (b.copied) repitch(b, g.B, true, w + a.copy_bytes, stream);

  const Choice c = choose(q, b.major == 1);
  CUtensorMap ta, tb;
  // a box past the end of a short A would have TMA fill rows that nobody stores (M = 1, 8192 x 8192: 38.9 -> 33.7 us)
  const uint32_t a_rows = g.M < kTileM && a.major == 0 ? static_cast<uint32_t>((g.M + 7) / 8 * 8) : static_cast<uint32_t>(kTileM);
  if (!encode(&ta, a.copied ? w : a.data, a, a_rows) ||
      !encode(&tb, b.copied ? w + a.copy_bytes : b.data, b, static_cast<uint32_t>(c.tn / c.cg)))
    return Status::Internal;

  Fp8Params p{};
  p.C = const_cast<void*>(g.C.data);
  p.ldc = g.M == 1 ? g.N : g.C.rs;
  p.c_dtype = static_cast<int>(g.C.dtype);
  const int64_t c_bytes = dtype_size_bytes(g.C.dtype);
  p.c_vec = aligned_to(p.C, 32) && (p.ldc * c_bytes) % 32 == 0;
  p.bias = g.bias;
  p.bias_stride = g.bias_stride;
  p.bias_dtype = g.bias ? static_cast<int>(g.bias_dtype) : 0;
  p.bias_vec = g.bias && g.bias_dtype == DType::kF32 && g.bias_stride == 1 && aligned_to(g.bias, 16);
  p.relu = g.relu ? 1 : 0;
  p.mask = g.mask;
  p.mask_ld = g.mask_ld;
  p.mask_vec = g.mask && aligned_to(g.mask, 16) && (g.mask_ld * c_bytes) % 16 == 0;
  p.sa = q.sa;
  p.sb = q.sb;
  p.M = static_cast<int>(g.M), p.N = static_cast<int>(g.N), p.K = static_cast<int>(g.K);
  p.a_mn_major = a.major, p.b_mn_major = b.major;
  p.a_bytes = static_cast<int>(a.major == 0 ? a_rows : kTileM) * kTileK;
  p.splits = c.splits;
  // instruction descriptor: D = f32 (bits 4-5 = 1), A / B format (bits 7-9 / 10-12: 0 = e4m3, 1 = e5m2), A / B major
  // (bits 15 / 16), N >> 3 (bits 17-22), M >> 4 (bits 24-28)
  p.idesc = (1u << 4) | (g.A.dtype == DType::kF8E5M2 ? 1u << 7 : 0u) | (g.B.dtype == DType::kF8E5M2 ? 1u << 10 : 0u) |
            (static_cast<uint32_t>(a.major) << 15) | (static_cast<uint32_t>(b.major) << 16) |
            (static_cast<uint32_t>(c.tn >> 3) << 17) | (static_cast<uint32_t>((c.cg * kTileM) >> 4) << 24);
  const bool vec = q.sb.per == 1;
  if (c.cg == 2) return vec ? launch_tiles<2, 256, true>(ta, tb, p, stream) : launch_tiles<2, 256, false>(ta, tb, p, stream);
  if (c.tn == 256) return vec ? launch_tiles<1, 256, true>(ta, tb, p, stream) : launch_tiles<1, 256, false>(ta, tb, p, stream);
  if (c.tn == 128) return vec ? launch_tiles<1, 128, true>(ta, tb, p, stream) : launch_tiles<1, 128, false>(ta, tb, p, stream);
  return vec ? launch_tiles<1, 64, true>(ta, tb, p, stream) : launch_tiles<1, 64, false>(ta, tb, p, stream);
}

// Bytes for the aligned copies of operands that TMA cannot address.
template <Epi kEpi>
size_t fp8_workspace(const TensorDesc* in, int ni, const void* attr) {
  if (!in || ni < 4 || in[0].rank() != 2 || in[1].rank() != 2) return 0;
  bool ta = false, tb = false, relu;
  if (kEpi == Epi::BiasRelu) read_gemm_epilogue_attr(attr, &ta, &tb, &relu);
  else read_gemm_attr(attr, &ta, &tb);
  const Operand a = operand_of(view_of(in[0], ta), false), b = operand_of(view_of(in[1], tb), true);
  return a.copied || b.copied ? a.copy_bytes + b.copy_bytes + 256 : 0;
}

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
  v.query_workspace = fp8_workspace<kEpi>;
  return v;
}

}  // namespace

// Status word of the bounded waits, as gemm_tcgen05_status().
int gemm_fp8_status(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_fp8_status, sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (clear && v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_fp8_status, &zero, sizeof(int));
  }
  return v;
}

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
