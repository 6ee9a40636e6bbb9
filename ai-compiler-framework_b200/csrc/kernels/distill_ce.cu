// OpKind::DistillCE: loss rows and logit gradient of a student distilled from a teacher's top logits, optionally mixed with
// the cross-entropy of labels.
//
//   inputs  [z (B,C) f32|bf16|f16, ids (B,K) i32, t (B,K) f32|bf16|f16 (, labels (B,) i32)]
//   outputs [dz like z, loss_row (B,) f32]  or  [loss_row]
//   attrs   'DSTL' <fff> scale, temperature T, alpha   (defaults 1/B, 1, 0)
//
// t holds the teacher's logits at the columns `ids`; an entry whose id lies outside [0,C) is padding. Per row, over the
// entries that are not padding, with p = softmax(t / T) and q = softmax(z / T):
//
//   loss = (1 - alpha) T^2 sum_k p_k (log p_k - log q_id(k))  +  alpha (logsumexp(z) - z_label)
//   dz_j = scale [ (1 - alpha) T (q_j - sum over k with id(k) = j of p_k)  +  alpha (softmax(z)_j - [j = label]) ]
//
// A row without entries has no distillation term, a row whose label lies outside [0,C) no label term (zero loss and zero
// gradient both times). The same column may stand in a row's list more than once. loss_row carries no `scale`.
// A row without either term gets zeros whatever its logits hold. dz may be z itself; otherwise outputs do not overlap inputs.
#include <array>
#include <map>
#include <mutex>

#include "row_pipeline.cuh"

namespace aicf::cuda {

namespace {

using rowk::block_reduce;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxTop = 1024;  // entries per row

struct DistillParams {
  const void* z;
  void* dz;                // null: loss only
  int64_t ldz, lddz;
  const int32_t* ids;
  const void* t;
  int t_dtype;
  const int32_t* labels;   // null: no label term
  float* loss;
  int64_t B, C;
  int K;
  float scale, temperature, alpha;
  // from these: 1 / T and log2(e) / T; the weights of both terms in the gradient, scale (1 - alpha) T and scale alpha;
  // (1 - alpha) T^2
  float invT, cT, grad_soft, grad_hard, loss_soft;
};

__device__ __forceinline__ float teacher_at(const DistillParams& p, int64_t i) {
  if (p.t_dtype == static_cast<int>(DType::kF32)) return static_cast<const float*>(p.t)[i];
  if (p.t_dtype == static_cast<int>(DType::kBF16)) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.t)[i]);
  return __half2float(static_cast<const __half*>(p.t)[i]);
}

// One block per row, the row read once per quantity: any row length, alignment and pitch.
template <typename T>
__global__ void __launch_bounds__(256) distill_multipass_kernel(const DistillParams p) {
  __shared__ float red[rowk::kMaxWarps + 1];
  __shared__ int col_s[kMaxTop + 1];    // columns to correct after the row is written: the row's entries, then its label
  __shared__ float w_s[kMaxTop + 1];    // what is taken from the gradient there
  const float invT = 1.0f / p.temperature;
  for (int64_t row = blockIdx.x; row < p.B; row += gridDim.x) {
    const T* z = static_cast<const T*>(p.z) + row * p.ldz;
    const int64_t label = p.labels && p.alpha > 0.0f ? p.labels[row] : -1;
    const bool known = label >= 0 && label < p.C;
    float m = -INFINITY;
    for (int64_t i = threadIdx.x; i < p.C; i += blockDim.x) m = fmaxf(m, Cvt<T>::to_f(z[i]));
    m = block_reduce<true>(m, red);
    float s = 0.0f, s1 = 0.0f;
    for (int64_t i = threadIdx.x; i < p.C; i += blockDim.x) {
      const float d = Cvt<T>::to_f(z[i]) - m;
      s += expf(d * invT);
      if (known) s1 += expf(d);
    }
    s = block_reduce<false>(s, red);
    s1 = block_reduce<false>(s1, red);
    // teacher
    float mt = -INFINITY;
    for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
      const int id = p.ids[row * p.K + k];
      const bool ok = id >= 0 && id < p.C;
      col_s[k] = ok ? id : -1;
      if (ok) mt = fmaxf(mt, teacher_at(p, row * p.K + k));
    }
    if (threadIdx.x == 0) {
      col_s[p.K] = known ? static_cast<int>(label) : -1;
      w_s[p.K] = p.alpha;
    }
    mt = block_reduce<true>(mt, red);
    if (mt == -INFINITY) mt = 0.0f;
    float st = 0.0f;
    for (int k = threadIdx.x; k < p.K; k += blockDim.x)
      if (col_s[k] >= 0) st += expf((teacher_at(p, row * p.K + k) - mt) * invT);
    st = block_reduce<false>(st, red);
    const bool some = !(st == 0.0f);  // no entries, or every entry has weight zero: no target
    float cross = 0.0f;
    const float soft_w = (1.0f - p.alpha) * p.temperature;
    for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
      if (!some || col_s[k] < 0) {
        w_s[k] = 0.0f;
        continue;
      }
      const float a = (teacher_at(p, row * p.K + k) - mt) * invT;
      const float pk = expf(a) / st;
      if (pk != 0.0f) cross += pk * (a - (Cvt<T>::to_f(z[col_s[k]]) - m) * invT);
      w_s[k] = soft_w * pk;
    }
    cross = block_reduce<false>(cross, red);
    if (threadIdx.x == 0) {
      float loss = 0.0f;
      if (some) loss = (1.0f - p.alpha) * p.temperature * p.temperature * (cross - logf(st) + logf(s));
      if (known) loss += p.alpha * (logf(s1) + m - Cvt<T>::to_f(z[label]));
      p.loss[row] = loss;
    }
    if (!p.dz) continue;
    T* dz = static_cast<T*>(p.dz) + row * p.lddz;
    const float c = some ? soft_w / s : 0.0f, c1 = known ? p.alpha / s1 : 0.0f;
    auto base = [&](float zi) {
      const float d = zi - m;
      float g = 0.0f;
      if (some) g = expf(d * invT) * c;
      if (known) g += expf(d) * c1;
      return g;
    };
    // the corrections first: the entries' own values are read before dz, which may be z, is written
    constexpr int kPer = (kMaxTop + 1 + 255) / 256;
    float fix[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int k = threadIdx.x + u * 256;
      fix[u] = 0.0f;
      if (k > p.K || col_s[k] < 0) continue;
      float w = 0.0f;
      bool first = true;
      for (int j = 0; j <= p.K; ++j)
        if (col_s[j] == col_s[k]) {
          if (j < k) first = false;
          w += w_s[j];
        }
      fix[u] = base(Cvt<T>::to_f(z[col_s[k]])) - w;
    }
    __syncthreads();
    for (int64_t i = threadIdx.x; i < p.C; i += blockDim.x) dz[i] = Cvt<T>::from_f(p.scale * base(Cvt<T>::to_f(z[i])));
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int k = threadIdx.x + u * 256;
      if (k <= p.K && col_s[k] >= 0) dz[col_s[k]] = Cvt<T>::from_f(p.scale * fix[u]);  // equal columns get equal values
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ one read, one write
// Exponentials are taken in powers of two: with c = log2(e) / T and n = max(z) c, rounded to fp32, softmax(z / T) is
// 2^(z c - n) / S, S the sum of the numerators. z c - n is one fused multiply-add, so n is an exact reference and a logit
// costs three instructions. (Rows whose maximum is a mask's lowest value: see far_off.) The three kinds of row differ in who holds it:
//
//   distill_warp_kernel    up to 2048 columns: one warp per row, the row in its registers, many short blocks
//   distill_block_kernel   longer rows: one CTA, or one per slice of the row in a cluster, the slice in shared memory; two or
//                          three CTAs per SM in different phases keep loads, exponentials and stores going side by side
//   distill_multipass_kernel  z and dz misaligned against each other, or a row past eight slices
//
// Measured: 65536 x 1000 bf16, T = 2 with labels, 82 us (3.2 TB/s; instruction issue bounds it), f32 without labels 106 us (4.9);
// 8192 x 32000 f32 in two slices 375 us (5.6 TB/s); 4096 x 100003 bf16, T = 1.5 with labels, 545 us (two exponentials per logit and
// pass are 365 us by themselves), without labels 377 us (4.3).
//
// A row may start anywhere: the whole 16-byte packets inside it are handled as packets, the up to 2 * (kN - 1) elements
// before and after them one per thread.
__device__ int g_distill_status = 0;

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// How the exponentials of the two softmaxes come about.
enum ExpMode : int {
  kOneExp = 0,    // no label term, or T = 1: one exponential serves both
  kSquares = 1,   // T = 2 or 4: exp(x) is exp(x / T) squared once or twice
  kTwoExps = 2,   // any other T
};

// n is off by up to half a step of its own size, and a logit of -1e30, the lowest value of its type above all, makes it too
// large for that (or infinite) although the differences inside the row are small. Where |n| >= 2^31 (squared exponentials:
// 2^29), neighbouring fp32 values near the maximum are 128 (32) apart in the exponent, so every logit below it weighs nothing
// (2^-32 at most) and every logit equal to it 1: any power of two of at least c says that without a rounding. 1 is one where
// the maximum is 2^40 or more, and the power above c stays in range otherwise (T is held to [2^-60, 2^60]).
template <int kMode>
__device__ __forceinline__ bool far_off(float n) { return !(fabsf(n) < (kMode == kSquares ? 0x1p29f : 0x1p31f)); }
template <int kMode>
__device__ __forceinline__ float factor_of(float ref, float c) {
  if (!far_off<kMode>(__fmul_rn(ref, c))) return c;
  return fabsf(ref) >= 0x1p40f ? 1.0f : __uint_as_float((__float_as_uint(c) & 0x7F800000u) + 0x00800000u);
}

// What a row's softmaxes come down to, in every thread.
struct RowStats {
  float ref;        // the maximum the exponentials refer to
  float c, n, S;    // factor, reference and sum at temperature T
  float c1, n1, S1; // at 1 (where squared, the sum's reference is T n)
  float ct, nt, St; // teacher
  bool some, known; // has a target, has a label
  float kT, k1;     // factors of the two numerators in the gradient
};

// Pairs of fp32 values: one instruction for two, which is what the 16-bit rows need (they are bound by issue).
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split(uint64_t v) {
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
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t ex2_pair(uint64_t v) {
  const float2 u = split(v);
  return pair(ex2(u.x), ex2(u.y));
}
// Exponentials of one row: log2(e) / T for the distillation term, log2(e) for the label term.
template <int kMode>
struct Exps {
  float cT;
  int squarings;
  __device__ __forceinline__ void refer(float m, RowStats& r) const {
    r.ref = m == -INFINITY ? 0.0f : m;
    r.c = factor_of<kMode>(r.ref, cT);
    r.n = __fmul_rn(r.ref, r.c);
    if constexpr (kMode == kOneExp) {
      r.c1 = r.c, r.n1 = r.n;
    } else {
      r.c1 = factor_of<kTwoExps>(r.ref, kLog2e);
      r.n1 = __fmul_rn(r.ref, r.c1);
    }
  }
  // what a sum with maximum `a` counts for in one with maximum m
  __device__ __forceinline__ float weight(float a, float m, float c) const {
    const float na = __fmul_rn(a, c), nm = __fmul_rn(m, c);
    if (a == m) return 1.0f;
    if (far_off<kMode>(nm)) return 0.0f;
    return ex2(far_off<kMode>(na) ? fmaf(a, c, -nm) : na - nm);
  }
  // the same for the sum at 1: squared sums refer to T n, so their weights are the others' squared
  __device__ __forceinline__ float weight1(float a, float m) const {
    if constexpr (kMode == kSquares) {
      const float w = weight(a, m, cT), w2 = w * w;
      return squarings == 2 ? w2 * w2 : w2;
    }
    return weight(a, m, kLog2e);
  }
  __device__ __forceinline__ uint64_t numerators1(uint64_t v, uint64_t e, const RowStats& r) const {
    if constexpr (kMode == kSquares) {
      const uint64_t e2 = mul2(e, e);
      return squarings == 2 ? mul2(e2, e2) : e2;
    }
    if constexpr (kMode == kTwoExps) return ex2_pair(fma2(v, pair(r.c1, r.c1), pair(-r.n1, -r.n1)));
    return e;
  }
  __device__ __forceinline__ void add(uint64_t v, const RowStats& r, uint64_t& s, uint64_t& s1) const {
    const uint64_t e = ex2_pair(fma2(v, pair(r.c, r.c), pair(-r.n, -r.n)));
    s = add2(s, e);
    if constexpr (kMode != kOneExp) s1 = add2(s1, numerators1(v, e, r));
  }
  __device__ __forceinline__ uint64_t grad(uint64_t v, const RowStats& r) const {
    const uint64_t e = ex2_pair(fma2(v, pair(r.c, r.c), pair(-r.n, -r.n)));
    if constexpr (kMode == kOneExp) return mul2(e, pair(r.kT, r.kT));  // kT holds both factors
    if constexpr (kMode == kSquares) {
      if (squarings == 1) return mul2(e, fma2(e, pair(r.k1, r.k1), pair(r.kT, r.kT)));
    }
    return fma2(numerators1(v, e, r), pair(r.k1, r.k1), mul2(e, pair(r.kT, r.kT)));
  }
  __device__ __forceinline__ float grad1(float v, const RowStats& r) const { return split(grad(pair(v, v), r)).x; }
};

// A packet's values as pairs, and back.
template <typename T>
__device__ __forceinline__ void unpack_pairs(const Pack16<T>& p, uint64_t (&v)[Pack16<T>::kN / 2]) {
  float f[Pack16<T>::kN];
  unpack16(p, f);
#pragma unroll
  for (int i = 0; i < Pack16<T>::kN / 2; ++i) v[i] = pair(f[2 * i], f[2 * i + 1]);
}
template <typename T>
__device__ __forceinline__ Pack16<T> pack_pairs(const uint64_t (&v)[Pack16<T>::kN / 2]) {
  float f[Pack16<T>::kN];
#pragma unroll
  for (int i = 0; i < Pack16<T>::kN / 2; ++i) {
    const float2 t = split(v[i]);
    f[2 * i] = t.x, f[2 * i + 1] = t.y;
  }
  Pack16<T> o;
  pack16(o, f);
  return o;
}
template <typename T>
__device__ __forceinline__ Pack16<T> zero_packet() {
  Pack16<T> o;
  *reinterpret_cast<int4*>(&o) = make_int4(0, 0, 0, 0);
  return o;
}

__device__ __forceinline__ float quotient(float a, float b) { return __fdividef(a, b); }  // 2 ulp for b < 2^126; the sums are

// From the sums to the factors of the numerators in the gradient.
template <int kMode>
__device__ __forceinline__ void finish_stats(const DistillParams& p, bool known, RowStats& r) {
  if (r.S == 0.0f) r.S = r.S1 = __int_as_float(0x7fc00000);  // a row of -inf has no softmax
  r.some = !(r.St == 0.0f);  // else no entries, or every entry has weight zero
  r.known = known;
  r.kT = r.some ? quotient(p.grad_soft, r.S) : 0.0f;
  r.k1 = known ? quotient(p.grad_hard, r.S1) : 0.0f;
  if (kMode == kOneExp) r.kT += r.k1;
}
// The teacher's reference: its largest logit as it stands, and what follows from it.
__device__ __forceinline__ void refer_teacher(const DistillParams& p, float mt, RowStats& r) {
  const float ref = mt == -INFINITY ? 0.0f : mt;
  r.ct = factor_of<kOneExp>(ref, p.cT);
  r.nt = __fmul_rn(ref, r.ct);
}
__device__ __forceinline__ float teacher_weight(const RowStats& r, float t) { return ex2(fmaf(t, r.ct, -r.nt)); }
// p_k
__device__ __forceinline__ float target(const RowStats& r, float t) { return r.some ? quotient(teacher_weight(r, t), r.St) : 0.0f; }
constexpr float kLn2 = 0.6931471805599453f;
// log q (at temperature 1 / inv) of a logit, without the sum's logarithm: by the factors of the row's exponentials, or, where
// these do not hold a difference as large, from the logits themselves
__device__ __forceinline__ float log_numerator(float zv, float ref, float c, float n, bool far, float inv) {
  const float l = kLn2 * fmaf(zv, c, -n);
  return l > -0x1p30f && !far ? l : (zv - ref) * inv;
}
// p_k (log p_k - log q_k) without the sums' logarithms
template <int kMode>
__device__ __forceinline__ float cross_term(const DistillParams& p, const RowStats& r, float t, float zv) {
  const float pk = target(r, t);
  return pk != 0.0f ? pk * (kLn2 * fmaf(t, r.ct, -r.nt) - log_numerator(zv, r.ref, r.c, r.n, far_off<kMode>(r.n), p.invT)) : 0.0f;
}
// The loss is what the sums contribute plus what the list's (`cross`: the sum of cross_term) and the label's logits do.
__device__ __forceinline__ float loss_of_sums(const DistillParams& p, const RowStats& r) {
  float loss = 0.0f;
  if (r.some) loss = p.loss_soft * logf(quotient(r.S, r.St));
  if (r.known) loss += p.alpha * logf(r.S1);
  return loss;
}
__device__ __forceinline__ float loss_of_list(const DistillParams& p, float cross) { return p.loss_soft * cross; }
template <int kMode>
__device__ __forceinline__ float loss_of_label(const DistillParams& p, const RowStats& r, float z_label) {
  return -p.alpha * log_numerator(z_label, r.ref, r.c1, r.n1, kMode == kSquares ? far_off<kMode>(r.n) : far_off<kMode>(r.n1), 1.0f);
}
__device__ __forceinline__ float max_of(const Pack16<float>& v) { return fmaxf(fmaxf(v.v[0], v.v[1]), fmaxf(v.v[2], v.v[3])); }
__device__ __forceinline__ float max_of(const Pack16<__nv_bfloat16>& v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__bfloat162float(m.x), __bfloat162float(m.y));
}
__device__ __forceinline__ float max_of(const Pack16<__half>& v) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
  const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__half2float(m.x), __half2float(m.y));
}
template <typename T>
__device__ __forceinline__ int head_elements(const T* row, int64_t C) {
  const int h = static_cast<int>(((16u - (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row)) & 15u)) & 15u) / sizeof(T));
  return h < C ? h : static_cast<int>(C);
}

struct RowPlan {
  int mode = 0, squarings = 0;
  int packets = 0;   // warp kernel: packets per lane; 0 = block kernel
  int threads = 0;   // block kernel
  int ranks = 1;     // CTAs of a cluster per row
  int slice = 0;     // packets per CTA (warp kernel: per row)
  size_t smem = 0;
};

constexpr int kRowsPerBlock = 8;

// One warp per row. kOneEach: the list with its label has at most 32 entries, one per lane and in registers; longer lists are
// staged in shared memory next to a bit per column that finds repeated columns.
template <typename T, int kPk, int kMode, bool kOneEach>
__global__ void __launch_bounds__(32 * kRowsPerBlock, kPk * Pack16<T>::kN <= 32 ? 4 : 2) distill_warp_kernel(const DistillParams p, const RowPlan g) {
  using PK = Pack16<T>;
  constexpr int kN = PK::kN;
  extern __shared__ __align__(16) uint8_t dsmem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int entries = p.K + 1;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRowsPerBlock + warp;
  if (row >= p.B) return;  // whole warps: nothing below meets another warp
  const bool hard = p.labels != nullptr && p.alpha > 0.0f;
  const Exps<kMode> x{p.cT, g.squarings};
  const T* z = static_cast<const T*>(p.z) + row * p.ldz;
  const int C = static_cast<int>(p.C);
  const int head = head_elements(z, p.C);
  const int pn = (C - head) / kN, tail0 = head + pn * kN;
  const int edges = head + C - tail0;
  const PK* packets = reinterpret_cast<const PK*>(z + head) + lane;
  PK raw[kPk];
#pragma unroll
  for (int q = 0; q < kPk; ++q)
    if (lane + 32 * q < pn) raw[q] = ld_stream(packets + 32 * q);
  // entry k of the row's list, or its label (k = K): column or -1, teacher logit, own logit
  auto load_entry = [&](int k, int* col, float* t, float* zv) {
    const int id = k < p.K ? __ldg(p.ids + row * p.K + k) : hard && k == p.K ? __ldg(p.labels + row) : -1;
    *t = k < p.K ? teacher_at(p, row * p.K + k) : 0.0f;
    *col = id >= 0 && id < C ? id : -1;
    *zv = *col >= 0 ? Cvt<T>::to_f(z[id]) : 0.0f;
  };
  int my_col = -1;
  float my_t = 0.0f, my_z = 0.0f;
  if (lane < entries) load_entry(lane, &my_col, &my_t, &my_z);
  int edge_col = -1;
  float fe = -INFINITY;
  if (edges > 0 && lane < edges) {
    edge_col = lane < head ? lane : tail0 + lane - head;
    fe = Cvt<T>::to_f(z[edge_col]);
  }
  const int words = (C + 31) / 32;
  uint32_t* bits_s = reinterpret_cast<uint32_t*>(dsmem) + warp * (words + 3 * entries);
  int* col_s = reinterpret_cast<int*>(bits_s + words);
  float* t_s = reinterpret_cast<float*>(col_s + entries);
  float* z_s = t_s + entries;
  RowStats r;
  bool twice = false;
  bool known;
  {
    float mt = my_col >= 0 && lane < p.K ? my_t : -INFINITY;
    if constexpr (kOneEach) {
      refer_teacher(p, warp_max(mt), r);
      r.St = warp_sum(my_col >= 0 && lane < p.K ? teacher_weight(r, my_t) : 0.0f);
      known = __shfl_sync(0xffffffffu, my_col, p.K) >= 0;
    } else {
      for (int i = lane; i < words; i += 32) bits_s[i] = 0u;
      __syncwarp();
      for (int k = lane; k < entries; k += 32) {
        if (k != lane) load_entry(k, &my_col, &my_t, &my_z);
        col_s[k] = my_col, t_s[k] = my_t, z_s[k] = my_z;
        if (my_col < 0) continue;
        if (k < p.K) mt = fmaxf(mt, my_t);
        if (p.dz && (atomicOr(bits_s + (my_col >> 5), 1u << (my_col & 31)) & (1u << (my_col & 31)))) twice = true;
      }
      refer_teacher(p, warp_max(mt), r);
      __syncwarp();
      float st = 0.0f;
      for (int k = lane; k < p.K; k += 32)
        if (col_s[k] >= 0) st += teacher_weight(r, t_s[k]);
      r.St = warp_sum(st);
      known = col_s[p.K] >= 0;
    }
  }
  float m = fe;
#pragma unroll
  for (int q = 0; q < kPk; ++q)
    if (lane + 32 * q < pn) m = fmaxf(m, max_of(raw[q]));
  m = warp_max(m);
  x.refer(m, r);
  uint64_t s2 = pair(0.0f, 0.0f), s12 = s2;
  if (edges > 0) x.add(pair(fe, -INFINITY), r, s2, s12);  // lanes without an edge element add zeros
#pragma unroll
  for (int q = 0; q < kPk; ++q)
    if (lane + 32 * q < pn) {
      uint64_t v[kN / 2];
      unpack_pairs<T>(raw[q], v);
#pragma unroll
      for (int e = 0; e < kN / 2; ++e) x.add(v[e], r, s2, s12);
    }
  {
    const float2 a = split(s2), b = split(s12);
    r.S = warp_sum(a.x + a.y);
    r.S1 = kMode == kOneExp ? r.S : warp_sum(b.x + b.y);
  }
  finish_stats<kMode>(p, known, r);
  float own = 0.0f;
  if (r.some) {
    if constexpr (kOneEach) {
      own = my_col >= 0 && lane < p.K ? cross_term<kMode>(p, r, my_t, my_z) : 0.0f;
    } else {
      for (int k = lane; k < p.K; k += 32)
        if (col_s[k] >= 0) own += cross_term<kMode>(p, r, t_s[k], z_s[k]);
    }
    own = loss_of_list(p, warp_sum(own));
  }
  if (known) {
    if constexpr (kOneEach) own += loss_of_label<kMode>(p, r, __shfl_sync(0xffffffffu, my_z, p.K));
    else own += loss_of_label<kMode>(p, r, z_s[p.K]);
  }
  if (lane == 0) p.loss[row] = loss_of_sums(p, r) + own;
  if (!p.dz) return;
  T* out = static_cast<T*>(p.dz) + row * p.lddz;
  PK* out_packets = reinterpret_cast<PK*>(out + head) + lane;
  if (!r.some && !known) {  // neither term: zeros, whatever the logits hold
#pragma unroll
    for (int q = 0; q < kPk; ++q)
      if (lane + 32 * q < pn) st_stream(out_packets + 32 * q, zero_packet<T>());
    if (edge_col >= 0) out[edge_col] = Cvt<T>::from_f(0.0f);
    return;
  }
#pragma unroll
  for (int q = 0; q < kPk; ++q)
    if (lane + 32 * q < pn) {
      uint64_t v[kN / 2];
      unpack_pairs<T>(raw[q], v);
#pragma unroll
      for (int e = 0; e < kN / 2; ++e) v[e] = x.grad(v[e], r);
      st_stream(out_packets + 32 * q, pack_pairs<T>(v));
    }
  if (edge_col >= 0) out[edge_col] = Cvt<T>::from_f(x.grad1(fe, r));
  // The corrections come behind the row: other lanes, the same addresses. Equal columns are corrected once, by their first
  // entry, for the sum of their weights in the list's order.
  if constexpr (kOneEach) {
    float w = lane == p.K ? p.grad_hard : p.grad_soft * target(r, my_t);
    bool first = my_col >= 0;
    const uint32_t same = __match_any_sync(0xffffffffu, first ? my_col : -1 - lane);
    if (__any_sync(0xffffffffu, (same & (same - 1)) != 0u)) {
      const float mine = w;
      w = 0.0f;
      for (int j = 0; j < entries; ++j) {
        const float other = __shfl_sync(0xffffffffu, mine, j);
        if ((same >> j) & 1u) w += other;
      }
      first = first && lane == __ffs(static_cast<int>(same)) - 1;
    }
    __syncwarp();
    if (first) out[my_col] = Cvt<T>::from_f(x.grad1(my_z, r) - w);
  } else {
    const bool dup = __any_sync(0xffffffffu, twice);
    __syncwarp();
    for (int k = lane; k < entries; k += 32) {
      const int col = col_s[k];
      if (col < 0) continue;
      float w = 0.0f;
      bool first = true;
      auto weight = [&](int j) { return j == p.K ? p.grad_hard : p.grad_soft * target(r, t_s[j]); };
      if (dup) {
        for (int j = 0; j < entries; ++j)
          if (col_s[j] == col) {
            if (j < k) first = false;
            w += weight(j);
          }
      } else {
        w = weight(k);
      }
      if (first) out[col] = Cvt<T>::from_f(x.grad1(z_s[k], r) - w);
    }
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_index() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_count() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%nclusterid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_peer_shared(const float* local, uint32_t rank, float v) {
  const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(local));
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(mine), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
}

constexpr int kRowThreads = 256;   // threads that work on the row; one more warp has the list
constexpr int kMaxRanks = 8;
constexpr int kRowCtas = 3;         // CTAs per SM that its registers allow: while one waits for its row, the others work

template <typename T, int kMode>
__global__ void __launch_bounds__(kRowThreads + 32, kRowCtas) distill_block_kernel(const DistillParams p, const RowPlan g) {
  using PK = Pack16<T>;
  constexpr int kN = PK::kN;
  extern __shared__ __align__(16) uint8_t dsmem[];
  // [slice][mbarrier 16 B][a bit per column][entries: column, teacher logit, own logit]
  const int words = (g.slice * kN + 2 * kN + 31) / 32;
  const int entries = p.K + 1;
  const PK* row_s = reinterpret_cast<const PK*>(dsmem);
  uint32_t* bits = reinterpret_cast<uint32_t*>(dsmem + static_cast<size_t>(g.slice) * 16 + 16);
  int* col_s = reinterpret_cast<int*>(bits + words);
  float* t_s = reinterpret_cast<float*>(col_s + entries);
  float* z_s = t_s + entries;
  __shared__ float red[2][3][kRowThreads / 32];
  __shared__ float teach[2][4];            // the teacher's factor, reference and sum; whether the row has a label
  __shared__ float peer[2][kMaxRanks][4];  // per CTA of the cluster: maximum, two sums, and its part of the loss
  __shared__ int wait_failed;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int nthreads = blockDim.x - 32, nwarps = nthreads >> 5;  // those that work on the row
  const bool list_warp = warp == nwarps;  // stages the row's list, sums the teacher, corrects the listed columns
  const uint32_t rank = g.ranks > 1 ? cluster_rank() : 0;
  const int64_t first_row = g.ranks > 1 ? cluster_index() : blockIdx.x, row_step = g.ranks > 1 ? cluster_count() : gridDim.x;
  const uint32_t buf = sm100::smem_addr(dsmem), bar = buf + static_cast<uint32_t>(g.slice) * 16;
  const bool hard = p.labels != nullptr && p.alpha > 0.0f;
  const Exps<kMode> x{p.cT, g.squarings};
  const int p0 = static_cast<int>(rank) * g.slice;
  const int C = static_cast<int>(p.C);

  auto packets_of = [&](int head) {
    const int n = (C - head) / kN - p0;
    return n < 0 ? 0 : n < g.slice ? n : g.slice;
  };
  auto fetch = [&](int64_t row) {  // thread 0
    const T* z = static_cast<const T*>(p.z) + row * p.ldz;
    const int head = head_elements(z, p.C), n = packets_of(head);
    if (n > 0) {
      sm100::mbar_expect_tx(bar, static_cast<uint32_t>(n) * 16);
      sm100::bulk_copy_g2s(buf, z + head + static_cast<int64_t>(p0) * kN, static_cast<uint32_t>(n) * 16, bar);
    }
  };
  // What threads read of a row from global memory themselves is asked for one row ahead: the list warp's first kAhead
  // entries per lane, and (warp 0 of rank 0) the elements outside the packets.
  constexpr int kAhead = 2;
  auto list_id = [&](int64_t row, int k) { return k < p.K ? __ldg(p.ids + row * p.K + k) : hard && k == p.K ? __ldg(p.labels + row) : -1; };
  auto list_t = [&](int64_t row, int k) { return k < p.K ? teacher_at(p, row * p.K + k) : 0.0f; };
  int ahead_id[kAhead];
  float ahead_t[kAhead], ahead_edge = -INFINITY;
  auto edge_of = [&](int64_t row) {
    const int head = head_elements(static_cast<const T*>(p.z) + row * p.ldz, p.C), tail0 = head + (C - head) / kN * kN;
    return tid < head + C - tail0 ? (tid < head ? tid : tail0 + tid - head) : -1;
  };
  auto look_ahead = [&](int64_t row) {
    if (list_warp) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) ahead_id[i] = list_id(row, lane + 32 * i), ahead_t[i] = list_t(row, lane + 32 * i);
    }
    if (warp == 0 && rank == 0) {
      const int col = edge_of(row);
      ahead_edge = col >= 0 ? Cvt<T>::to_f(static_cast<const T*>(p.z)[row * p.ldz + col]) : -INFINITY;
    }
  };

  if (tid == 0) {
    sm100::mbar_init(bar, 1);
    sm100::mbar_init_fence();
    wait_failed = 0;
  }
  for (int i = tid; i < words; i += blockDim.x) bits[i] = 0u;
  __syncthreads();
  if (first_row < p.B) {
    if (tid == 0) fetch(first_row);
    look_ahead(first_row);
  }
  bool piped = true;  // false once a copy did not arrive: the remaining rows run on what the buffer holds
  uint32_t phase = 0;
  int par = 0;
  int64_t owed = -1;  // cluster: the row whose loss waits for the other CTAs' parts
  float owed_base = 0.0f;
  for (int64_t row = first_row; row < p.B; row += row_step, par ^= 1) {
    const T* z = static_cast<const T*>(p.z) + row * p.ldz;
    const int head = head_elements(z, p.C), pn = packets_of(head);
    const int tail0 = head + (C - head) / kN * kN;
    const int edge_col = warp == 0 && rank == 0 ? edge_of(row) : -1;
    const float fe = ahead_edge;
    bool twice = false;  // list warp: some column occurs more than once
    // the place of a column among this CTA's elements, -1 for another CTA's column
    auto place = [&](int col) {
      if (col < 0) return -1;
      if (col < head) return rank == 0 ? g.slice * kN + col : -1;
      if (col >= tail0) return rank == 0 ? g.slice * kN + kN + col - tail0 : -1;
      const int at = col - head - p0 * kN;
      return at >= 0 && at < pn * kN ? at : -1;
    };
    if (list_warp) {
      // The row's list: every CTA of a cluster has all of it, sums the teacher's weights and marks its own columns.
      float mt = -INFINITY;
      auto stage = [&](int k, int id, float t) {
        const int col = id >= 0 && id < C ? id : -1, at = place(col);
        col_s[k] = col, t_s[k] = t;
        if (col >= 0 && k < p.K) mt = fmaxf(mt, t);
        if (p.dz && at >= 0 && (atomicOr(bits + (at >> 5), 1u << (at & 31)) & (1u << (at & 31)))) twice = true;
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (lane + 32 * i < entries) stage(lane + 32 * i, ahead_id[i], ahead_t[i]);
      for (int k = lane + 32 * kAhead; k < entries; k += 32) stage(k, list_id(row, k), list_t(row, k));
      RowStats rt;
      refer_teacher(p, warp_max(mt), rt);
      __syncwarp();
      float st = 0.0f;
      for (int k = lane; k < p.K; k += 32)
        if (col_s[k] >= 0) st += teacher_weight(rt, t_s[k]);
      st = warp_sum(st);
      if (lane == 0) teach[par][0] = rt.ct, teach[par][1] = rt.nt, teach[par][2] = st, teach[par][3] = col_s[p.K] >= 0 ? 1.0f : 0.0f;
    }
    if (pn > 0 && piped) {
      if (!sm100::mbar_wait_bounded(bar, phase, rowk::kRowWaitBudgetNs)) wait_failed = 1;
      phase ^= 1u;
    }
    float m = edge_col >= 0 ? fe : -INFINITY;
    RowStats r;
    if (!list_warp) {
      // Maximum first: its pass takes three instructions for eight 16-bit logits.
#pragma unroll 4
      for (int pi = tid; pi < pn; pi += nthreads) m = fmaxf(m, max_of(row_s[pi]));
      m = warp_max(m);
      x.refer(m, r);
      uint64_t s2 = pair(0.0f, 0.0f), s12 = s2;
      if (warp == 0 && rank == 0) x.add(pair(edge_col >= 0 ? fe : -INFINITY, -INFINITY), r, s2, s12);
#pragma unroll 4
      for (int pi = tid; pi < pn; pi += nthreads) {
        uint64_t f[kN / 2];
        unpack_pairs<T>(row_s[pi], f);
#pragma unroll
        for (int e = 0; e < kN / 2; ++e) x.add(f[e], r, s2, s12);
      }
      const float2 a = split(s2), b = split(s12);
      const float s = warp_sum(a.x + a.y), s1 = kMode == kOneExp ? 0.0f : warp_sum(b.x + b.y);
      if (lane == 0) red[par][0][warp] = m, red[par][1][warp] = s, red[par][2][warp] = s1;
    } else {  // the list's own logits, of this CTA's columns
      for (int k = lane; k < entries; k += 32) {
        const int col = col_s[k], at = place(col);
        if (at >= 0) z_s[k] = at < g.slice * kN ? Cvt<T>::to_f(reinterpret_cast<const T*>(dsmem)[at]) : Cvt<T>::to_f(z[col]);
      }
    }
    __syncthreads();
    {
      // every warp folds the warps' parts for itself, in the same order
      const bool in = lane < nwarps;
      const float a = in ? red[par][0][lane] : -INFINITY;
      m = warp_max(a);
      r.S = warp_sum(in ? red[par][1][lane] * x.weight(a, m, p.cT) : 0.0f);
      r.S1 = kMode == kOneExp ? r.S : warp_sum(in ? red[par][2][lane] * x.weight1(a, m) : 0.0f);
      r.ct = teach[par][0], r.nt = teach[par][1], r.St = teach[par][2];
    }
    if (g.ranks > 1) {
      if (warp == 0 && lane < g.ranks) {
        st_peer_shared(&peer[par][rank][0], lane, m);
        st_peer_shared(&peer[par][rank][1], lane, r.S);
        st_peer_shared(&peer[par][rank][2], lane, r.S1);
      }
      __syncwarp();
      cluster_barrier();  // the other parity's slots are rewritten behind this row's barrier only
      float a = -INFINITY;
      for (int k = 0; k < g.ranks; ++k) a = fmaxf(a, peer[par][k][0]);
      r.S = r.S1 = 0.0f;
      for (int k = 0; k < g.ranks; ++k) {
        const float pm = peer[par][k][0];
        r.S += peer[par][k][1] * x.weight(pm, a, p.cT);
        r.S1 += peer[par][k][2] * x.weight1(pm, a);
      }
      m = a;
      if constexpr (kMode == kOneExp) r.S1 = r.S;
      if (rank == 0 && tid == 0 && owed >= 0) {  // the parts of the row before have arrived behind this barrier
        for (int k = 0; k < g.ranks; ++k) owed_base += peer[par ^ 1][k][3];
        p.loss[owed] = owed_base;
      }
    }
    x.refer(m, r);
    finish_stats<kMode>(p, teach[par][3] != 0.0f, r);
    const bool dead = !r.some && !r.known;
    T* out = static_cast<T*>(p.dz) + row * p.lddz;
    if (p.dz && !list_warp) {
      PK* packets = reinterpret_cast<PK*>(out + head) + p0;
      if (dead) {  // neither term: zeros, whatever the logits hold
        for (int pi = tid; pi < pn; pi += nthreads) st_stream(packets + pi, zero_packet<T>());
      } else {
#pragma unroll 4
        for (int pi = tid; pi < pn; pi += nthreads) {
          uint64_t f[kN / 2];
          unpack_pairs<T>(row_s[pi], f);
#pragma unroll
          for (int e = 0; e < kN / 2; ++e) f[e] = x.grad(f[e], r);
          st_stream(packets + pi, pack_pairs<T>(f));
        }
      }
      if (edge_col >= 0) out[edge_col] = Cvt<T>::from_f(dead ? 0.0f : x.grad1(fe, r));
    }
    __syncthreads();  // the buffer is free; the corrections below come behind the row's stores
    if (wait_failed) piped = false;
    const int64_t next = row + row_step;
    if (next < p.B) {
      if (tid == 0 && piped) {
        sm100::fence_generic_to_async_smem();
        fetch(next);
      }
      look_ahead(next);
    }
    if (rank == 0 && tid == 0 && g.ranks > 1) owed = row, owed_base = loss_of_sums(p, r);
    if (list_warp) {
      // this CTA's part of the loss, and the corrections of its columns: equal columns are corrected once, by their first
      // entry, for the sum of their weights in the list's order
      const bool dup = __any_sync(0xffffffffu, twice);
      auto weight = [&](int j) { return j == p.K ? p.grad_hard : p.grad_soft * target(r, t_s[j]); };
      float own = 0.0f;
      for (int k = lane; k < entries; k += 32) {
        const int col = col_s[k], at = place(col);
        if (at < 0) continue;
        if (k < p.K && r.some) own += cross_term<kMode>(p, r, t_s[k], z_s[k]);
        if (!p.dz) continue;
        bits[at >> 5] = 0u;  // this row's marks go
        float w = 0.0f;
        bool first = !dead;
        if (dup) {
          for (int j = 0; j < entries; ++j)
            if (col_s[j] == col) {
              if (j < k) first = false;
              w += weight(j);
            }
        } else {
          w = weight(k);
        }
        if (first) out[col] = Cvt<T>::from_f(x.grad1(z_s[k], r) - w);
      }
      own = loss_of_list(p, warp_sum(own));
      if (lane == 0) {
        if (r.known && place(col_s[p.K]) >= 0) own += loss_of_label<kMode>(p, r, z_s[p.K]);
        if (g.ranks > 1) st_peer_shared(&peer[par][rank][3], 0, own);
        else p.loss[row] = loss_of_sums(p, r) + own;
      }
      __syncwarp();  // the list is the next row's from here on
    }
  }
  if (g.ranks > 1) {
    cluster_barrier();  // nobody leaves while a peer may still write its shared memory
    if (rank == 0 && tid == 0 && owed >= 0) {
      for (int k = 0; k < g.ranks; ++k) owed_base += peer[par ^ 1][k][3];
      p.loss[owed] = owed_base;
    }
  }
  if (wait_failed) {
    if (tid == 0) atomicExch(&g_distill_status, 1);
    for (int i = 0; i < 64; ++i) __nanosleep(16384);  // error path only: let a late copy land
  }
}

template <typename T>
bool plan_rows(const DistillParams& p, RowPlan* out) {
  constexpr int kN = Pack16<T>::kN;
  RowPlan g;
  if (!aligned_to(p.z, sizeof(T)) || (p.dz && !aligned_to(p.dz, sizeof(T)))) return false;
  if (p.dz) {  // packets of z and dz have to start at the same places in every row
    const uintptr_t a = reinterpret_cast<uintptr_t>(p.z), b = reinterpret_cast<uintptr_t>(p.dz);
    if (((a ^ b) & 15) != 0 || ((p.ldz - p.lddz) * static_cast<int64_t>(sizeof(T))) % 16 != 0) return false;
  }
  const bool hard = p.labels != nullptr && p.alpha > 0.0f;
  g.mode = !hard || p.temperature == 1.0f ? kOneExp : p.temperature == 2.0f || p.temperature == 4.0f ? kSquares : kTwoExps;
  g.squarings = p.temperature == 4.0f ? 2 : 1;
  const int64_t packets = p.C / kN > 0 ? p.C / kN : 1;
  const size_t list = static_cast<size_t>(p.K + 1) * 12;
  if (p.C <= 2048) {
    const int per = static_cast<int>((packets + 31) / 32);
    g.packets = 1;
    while (g.packets < per) g.packets *= 2;
    g.slice = static_cast<int>(packets);
    g.smem = p.K < 32 ? 0 : kRowsPerBlock * (static_cast<size_t>((p.C + 31) / 32) * 4 + list);
    *out = g;
    return true;
  }
  auto bytes = [&](int64_t slice) {
    return static_cast<size_t>(slice) * 16 + 16 + static_cast<size_t>((slice * kN + 2 * kN + 31) / 32) * 4 + list;
  };
  // The fewest CTAs per row of which an SM still holds two: one alone would leave the SM idle while it waits for its row
  // (8192 x 32000 f32 in 374 us as two slices per row, 528 as one), and every doubling costs a cluster barrier more than it
  // hides (4096 x 100003 bf16: 375 us as two slices, 412 as four; 8192 x 32000 bf16: 203 as one, 303 as two).
  constexpr size_t kShare = (227 * 1024) / 2 - 2048;  // half an SM's shared memory, less the static part
  while (g.ranks < kMaxRanks && bytes((packets + g.ranks - 1) / g.ranks) > kShare) g.ranks *= 2;
  const int64_t slice = (packets + g.ranks - 1) / g.ranks;
  g.smem = bytes(slice);
  if (g.smem > 200 * 1024) return false;
  g.slice = static_cast<int>(slice);
  // Sixteen packets per thread before the block grows: what a thread does per row besides its packets (folding the warps'
  // parts, the factors) costs as much as eight of them (16384 x 8192 bf16: 216 / 166 / 152 us at 4 / 8 / 16).
  g.threads = 32;
  while (g.threads < kRowThreads && static_cast<int64_t>(g.threads) * 16 < slice) g.threads *= 2;
  *out = g;
  return true;
}

template <typename T, int kMode>
Status launch_block_rows(const DistillParams& p, const RowPlan& g, cudaStream_t stream) {
  auto kernel = distill_block_kernel<T, kMode>;
  static PerDeviceOnce opt_in;
  if (!opt_in.run([&] { return rowk::allow_smem(kernel, 200 * 1024); })) {
    cudaGetLastError();
    return Status::Internal;
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(g.ranks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  // registers allow kRowCtas blocks of kRowThreads + 32 threads
  const int threads = g.threads + 32;
  int resident = rowk::row_pipe_blocks_per_sm(threads, g.smem + 1024);
  if (resident > kRowCtas * (kRowThreads + 32) / threads) resident = kRowCtas * (kRowThreads + 32) / threads;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = g.smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = g.ranks > 1 ? 1 : 0;
  int64_t slots = static_cast<int64_t>(sm_count()) * resident / g.ranks;
  if (g.ranks > 1) {
    // Clusters do not fill every SM (a cluster stays inside one group of SMs): a grid larger than what fits at once would
    // run its last clusters as a second wave. Asked of the runtime once per shape.
    static std::mutex mu;
    static std::map<std::array<int64_t, 4>, int> known;
    const std::array<int64_t, 4> key{device_slot(), g.ranks, g.threads, static_cast<int64_t>(g.smem)};
    std::lock_guard<std::mutex> lock(mu);
    auto it = known.find(key);
    if (it == known.end()) {
      cfg.gridDim = dim3(static_cast<unsigned>(sm_count() * resident / g.ranks * g.ranks));
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = static_cast<int>(slots > 0 ? slots : 1);
      }
      if (known.size() > 256) known.clear();
      it = known.emplace(key, n).first;
    }
    if (it->second < slots) slots = it->second;
  }
  const int64_t rows = p.B < slots ? p.B : (slots > 0 ? slots : 1);
  cfg.gridDim = dim3(static_cast<unsigned>(rows * g.ranks));
  if (cudaLaunchKernelEx(&cfg, kernel, p, g) != cudaSuccess) {
    cudaGetLastError();
    return Status::Internal;
  }
  return launch_status();
}
template <typename T, int kPk, int kMode, bool kOneEach>
Status launch_warp_list(const DistillParams& p, const RowPlan& g, cudaStream_t stream) {
  auto kernel = distill_warp_kernel<T, kPk, kMode, kOneEach>;
  static PerDeviceOnce opt_in;
  if (!opt_in.run([&] { return rowk::allow_smem(kernel, 110 * 1024); })) {
    cudaGetLastError();
    return Status::Internal;
  }
  const int64_t blocks = (p.B + kRowsPerBlock - 1) / kRowsPerBlock;
  if (blocks > 0x7fffffff) return Status::InvalidArgument;
  kernel<<<static_cast<unsigned>(blocks), 32 * kRowsPerBlock, g.smem, stream>>>(p, g);
  return launch_status();
}
template <typename T, int kPk, int kMode>
Status launch_warp_rows(const DistillParams& p, const RowPlan& g, cudaStream_t stream) {
  return p.K < 32 ? launch_warp_list<T, kPk, kMode, true>(p, g, stream) : launch_warp_list<T, kPk, kMode, false>(p, g, stream);
}
template <typename T, int kMode>
Status launch_mode(const DistillParams& p, const RowPlan& g, cudaStream_t stream) {
  switch (g.packets) {
    case 0: return launch_block_rows<T, kMode>(p, g, stream);
    case 1: return launch_warp_rows<T, 1, kMode>(p, g, stream);
    case 2: return launch_warp_rows<T, 2, kMode>(p, g, stream);
    case 4: return launch_warp_rows<T, 4, kMode>(p, g, stream);
    case 8: return launch_warp_rows<T, 8, kMode>(p, g, stream);
    default: break;
  }
  if constexpr (sizeof(T) == 4) return launch_warp_rows<T, 16, kMode>(p, g, stream);
  return Status::Internal;
}
template <typename T>
Status run_rows(const DistillParams& p, const RowPlan& g, cudaStream_t stream) {
  if (g.mode == kOneExp) return launch_mode<T, kOneExp>(p, g, stream);
  if (g.mode == kSquares) return launch_mode<T, kSquares>(p, g, stream);
  return launch_mode<T, kTwoExps>(p, g, stream);
}

bool rows_ok(const TensorDesc& t, int64_t B, int64_t C) {
  return t.rank() == 2 && t.shape[0] == B && t.shape[1] == C && (C == 1 || t.stride[1] == 1) && (B == 1 || t.stride[0] >= C);
}

bool distill_check(DType dt, const TensorDesc* in, int ni, const TensorDesc* out, int no, const void* attr, DistillParams* prob) {
  if (!in || !out || (ni != 3 && ni != 4) || (no != 1 && no != 2)) return false;
  const TensorDesc &Z = in[0], &I = in[1], &T = in[2], &L = out[no - 1];
  if (Z.dtype != dt || Z.rank() != 2 || Z.shape[0] <= 0 || Z.shape[1] <= 0 || Z.shape[1] > 0x7fffffff - 64) return false;
  DistillParams p{};
  p.B = Z.shape[0], p.C = Z.shape[1];
  if (!rows_ok(Z, p.B, p.C)) return false;
  if (I.dtype != DType::kI32 || I.rank() != 2 || !I.contiguous || I.shape[0] != p.B || I.shape[1] < 1 || I.shape[1] > kMaxTop) return false;
  if (!dtype_is_float(T.dtype) || T.rank() != 2 || !T.contiguous || !same_shape(T, I)) return false;
  if (L.dtype != DType::kF32 || L.rank() != 1 || !L.contiguous || L.shape[0] != p.B) return false;
  if (no == 2 && (out[0].dtype != dt || !rows_ok(out[0], p.B, p.C))) return false;
  p.scale = 1.0f / static_cast<float>(p.B), p.temperature = 1.0f, p.alpha = 0.0f;
  const AttrBlob& b = blob_of(attr);
  if (b.schema_id != 0 || b.bytes != 0) {
    float v[3];
    if (!read_attr_payload(attr, schema::kDistill, false, v, 12)) return false;
    p.scale = v[0], p.temperature = v[1], p.alpha = v[2];
  }
  if (!(p.temperature >= 0x1p-60f) || !(p.temperature <= 0x1p60f) || !(p.alpha >= 0.0f) || !(p.alpha <= 1.0f)) return false;
  if (ni == 4) {
    const TensorDesc& Y = in[3];
    if (Y.dtype != DType::kI32 || Y.rank() != 1 || !Y.contiguous || Y.shape[0] != p.B) return false;
    p.labels = static_cast<const int32_t*>(Y.data);
  } else if (p.alpha > 0.0f) {
    return false;  // a label term without labels
  }
  p.invT = 1.0f / p.temperature;
  p.cT = kLog2e / p.temperature;
  p.grad_soft = p.scale * (1.0f - p.alpha) * p.temperature;
  p.grad_hard = p.scale * p.alpha;
  p.loss_soft = (1.0f - p.alpha) * p.temperature * p.temperature;
  p.z = Z.data, p.ldz = p.B == 1 ? p.C : Z.stride[0];
  if (no == 2) p.dz = out[0].data, p.lddz = p.B == 1 ? p.C : out[0].stride[0];
  p.ids = static_cast<const int32_t*>(I.data);
  p.t = T.data, p.t_dtype = static_cast<int>(T.dtype), p.K = static_cast<int>(I.shape[1]);
  p.loss = static_cast<float*>(L.data);
  if (prob) *prob = p;
  return true;
}

template <DType kDt>
bool distill_supported(const TensorDesc* in, int ni, const TensorDesc* out, int no, const void* attr) {
  return distill_check(kDt, in, ni, out, no, attr, nullptr);
}
template <DType kDt, typename T>
Status distill_launch(const TensorDesc* in, int ni, TensorDesc* out, int no, const void* attr, void*, size_t, cudaStream_t stream) {
  DistillParams p;
  if (!distill_check(kDt, in, ni, out, no, attr, &p)) return Status::InvalidArgument;
  cudaGetLastError();
  RowPlan plan;
  if (plan_rows<T>(p, &plan)) return run_rows<T>(p, plan, stream);
  distill_multipass_kernel<T><<<streaming_grid(p.B, 1, 8), 256, 0, stream>>>(p);
  return launch_status();
}

size_t no_workspace(const TensorDesc*, int, const void*) { return 0; }
template <DType kDt, typename T>
KernelVariant make(const char* name) {
  KernelVariant v{};
  v.name = name;
  v.flags = kKV_CaptureSafe;
  v.launch = distill_launch<kDt, T>;
  v.supported = distill_supported<kDt>;
  v.query_workspace = no_workspace;
  return v;
}

}  // namespace

// Status word of the row copies' bounded waits: non-zero once one ran out. Synchronises the device.
int distill_pipeline_status(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_distill_status, sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (clear && v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_distill_status, &zero, sizeof(int));
  }
  return v;
}

KernelVariant make_distill_ce_f32_variant() { return make<DType::kF32, float>("distill_ce_f32_sm100"); }
KernelVariant make_distill_ce_bf16_variant() { return make<DType::kBF16, __nv_bfloat16>("distill_ce_bf16_sm100"); }
KernelVariant make_distill_ce_f16_variant() { return make<DType::kF16, __half>("distill_ce_f16_sm100"); }

}  // namespace aicf::cuda
