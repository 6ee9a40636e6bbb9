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
#include <cstdlib>

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
__device__ int g_distill_status = 0;

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
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

constexpr int kRowThreads = 512;
constexpr int kMaxRanks = 8;

// How the exponentials of the two softmaxes come about.
enum ExpMode : int {
  kOneExp = 0,    // no label term, or T = 1: one exponential serves both
  kSquares = 1,   // T = 2 or 4: exp(x) is exp(x / T) squared once or twice
  kTwoExps = 2,   // any other T: the logits stay in registers and both are taken again when the gradient is written
};

struct RowPlan {
  int mode = 0;
  int squarings = 0;
  int threads = 0, packets = 0;  // packets of 16 bytes per thread
  int ranks = 1;                 // CTAs (of a cluster) per row
  int slice = 0;                 // packets per CTA
  size_t smem = 0;
  int early = 0;                 // one CTA per SM: request the next row before any arithmetic
};

// A running maximum and the sum of exponentials below it.
__device__ __forceinline__ float rescale(float m, float to, float c) { return m == to ? 1.0f : ex2((m - to) * c); }

// One row per CTA, or per cluster with a contiguous slice for each CTA. The slice sits in registers; the next row's is
// on its way to shared memory meanwhile. A row may start anywhere: the whole 16-byte packets inside it are copied and kept as
// packets, and the up to 2 * (kN - 1) elements before and after them by one thread each of rank 0.
//
// Each thread takes its exponentials below its own maximum, so a row needs one reduction (and in a cluster one barrier)
// for maximum and sum together; the thread's factor to the row's maximum joins the normalisation.
template <typename T, int kPk, int kMode>
__global__ void __launch_bounds__(kRowThreads) distill_row_kernel(const DistillParams p, const RowPlan g) {
  using PK = Pack16<T>;
  constexpr int kN = PK::kN;
  extern __shared__ __align__(16) uint8_t dsmem[];
  // [slice][mbarrier 16 B][bitmap x 2][entries x 2: column, teacher logit, own logit]
  const int bits_words = (g.slice * kN + 2 * kN + 31) / 32;
  const int entries = p.K + 1;  // the row's list, then its label
  const PK* row_s = reinterpret_cast<const PK*>(dsmem);
  uint32_t* bits_s = reinterpret_cast<uint32_t*>(dsmem + static_cast<size_t>(g.slice) * 16 + 16);
  int* col_s = reinterpret_cast<int*>(bits_s + 2 * bits_words);
  float* t_s = reinterpret_cast<float*>(col_s + 2 * entries);
  float* z_s = t_s + 2 * entries;
  __shared__ float red[2][5][kRowThreads / 32];
  __shared__ float peer[2][kMaxRanks][3];
  __shared__ int twice[2];    // some column occurs more than once
  __shared__ int wait_failed;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nthreads = blockDim.x, nwarps = nthreads >> 5;
  const uint32_t nranks = g.ranks > 1 ? cluster_size() : 1, rank = g.ranks > 1 ? cluster_rank() : 0;
  const int64_t first_row = g.ranks > 1 ? cluster_index() : blockIdx.x, row_step = g.ranks > 1 ? cluster_count() : gridDim.x;
  const uint32_t buf = sm100::smem_addr(dsmem), bar = buf + static_cast<uint32_t>(g.slice) * 16;
  const T* z = static_cast<const T*>(p.z);
  T* dz = static_cast<T*>(p.dz);
  const bool hard = p.labels != nullptr && p.alpha > 0.0f;
  const float cT = kLog2e / p.temperature, c1 = kLog2e;
  const float wT = p.scale * (1.0f - p.alpha) * p.temperature, w1 = p.scale * p.alpha;
  const int p0 = static_cast<int>(rank) * g.slice;

  // elements before the first whole packet of a row, and packets of this CTA
  auto head_of = [&](int64_t row) {
    const uint32_t a = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(z + row * p.ldz)) & 15u;
    const int h = static_cast<int>(((16u - a) & 15u) / sizeof(T));
    return h < p.C ? h : static_cast<int>(p.C);
  };
  auto packets_of = [&](int head) {
    const int n = static_cast<int>((p.C - head) / kN) - p0;
    return n < 0 ? 0 : n < g.slice ? n : g.slice;
  };
  bool piped = true;  // false once a copy did not arrive: the rest of the rows runs on what the buffer holds
  auto fetch = [&](int64_t row) {  // thread 0
    const int head = head_of(row), n = packets_of(head);
    if (n > 0) {
      sm100::mbar_expect_tx(bar, static_cast<uint32_t>(n) * 16);
      sm100::bulk_copy_g2s(buf, z + row * p.ldz + head + static_cast<int64_t>(p0) * kN, static_cast<uint32_t>(n) * 16, bar);
    }
  };
  // an entry of a row's list (k < K) or its label (k = K)
  auto entry = [&](int64_t row, int k, int* col, float* t, float* zv) {
    int id = -1;
    *t = 0.0f;
    *zv = 0.0f;
    if (k < p.K) id = __ldg(p.ids + row * p.K + k);
    else if (hard) id = __ldg(p.labels + row);
    const bool ok = id >= 0 && id < p.C;
    *col = ok ? id : -1;
    if (ok) {
      if (k < p.K) *t = teacher_at(p, row * p.K + k);
      *zv = Cvt<T>::to_f(z[row * p.ldz + id]);
    }
  };

  if (tid == 0) {
    sm100::mbar_init(bar, 1);
    sm100::mbar_init_fence();
    wait_failed = 0;
    twice[0] = twice[1] = 0;
  }
  for (int i = tid; i < 2 * bits_words; i += nthreads) bits_s[i] = 0u;
  __syncthreads();
  int my_col = -1;
  float my_t = 0.0f, my_z = 0.0f;  // entry `tid` of the row at hand, read one row ahead
  if (first_row < p.B) {
    if (tid == 0) fetch(first_row);
    if (tid < entries) entry(first_row, tid, &my_col, &my_t, &my_z);
  }
  uint32_t phase = 0;
  int par = 0;
  for (int64_t row = first_row; row < p.B; row += row_step, par ^= 1) {
    const int head = head_of(row), pn = packets_of(head);
    const int64_t next = row + row_step;
    // the edges: elements [0, head) and [tail0, C), one per thread of rank 0
    const int tail0 = head + static_cast<int>((p.C - head) / kN) * kN;
    const int edges = rank == 0 ? head + static_cast<int>(p.C) - tail0 : 0;
    const int edge_col = tid < edges ? (tid < head ? tid : tail0 + tid - head) : -1;
    float fe = edge_col >= 0 ? Cvt<T>::to_f(z[row * p.ldz + edge_col]) : -INFINITY;
    if (pn > 0 && piped) {
      if (!sm100::mbar_wait_bounded(bar, phase, rowk::kRowWaitBudgetNs)) wait_failed = 1;
      phase ^= 1u;
    }
    float f[kPk][kN];
#pragma unroll
    for (int q = 0; q < kPk; ++q) {
      const int pi = tid + q * nthreads;
      if (pi < pn) {
        unpack16(row_s[pi], f[q]);
      } else {
#pragma unroll
        for (int e = 0; e < kN; ++e) f[q][e] = -INFINITY;
      }
    }
    auto refill = [&]() {  // behind a barrier: everybody holds its packets
      if (wait_failed) piped = false;
      if (tid == 0 && next < p.B && piped) {
        sm100::fence_generic_to_async_smem();
        fetch(next);
      }
    };
    if (g.early) {
      __syncthreads();
      refill();
    }
    float m = fe;
#pragma unroll
    for (int q = 0; q < kPk; ++q)
#pragma unroll
      for (int e = 0; e < kN; ++e) m = fmaxf(m, f[q][e]);
    // the row's list: staged for everybody, its columns marked, the teacher's sum
    float mt = -INFINITY, st = 0.0f;
    for (int k = tid; k < entries; k += nthreads) {
      if (k != tid) entry(row, k, &my_col, &my_t, &my_z);
      col_s[par * entries + k] = my_col;
      t_s[par * entries + k] = my_t;
      z_s[par * entries + k] = my_z;
      if (my_col >= 0) {
        if (k < p.K) {
          const float to = fmaxf(mt, my_t), ref = to == -INFINITY ? 0.0f : to;
          st = st * (mt == -INFINITY ? 0.0f : rescale(mt, ref, cT)) + ex2((my_t - ref) * cT);
          mt = to;
        }
        if (p.dz) {
          const int at = my_col < head || my_col >= tail0 ? -1 : my_col - head - p0 * kN;
          const bool mine = at >= 0 ? at < pn * kN : at == -1 && rank == 0 && (my_col < head || my_col >= tail0);
          if (mine) {
            const int bit = at >= 0 ? at : g.slice * kN + (my_col < head ? my_col : kN + my_col - tail0);
            if (atomicOr(bits_s + par * bits_words + (bit >> 5), 1u << (bit & 31)) & (1u << (bit & 31))) twice[par] = 1;
          }
        }
      }
    }
    // exponentials below the thread's own maximum
    const float ref = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, s1 = 0.0f;
    auto both = [&](float& v) {  // v: logit -> exponential (kTwoExps: stays a logit)
      const float d = v - ref;
      const float e = ex2(d * cT);
      s += e;
      if constexpr (kMode == kSquares) {
        const float e2 = e * e;
        s1 += g.squarings == 2 ? e2 * e2 : e2;
      }
      if constexpr (kMode == kTwoExps) s1 += ex2(d * c1);
      else v = e;
    };
#pragma unroll
    for (int q = 0; q < kPk; ++q)
#pragma unroll
      for (int e = 0; e < kN; ++e) both(f[q][e]);
    both(fe);
    {
      const float mw = warp_max(m), mtw = warp_max(mt);
      const float k = m == -INFINITY ? (s != s ? s : 0.0f) : rescale(m, mw, cT);
      s = warp_sum(s * k);
      if constexpr (kMode != kOneExp) s1 = warp_sum(s1 * (m == -INFINITY ? 0.0f : rescale(m, mw, c1)));
      st = warp_sum(mt == -INFINITY ? st : st * rescale(mt, mtw, cT));
      if (lane == 0) {
        red[par][0][warp] = mw;
        red[par][1][warp] = s;
        red[par][2][warp] = s1;
        red[par][3][warp] = mtw;
        red[par][4][warp] = st;
      }
    }
    __syncthreads();
    if (!g.early) refill();
    float M, S, S1, Mt, St;
    {
      const bool in = lane < nwarps;
      const float a = in ? red[par][0][lane] : -INFINITY, at = in ? red[par][3][lane] : -INFINITY;
      M = warp_max(a);
      Mt = warp_max(at);
      S = warp_sum(in ? red[par][1][lane] * (a == -INFINITY ? 1.0f : rescale(a, M, cT)) : 0.0f);
      S1 = kMode == kOneExp ? S : warp_sum(in ? red[par][2][lane] * (a == -INFINITY ? 1.0f : rescale(a, M, c1)) : 0.0f);
      St = warp_sum(in ? red[par][4][lane] * (at == -INFINITY ? 1.0f : rescale(at, Mt, cT)) : 0.0f);
    }
    if (nranks > 1) {
      if (warp == 0 && lane < static_cast<int>(nranks)) {
        st_peer_shared(&peer[par][rank][0], lane, M);
        st_peer_shared(&peer[par][rank][1], lane, S);
        st_peer_shared(&peer[par][rank][2], lane, S1);
      }
      __syncwarp();
      cluster_barrier();  // the other parity's slots are rewritten behind this row's barrier only
      float a = -INFINITY, b = 0.0f, c = 0.0f;
      for (uint32_t r = 0; r < nranks; ++r) a = fmaxf(a, peer[par][r][0]);
      for (uint32_t r = 0; r < nranks; ++r) {
        const float pm = peer[par][r][0];
        b += peer[par][r][1] * (pm == -INFINITY ? 1.0f : rescale(pm, a, cT));
        c += peer[par][r][2] * (pm == -INFINITY ? 1.0f : rescale(pm, a, c1));
      }
      M = a, S = b, S1 = kMode == kOneExp ? b : c;
    }
    if (M == -INFINITY && !(S != S)) S = S1 = __int_as_float(0x7fc00000);  // a row of -inf has no softmax
    if (Mt == -INFINITY) Mt = 0.0f;
    const bool some = !(St == 0.0f);  // no entries, or every entry has weight zero: no target
    const bool known = hard && col_s[par * entries + p.K] >= 0;
    const float kT = some ? wT / S : 0.0f, k1 = known ? w1 / S1 : 0.0f;
    // the next row's entries: their loads run while this row is written
    int next_col = -1;
    float next_t = 0.0f, next_z = 0.0f;
    if (next < p.B && tid < entries) entry(next, tid, &next_col, &next_t, &next_z);

    if (rank == 0 && warp == 0) {
      const float invT = 1.0f / p.temperature;
      float cross = 0.0f;
      if (some) {
        for (int k = lane; k < p.K; k += 32) {
          if (col_s[par * entries + k] < 0) continue;
          const float a = (t_s[par * entries + k] - Mt) * invT;
          const float pk = ex2((t_s[par * entries + k] - Mt) * cT) / St;
          if (pk != 0.0f) cross += pk * (a - (z_s[par * entries + k] - M) * invT);
        }
        cross = warp_sum(cross);
      }
      if (lane == 0) {
        float loss = 0.0f;
        if (some) loss = (1.0f - p.alpha) * p.temperature * p.temperature * (cross - logf(St) + logf(S));
        if (known) loss += p.alpha * (logf(S1) + M - z_s[par * entries + p.K]);
        p.loss[row] = loss;
      }
    }
    if (p.dz) {
      T* out = dz + row * p.lddz;
      PK* packets = reinterpret_cast<PK*>(out + head) + p0;
      const bool dead = !some && !known;
      const float up = m == -INFINITY ? 0.0f : rescale(m, M, cT);
      const float gT = kMode == kOneExp ? up * (kT + k1) : up * kT;
      const float g1 = kMode == kSquares ? (m == -INFINITY ? 0.0f : rescale(m, M, c1)) * k1 : 0.0f;
      auto grad = [&](float v) {
        if constexpr (kMode == kOneExp) return v * gT;
        if constexpr (kMode == kSquares) {
          const float v2 = v * v;
          return v * gT + (g.squarings == 2 ? v2 * v2 : v2) * g1;
        }
        const float d = v - M;
        return ex2(d * cT) * kT + ex2(d * c1) * k1;
      };
#pragma unroll
      for (int q = 0; q < kPk; ++q) {
        const int pi = tid + q * nthreads;
        if (pi < pn) {
          PK o;
          float v[kN];
#pragma unroll
          for (int e = 0; e < kN; ++e) v[e] = dead ? 0.0f : grad(f[q][e]);
          pack16(o, v);
          st_stream(packets + pi, o);
        }
      }
      if (edge_col >= 0) out[edge_col] = Cvt<T>::from_f(dead ? 0.0f : grad(fe));
      if (tid == 0) twice[par ^ 1] = 0;  // last read one row ago, next set behind this barrier
      __syncthreads();  // the corrections come behind the row: other threads, the same addresses
      if (!dead) {
        const bool dup = twice[par] != 0;
        for (int k = tid; k < entries; k += nthreads) {
          const int col = col_s[par * entries + k];
          if (col < 0) continue;
          const bool edge = col < head || col >= tail0;
          const int at = col - head - p0 * kN;
          if (edge ? rank != 0 : (at < 0 || at >= pn * kN)) continue;
          auto weight = [&](int j) {
            return j == p.K ? w1 : some ? wT * (ex2((t_s[par * entries + j] - Mt) * cT) / St) : 0.0f;
          };
          float w = 0.0f;
          bool first = true;
          if (dup) {
            for (int j = 0; j < entries; ++j)
              if (col_s[par * entries + j] == col) {
                if (j < k) first = false;
                w += weight(j);
              }
          } else {
            w = weight(k);
          }
          if (!first) continue;
          const float d = z_s[par * entries + k] - M;
          out[col] = Cvt<T>::from_f(ex2(d * cT) * kT + (k1 != 0.0f ? ex2(d * c1) * k1 : 0.0f) - w);
        }
      }
      // this row's marks
      for (int k = tid; k < entries; k += nthreads) {
        const int col = col_s[par * entries + k];
        if (col < 0) continue;
        const bool edge = col < head || col >= tail0;
        const int at = col - head - p0 * kN;
        if (edge ? rank != 0 : (at < 0 || at >= pn * kN)) continue;
        const int bit = !edge ? at : g.slice * kN + (col < head ? col : kN + col - tail0);
        bits_s[par * bits_words + (bit >> 5)] = 0u;
      }
    }
    my_col = next_col, my_t = next_t, my_z = next_z;
  }
  if (nranks > 1) cluster_barrier();  // nobody leaves while a peer may still write its shared memory
  if (wait_failed) {
    if (tid == 0) atomicExch(&g_distill_status, 1);
    for (int i = 0; i < 64; ++i) __nanosleep(16384);  // error path only: let a late copy land
  }
}

template <typename T>
bool plan_rows(const DistillParams& p, RowPlan* out) {
  constexpr int kN = Pack16<T>::kN;
  constexpr int kMaxPk = 64 / kN;
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
  g.ranks = 1;
  while (g.ranks < kMaxRanks && (packets + g.ranks - 1) / g.ranks > static_cast<int64_t>(kRowThreads) * kMaxPk) g.ranks *= 2;
  if (const char* e = std::getenv("AICF_DISTILL_RANKS")) { const int v = std::atoi(e); if (v > g.ranks) g.ranks = v; }
  const int64_t slice = (packets + g.ranks - 1) / g.ranks;
  if (slice > static_cast<int64_t>(kRowThreads) * kMaxPk) return false;
  g.slice = static_cast<int>(slice);
  int grow = 32 / kN; 
  if (const char* e = std::getenv("AICF_DISTILL_GROW")) grow = std::atoi(e);
  g.threads = 32;
  while (g.threads < kRowThreads && static_cast<int64_t>(g.threads) * grow < slice) g.threads *= 2;
  const int per = static_cast<int>((slice + g.threads - 1) / g.threads);
  g.packets = 1;
  while (g.packets < per) g.packets *= 2;
  const size_t words = (slice * kN + 2 * kN + 31) / 32;
  g.smem = static_cast<size_t>(slice) * 16 + 16 + 2 * words * 4 + 2 * static_cast<size_t>(p.K + 1) * 12;
  if (g.smem > 200 * 1024) return false;
  *out = g;
  return true;
}

template <typename T, int kPk, int kMode>
Status launch_rows(const DistillParams& p, RowPlan g, cudaStream_t stream) {
  auto kernel = distill_row_kernel<T, kPk, kMode>;
  static PerDeviceOnce opt_in;
  if (!opt_in.run([&] { return rowk::allow_smem(kernel, 200 * 1024); })) {
    cudaGetLastError();
    return Status::Internal;
  }
  // resident blocks per SM, by threads, registers (allocated to warps in units of 256) and shared memory
  static std::atomic<int> kernel_regs{0};
  int regs = kernel_regs.load(std::memory_order_relaxed);
  if (regs == 0) {
    cudaFuncAttributes a{};
    if (cudaFuncGetAttributes(&a, kernel) != cudaSuccess) {
      cudaGetLastError();
      return Status::Internal;
    }
    regs = a.numRegs;
    kernel_regs.store(regs, std::memory_order_relaxed);
  }
  const int by_regs = 65536 / (((regs + 7) / 8 * 8) * g.threads);
  int resident = rowk::row_pipe_blocks_per_sm(g.threads, g.smem + 1024);
  if (resident > by_regs) resident = by_regs > 0 ? by_regs : 1;
  g.early = resident == 1;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(g.ranks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  int over = 1;
  if (const char* e = std::getenv("AICF_DISTILL_OVER")) over = std::atoi(e);
  const int64_t slots = static_cast<int64_t>(sm_count()) * resident * over / g.ranks;
  const int64_t rows = p.B < slots ? p.B : (slots > 0 ? slots : 1);
  cfg.gridDim = dim3(static_cast<unsigned>(rows * g.ranks));
  cfg.blockDim = dim3(static_cast<unsigned>(g.threads));
  cfg.dynamicSmemBytes = g.smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = g.ranks > 1 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, p, g) != cudaSuccess) {
    cudaGetLastError();
    return Status::Internal;
  }
  return launch_status();
}
template <typename T, int kPk>
Status launch_mode(const DistillParams& p, const RowPlan& g, cudaStream_t stream) {
  if (g.mode == kOneExp) return launch_rows<T, kPk, kOneExp>(p, g, stream);
  if (g.mode == kSquares) return launch_rows<T, kPk, kSquares>(p, g, stream);
  return launch_rows<T, kPk, kTwoExps>(p, g, stream);
}
template <typename T>
Status run_rows(const DistillParams& p, const RowPlan& g, cudaStream_t stream) {
  switch (g.packets) {
    case 1: return launch_mode<T, 1>(p, g, stream);
    case 2: return launch_mode<T, 2>(p, g, stream);
    case 4: return launch_mode<T, 4>(p, g, stream);
    case 8: return launch_mode<T, 8>(p, g, stream);
    default: break;
  }
  if constexpr (sizeof(T) == 4) return launch_mode<T, 16>(p, g, stream);
  return Status::Internal;
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
  if (!(p.temperature > 0.0f) || !(p.temperature <= 3.0e38f) || !(p.alpha >= 0.0f) || !(p.alpha <= 1.0f)) return false;
  if (ni == 4) {
    const TensorDesc& Y = in[3];
    if (Y.dtype != DType::kI32 || Y.rank() != 1 || !Y.contiguous || Y.shape[0] != p.B) return false;
    p.labels = static_cast<const int32_t*>(Y.data);
  } else if (p.alpha > 0.0f) {
    return false;  // a label term without labels
  }
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
