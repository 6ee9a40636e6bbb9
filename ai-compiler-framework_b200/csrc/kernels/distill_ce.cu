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
// dz may be z itself; otherwise outputs do not overlap inputs.
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
    int some = 0;
    for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
      const int id = p.ids[row * p.K + k];
      const bool ok = id >= 0 && id < p.C;
      col_s[k] = ok ? id : -1;
      some |= ok;
      if (ok) mt = fmaxf(mt, teacher_at(p, row * p.K + k));
    }
    if (threadIdx.x == 0) {
      col_s[p.K] = known ? static_cast<int>(label) : -1;
      w_s[p.K] = p.alpha;
    }
    some = __syncthreads_or(some);
    mt = block_reduce<true>(mt, red);
    if (mt == -INFINITY) some = 0;  // every entry has weight zero: no target
    float st = 0.0f;
    for (int k = threadIdx.x; k < p.K; k += blockDim.x)
      if (some && col_s[k] >= 0) st += expf((teacher_at(p, row * p.K + k) - mt) * invT);
    st = block_reduce<false>(st, red);
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

KernelVariant make_distill_ce_f32_variant() { return make<DType::kF32, float>("distill_ce_f32_sm100"); }
KernelVariant make_distill_ce_bf16_variant() { return make<DType::kBF16, __nv_bfloat16>("distill_ce_bf16_sm100"); }
KernelVariant make_distill_ce_f16_variant() { return make<DType::kF16, __half>("distill_ce_f16_sm100"); }

}  // namespace aicf::cuda
