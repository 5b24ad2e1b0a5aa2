// Log probabilities of given classes, the entropy and the best alternatives of
// each row of logits, and their gradient (gfx950).
//
//   m = max z, s = sum e^(z-m), a = sum (z-m) e^(z-m)
//   log p_j = (z_j - m) - log s        H = log s - a / s
// (z - m) and log s are kept apart: their difference keeps its digits however
// large the logits are. A logit of -inf is a class that the mask took away:
// probability 0, nothing to H; a row with no class left has log p = -inf, H = 0
// and gradient 0. NaN or +inf in a row make its numbers NaN.
//
// Order of the alternatives: by value, NaN first, equal values by index.

#include "vec.h"

namespace doa {

constexpr int kTopMost = 32;

// larger key = earlier alternative; 0 is below every element's key
__device__ inline uint64_t top_key(float z, int j) {
  // -0 and +0 are equal values; every NaN is the largest
  uint32_t b = __float_as_uint(z == 0.f ? 0.f : z);
  if (z != z) b = 0x7fffffffu;
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((uint64_t)b << 32) | (uint32_t)~j;
}
__device__ inline int key_index(uint64_t k) { return (int)~(uint32_t)k; }
__device__ inline float key_value(uint64_t k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}

template <typename F, typename Op>
__device__ inline F block_reduce(F v, F* tmp, Op op) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = op(v, __shfl_xor(v, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  v = tmp[0];
  for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v = op(v, tmp[w]);
  return v;
}

template <typename T>
__global__ __launch_bounds__(256) void log_probs_kernel(
    const T* __restrict__ z, int64_t zs, const int64_t* __restrict__ target,
    int64_t ignore, int C, int k, float* __restrict__ lp,
    float* __restrict__ ent, float* __restrict__ top_lp,
    int64_t* __restrict__ top_idx, float* __restrict__ stats) {
  __shared__ float tmp[4];
  __shared__ uint64_t ktmp[4];
  const int64_t row = blockIdx.x;
  const T* zr = z + row * zs;
  float m = -INFINITY;
  for (int j = threadIdx.x; j < C; j += 256) m = fmaxf(m, (float)zr[j]);
  m = block_reduce(m, tmp, [](float a, float b) { return fmaxf(a, b); });
  const float base = m == -INFINITY ? 0.f : m;
  float s = 0.f, a = 0.f;
  for (int j = threadIdx.x; j < C; j += 256) {
    const float d = (float)zr[j] - base;
    const float e = __expf(d);
    s += e;
    a += fmaxf(d, -1e30f) * e;  // -inf * 0
  }
  s = block_reduce(s, tmp, [](float x, float y) { return x + y; });
  a = block_reduce(a, tmp, [](float x, float y) { return x + y; });
  const bool none = s == 0.f;
  const float logs = none ? 0.f : logf(s);
  if (threadIdx.x == 0) {
    ent[row] = none ? 0.f : logs - a / s;
    stats[2 * row] = base;
    stats[2 * row + 1] = none ? INFINITY : logs;  // the mark of an empty row
    if (target) {
      const int64_t t = target[row];
      float v = NAN;
      if (t == ignore) v = 0.f;
      else if (t >= 0 && t < C)
        v = none ? -INFINITY : ((float)zr[t] - base) - logs;
      lp[row] = v;
    }
  }
  uint64_t last = ~0ull;
  for (int i = 0; i < k; ++i) {
    uint64_t best = 0;
    for (int j = threadIdx.x; j < C; j += 256) {
      const uint64_t key = top_key((float)zr[j], j);
      if (key < last && key > best) best = key;
    }
    best = block_reduce(best, ktmp, [](uint64_t x, uint64_t y) {
      return x > y ? x : y;
    });
    if (threadIdx.x == 0) {
      top_idx[row * k + i] = key_index(best);
      top_lp[row * k + i] = (key_value(best) - base) - logs;
    }
    last = best;
  }
}

// dz_j = g_lp [j = t] + sum_i g_i [j = idx_i]
//        - p_j (g_lp + sum_i g_i + g_H (log p_j + H))
template <typename T>
__global__ __launch_bounds__(256) void log_probs_bwd_kernel(
    const T* __restrict__ z, int64_t zs, const int64_t* __restrict__ target,
    int64_t ignore, const int64_t* __restrict__ top_idx,
    const float* __restrict__ stats, const float* __restrict__ ent,
    const float* __restrict__ g_lp, const float* __restrict__ g_ent,
    const float* __restrict__ g_top, int C, int k, T* __restrict__ dz) {
  const int64_t row = blockIdx.x;
  const T* zr = z + row * zs;
  T* out = dz + row * C;
  const float base = stats[2 * row], logs = stats[2 * row + 1];
  const float H = ent[row];
  int64_t t = -1;
  float gl = 0.f;
  if (target && g_lp) {
    t = target[row];
    gl = t == ignore ? 0.f : (t >= 0 && t < C) ? g_lp[row] : NAN;
  }
  float pull = gl;
  if (g_top)
    for (int i = 0; i < k; ++i) pull += g_top[row * k + i];
  const float gh = g_ent ? g_ent[row] : 0.f;
  const bool none = logs == INFINITY;
  for (int j = threadIdx.x; j < C; j += 256) {
    float g = 0.f;
    if (!none) {
      const float l = ((float)zr[j] - base) - logs;
      const float p = __expf(l);
      g = -p * (pull + gh * (fmaxf(l, -1e30f) + H));
      if (j == t) g += gl;
      if (g_top)
        for (int i = 0; i < k; ++i)
          if (top_idx[row * k + i] == j) g += g_top[row * k + i];
    }
    out[j] = (T)g;
  }
}

static at::Tensor logits_rows(const at::Tensor& z) {
  return (z.size(1) <= 1 || z.stride(1) == 1) && z.stride(0) >= 0
             ? z
             : z.contiguous();
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>
log_probs_fwd(at::Tensor logits, c10::optional<at::Tensor> target, int64_t k,
              int64_t ignore) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2,
              "log_probs: [rows, classes] GPU logits expected");
  const int64_t rows = logits.size(0), C = logits.size(1);
  TORCH_CHECK(C >= 1 && C < INT32_MAX, "log_probs: 1 to 2^31 - 2 classes");
  TORCH_CHECK(k >= 0 && k <= kTopMost && k <= C, "log_probs: top_k is at most ",
              kTopMost, " and the number of classes, got ", k);
  if (target.has_value())
    TORCH_CHECK(target->scalar_type() == at::kLong && target->dim() == 1 &&
                    target->size(0) == rows && target->is_contiguous() &&
                    target->device() == logits.device(),
                "log_probs: contiguous int64 [rows] targets expected");
  c10::DeviceGuard guard(logits.device());
  auto zc = logits_rows(logits);
  auto f32 = logits.options().dtype(at::kFloat);
  at::Tensor lp;
  if (target.has_value()) lp = at::empty({rows}, f32);
  auto ent = at::empty({rows}, f32);
  auto top_lp = at::empty({rows, k}, f32);
  auto top_idx = at::empty({rows, k}, logits.options().dtype(at::kLong));
  auto stats = at::empty({rows, 2}, f32);
  if (rows > 0)
    DOA_FLOAT_TYPES(logits.scalar_type(), "log_probs", [&] {
      TORCH_CHECK(rows < INT32_MAX, "log_probs: too many rows");
      hipLaunchKernelGGL(
          (log_probs_kernel<T>), dim3(rows), dim3(256), 0, stream_of_current(),
          (const T*)zc.data_ptr(), zc.stride(0),
          target.has_value() ? target->data_ptr<int64_t>() : nullptr, ignore,
          (int)C, (int)k, lp.defined() ? lp.data_ptr<float>() : nullptr,
          ent.data_ptr<float>(), top_lp.data_ptr<float>(),
          top_idx.data_ptr<int64_t>(), stats.data_ptr<float>());
    });
  DOA_CHECK_HIP(hipGetLastError());
  return {lp, ent, top_lp, top_idx, stats};
}

at::Tensor log_probs_bwd(at::Tensor logits, c10::optional<at::Tensor> target,
                         int64_t ignore, at::Tensor top_idx, at::Tensor stats,
                         at::Tensor ent, c10::optional<at::Tensor> g_lp,
                         c10::optional<at::Tensor> g_ent,
                         c10::optional<at::Tensor> g_top) {
  const int64_t rows = logits.size(0), C = logits.size(1), k = top_idx.size(1);
  c10::DeviceGuard guard(logits.device());
  auto zc = logits_rows(logits);
  auto dz = at::empty({rows, C}, logits.options());
  at::Tensor keep[3];
  const float* gp[3] = {nullptr, nullptr, nullptr};
  const c10::optional<at::Tensor>* gs[3] = {&g_lp, &g_ent, &g_top};
  for (int i = 0; i < 3; ++i)
    if (gs[i]->has_value()) {
      keep[i] = (*gs[i])->contiguous();
      TORCH_CHECK(keep[i].scalar_type() == at::kFloat &&
                      keep[i].numel() == rows * (i == 2 ? k : 1),
                  "log_probs: gradient of another shape or type");
      gp[i] = keep[i].data_ptr<float>();
    }
  if (rows > 0)
    DOA_FLOAT_TYPES(logits.scalar_type(), "log_probs", [&] {
      hipLaunchKernelGGL(
          (log_probs_bwd_kernel<T>), dim3(rows), dim3(256), 0,
          stream_of_current(), (const T*)zc.data_ptr(), zc.stride(0),
          target.has_value() ? target->data_ptr<int64_t>() : nullptr, ignore,
          top_idx.data_ptr<int64_t>(), stats.data_ptr<float>(),
          ent.data_ptr<float>(), gp[0], gp[1], gp[2], (int)C, (int)k,
          (T*)dz.data_ptr());
    });
  DOA_CHECK_HIP(hipGetLastError());
  return dz;
}

}  // namespace doa
