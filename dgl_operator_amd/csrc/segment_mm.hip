// Product of each group of rows with its own weight (gfx950, MFMA):
//
//   y[r] = x[r] W[g]          for offsets[g] <= r < offsets[g+1]
//   dx[r] = dy[r] W[g]^T      the same with the weight's strides swapped
//   dW[g] = x_g^T dy_g        a reduction over the group's rows
//
// Products accumulate in fp32 and are rounded once. Rows outside every group
// are zero, and so is an empty group's dW. The grid is sized from the host's
// numbers alone (rows, groups): group g's row tiles start at the virtual tile
// offsets[g] / BM + g, which grows with g and leaves each group room for its
// last, partial tile, so a block finds its group by a search of the offsets.

#include "vec.h"

namespace doa {

using f32x4 = __attribute__((__vector_size__(4 * sizeof(float)))) float;

template <typename T>
struct Mma;
template <>
struct Mma<float> {
  static constexpr int K = 4;  // depth of one instruction
  using Frag = float;
  static __device__ f32x4 run(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<__bf16> {
  static constexpr int K = 32;
  using Frag = __attribute__((__vector_size__(16))) __bf16;
  static __device__ f32x4 run(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<_Float16> {
  static constexpr int K = 32;
  using Frag = __attribute__((__vector_size__(16))) _Float16;
  static __device__ f32x4 run(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

constexpr int kTile = 64;  // rows and columns of a block's tile

// c[m][n] = sum_k a(m, k) b(k, n) for one tile of 64 x 64, 4 waves of 32 x 32
template <typename T>
__device__ inline void tile_product(const T* a, int64_t am, int64_t ak, int M,
                                    const T* b, int64_t bk, int64_t bn, int N,
                                    int64_t K, T* c, int64_t ldc) {
  constexpr int BK = sizeof(T) == 4 ? 16 : 32;
  constexpr int LD = BK + 16 / sizeof(T);
  __shared__ __align__(16) T As[kTile * LD];
  __shared__ __align__(16) T Bs[kTile * LD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  f32x4 acc[2][2] = {};
  for (int64_t k0 = 0; k0 < K; k0 += BK) {
    __syncthreads();
    for (int i = threadIdx.x; i < kTile * BK; i += 256) {
      // consecutive threads along whichever of the two is contiguous
      const int m = ak == 1 ? i / BK : i % kTile;
      const int k = ak == 1 ? i % BK : i / kTile;
      As[m * LD + k] = (m < M && k0 + k < K) ? a[m * am + (k0 + k) * ak] : (T)0.f;
    }
    for (int i = threadIdx.x; i < kTile * BK; i += 256) {
      const int n = bk == 1 ? i / BK : i % kTile;
      const int k = bk == 1 ? i % BK : i / kTile;
      Bs[n * LD + k] = (n < N && k0 + k < K) ? b[(k0 + k) * bk + n * bn] : (T)0.f;
    }
    __syncthreads();
    constexpr int per = Mma<T>::K / 4;
    using Frag = typename Mma<T>::Frag;
#pragma unroll
    for (int k = 0; k < BK; k += Mma<T>::K) {
      Frag fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = *reinterpret_cast<const Frag*>(
            &As[(wm + i * 16 + (lane & 15)) * LD + k + (lane >> 4) * per]);
        fb[i] = *reinterpret_cast<const Frag*>(
            &Bs[(wn + i * 16 + (lane & 15)) * LD + k + (lane >> 4) * per]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = Mma<T>::run(fa[i], fb[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = wm + i * 16 + (lane >> 4) * 4 + r;
        const int n = wn + j * 16 + (lane & 15);
        if (m < M && n < N) c[m * ldc + n] = (T)acc[i][j][r];
      }
}

__device__ inline int64_t offset_at(const int64_t* offsets, int g,
                                    int64_t rows) {
  const int64_t o = offsets[g];
  return o < 0 ? 0 : o > rows ? rows : o;  // never outside the rows
}

template <typename T>
__global__ __launch_bounds__(256) void segment_mm_kernel(
    const T* __restrict__ x, int64_t xs, const T* __restrict__ w, int64_t wg,
    int64_t wk, int64_t wn, const int64_t* __restrict__ offsets,
    T* __restrict__ y, int64_t rows, int G, int K, int N) {
  // rows of no group
  const int64_t first = offset_at(offsets, 0, rows);
  const int64_t end = offset_at(offsets, G, rows);
  if (blockIdx.y == 0) {
    const int64_t outside = (first + rows - end) * N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < outside;
         i += (int64_t)gridDim.x * 256)
      y[i < first * N ? i : i + (end - first) * N] = (T)0.f;
  }
  const int64_t v = blockIdx.x;
  int lo = 0, hi = G;  // the last g with start(g) <= v
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offset_at(offsets, mid, rows) / kTile + mid <= v) lo = mid; else hi = mid;
  }
  const int64_t begin = offset_at(offsets, lo, rows);
  const int64_t r0 = begin + (v - begin / kTile - lo) * kTile;
  const int64_t stop = offset_at(offsets, lo + 1, rows);
  if (r0 < begin || r0 >= stop) return;
  const int n0 = blockIdx.y * kTile;
  tile_product<T>(x + r0 * xs, xs, 1, (int)min((int64_t)kTile, stop - r0),
                  w + lo * wg + n0 * wn, wk, wn, min(kTile, N - n0), K,
                  y + r0 * N + n0, N);
}

template <typename T>
__global__ __launch_bounds__(256) void segment_mm_wgrad_kernel(
    const T* __restrict__ x, int64_t xs, const T* __restrict__ g, int64_t gs,
    const int64_t* __restrict__ offsets, T* __restrict__ dw, int64_t rows,
    int K, int N, int tiles_n) {
  const int e = blockIdx.y;
  const int64_t begin = offset_at(offsets, e, rows);
  const int64_t stop = offset_at(offsets, e + 1, rows);
  const int k0 = blockIdx.x / tiles_n * kTile, n0 = blockIdx.x % tiles_n * kTile;
  tile_product<T>(x + begin * xs + k0, 1, xs, min(kTile, K - k0),
                  g + begin * gs + n0, gs, 1, min(kTile, N - n0),
                  max((int64_t)0, stop - begin),
                  dw + ((int64_t)e * K + k0) * N + n0, N);
}

static at::Tensor mm_rows(const at::Tensor& t) {
  return (t.size(1) <= 1 || t.stride(1) == 1) && t.stride(0) >= 0
             ? t
             : t.contiguous();
}

static void check_offsets(const at::Tensor& offsets, const at::Tensor& x,
                          int64_t groups, const char* what) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, what, ": 2-D GPU rows expected");
  TORCH_CHECK(offsets.scalar_type() == at::kLong && offsets.dim() == 1 &&
                  offsets.is_contiguous() && offsets.numel() == groups + 1 &&
                  offsets.device() == x.device() && groups >= 1,
              what, ": int64 offsets [groups + 1] on the rows' device expected");
  TORCH_CHECK(groups <= 65535, what, ": at most 65535 groups");
}

// x [R, K] by weight [G, K, N] (any strides); transposed: x [R, N] by its
// transpose
at::Tensor segment_mm(at::Tensor offsets, at::Tensor x, at::Tensor weight,
                      bool transposed) {
  const int64_t G = weight.size(0);
  check_offsets(offsets, x, G, "segment_mm");
  TORCH_CHECK(weight.dim() == 3 && weight.device() == x.device() &&
                  weight.scalar_type() == x.scalar_type(),
              "segment_mm: weight [groups, K, N] of the rows' type expected");
  const int64_t K = weight.size(transposed ? 2 : 1);
  const int64_t N = weight.size(transposed ? 1 : 2);
  TORCH_CHECK(x.size(1) == K, "segment_mm: rows of ", K, " expected, got ",
              x.size(1));
  TORCH_CHECK(K < INT32_MAX && N < INT32_MAX, "segment_mm: too wide");
  c10::DeviceGuard guard(x.device());
  auto xc = mm_rows(x);
  const int64_t R = x.size(0);
  auto y = at::empty({R, N}, x.options());
  if (R * N == 0) return y;
  const int64_t wk = weight.stride(transposed ? 2 : 1);
  const int64_t wn = weight.stride(transposed ? 1 : 2);
  const int64_t tiles = R / kTile + G;
  TORCH_CHECK(tiles < INT32_MAX && ceil_div(N, kTile) <= 65535,
              "segment_mm: too many tiles");
  DOA_FLOAT_TYPES(x.scalar_type(), "segment_mm", [&] {
    hipLaunchKernelGGL((segment_mm_kernel<T>),
                       dim3(tiles, ceil_div(N, kTile)), dim3(256), 0,
                       stream_of_current(), (const T*)xc.data_ptr(),
                       xc.stride(0), (const T*)weight.data_ptr(),
                       weight.stride(0), wk, wn, offsets.data_ptr<int64_t>(),
                       (T*)y.data_ptr(), R, (int)G, (int)K, (int)N);
  });
  DOA_CHECK_HIP(hipGetLastError());
  return y;
}

at::Tensor segment_mm_wgrad(at::Tensor offsets, at::Tensor x, at::Tensor grad) {
  const int64_t G = offsets.numel() - 1;
  check_offsets(offsets, x, G, "segment_mm");
  TORCH_CHECK(grad.dim() == 2 && grad.size(0) == x.size(0) &&
                  grad.device() == x.device() &&
                  grad.scalar_type() == x.scalar_type(),
              "segment_mm: gradient rows of another shape or type");
  c10::DeviceGuard guard(x.device());
  auto xc = mm_rows(x);
  auto gc = mm_rows(grad);
  const int64_t K = x.size(1), N = grad.size(1);
  auto dw = at::empty({G, K, N}, x.options());
  if (dw.numel() == 0) return dw;
  const int64_t tn = ceil_div(N, kTile);
  DOA_FLOAT_TYPES(x.scalar_type(), "segment_mm", [&] {
    hipLaunchKernelGGL((segment_mm_wgrad_kernel<T>),
                       dim3(ceil_div(K, kTile) * tn, G), dim3(256), 0,
                       stream_of_current(), (const T*)xc.data_ptr(),
                       xc.stride(0), (const T*)gc.data_ptr(), gc.stride(0),
                       offsets.data_ptr<int64_t>(), (T*)dw.data_ptr(),
                       x.size(0), (int)K, (int)N, (int)tn);
  });
  DOA_CHECK_HIP(hipGetLastError());
  return dw;
}

}  // namespace doa
