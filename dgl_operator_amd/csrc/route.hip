// Rows sorted by group and back (gfx950): the plan, the copy out, the
// weighted sum home, and their gradients.
//
// Slot f = t*k + j asks for group ids[t, j]. The plan is a STABLE counting
// sort of the slots by group: position[f] = offsets[id_f] + #{f' < f of the
// same id}; a slot whose id lies outside [0, G) is dropped (position -1) and
// the rows behind the last group hold nothing (source -1, zeros). Everything
// is a sum of integers or of floats in a fixed order, so a run repeats bit
// for bit. No host synchronisation: the number of kept slots stays on the
// device.
//
// Measured on one MI355X, where a large copy moves 4.8 TB/s: the plan of 53504
// slots in 16 groups 12 us in three launches, of 16 slots 3 us in one, of 65536
// slots in 1345 groups 32 us (there each wave's own start of every group is
// what counts).

#include "vec.h"

namespace doa {

constexpr int kRouteMaxGroups = 16384;  // one wave's counters: 64 KiB of LDS

// lanes of this wave with my id (a match by ballots over the id's bits)
__device__ inline uint64_t same_id_lanes(int id, bool valid, int bits) {
  uint64_t m = __ballot(valid);
  for (int b = 0; b < bits; ++b) {
    const bool on = (id >> b) & 1;
    const uint64_t v = __ballot(on);
    m &= on ? v : ~v;
  }
  return m;
}

template <typename IdT>
__device__ inline int load_id(const IdT* ids, int64_t f, int64_t n, int G) {
  if (f >= n) return -1;
  const IdT id = ids[f];
  return (id >= 0 && id < (IdT)G) ? (int)id : -1;
}

// exclusive scan of one value a thread over the block; `sums` holds one int a
// wave; returns the block's total through `total`
__device__ inline int block_exclusive(int v, int* sums, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int inc = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(inc, d);
    if (lane >= d) inc += o;
  }
  __syncthreads();  // the last round's reads of sums are over
  if (lane == 63) sums[wave] = inc;
  __syncthreads();
  int before = 0, all = 0;
  const int waves = blockDim.x >> 6;
  for (int w = 0; w < waves; ++w) {
    if (w < wave) before += sums[w];
    all += sums[w];
  }
  *total = all;
  return before + inc - v;
}

// one wave puts its slots [lo, hi) in order, from where `next` says the next
// slot of each group goes; 4 x 64 ids are on their way at once
template <typename IdT>
__device__ inline void place_tile(const IdT* ids, int64_t lo, int64_t hi,
                                  int G, int bits, int* next,
                                  int* __restrict__ position,
                                  int* __restrict__ source) {
  const int lane = threadIdx.x & 63;
  for (int64_t base = lo; base < hi; base += 256) {
    int id[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) id[u] = load_id(ids, base + u * 64 + lane, hi, G);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t f = base + u * 64 + lane;
      const bool valid = id[u] >= 0;
      const uint64_t same = same_id_lanes(id[u], valid, bits);
      int p = -1;
      if (valid) {
        const uint64_t below = same & ((1ull << lane) - 1);
        p = next[id[u]] + __popcll(below);
        // the last of the lanes moves the group's counter on (a wave's LDS
        // operations keep their order)
        if ((same >> lane) == 1ull) next[id[u]] = p + 1;
        source[p] = (int)f;
      }
      wave_sync();
      if (f < hi) position[f] = p;
    }
  }
}

// ---- few slots: the whole plan in one block, one launch --------------------
template <typename IdT>
__global__ __launch_bounds__(1024) void route_small_kernel(
    const IdT* __restrict__ ids, int n, int G, int bits, int tile,
    int64_t* __restrict__ offsets, int* __restrict__ position,
    int* __restrict__ source) {
  extern __shared__ int hist[];  // [waves][G]
  __shared__ int sums[16];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int waves = blockDim.x >> 6;
  int* mine = hist + wave * G;
  for (int g = lane; g < G; g += 64) mine[g] = 0;
  wave_sync();
  const int lo = wave * tile, hi = min(n, lo + tile);
  for (int f = lo + lane; f < hi; f += 64) {
    const int id = load_id(ids, f, n, G);
    if (id >= 0) atomicAdd(&mine[id], 1);
  }
  __syncthreads();
  int carry = 0;
  for (int base = 0; base < G; base += blockDim.x) {
    const int g = base + threadIdx.x;
    int total = 0;
    if (g < G)
      for (int w = 0; w < waves; ++w) total += hist[w * G + g];
    int all;
    int at = carry + block_exclusive(total, sums, &all);
    carry += all;
    if (g < G) {
      offsets[g] = at;
      for (int w = 0; w < waves; ++w) {
        const int c = hist[w * G + g];
        hist[w * G + g] = at;
        at += c;
      }
    }
  }
  if (threadIdx.x == 0) offsets[G] = carry;
  __syncthreads();
  place_tile(ids, lo, hi, G, bits, mine, position, source);
  for (int p = carry + threadIdx.x; p < n; p += blockDim.x) source[p] = -1;
}

// ---- many slots: count, scan over tiles, place; a wave a tile --------------
template <typename IdT>
__global__ __launch_bounds__(64) void route_count_kernel(
    const IdT* __restrict__ ids, int64_t n, int G, int tile, int tiles,
    int* __restrict__ counts) {  // [G][tiles]
  extern __shared__ int hist[];
  const int lane = threadIdx.x, t = blockIdx.x;
  for (int g = lane; g < G; g += 64) hist[g] = 0;
  wave_sync();
  const int64_t lo = (int64_t)t * tile, hi = min(n, lo + tile);
  for (int64_t f = lo + lane; f < hi; f += 64) {
    const int id = load_id(ids, f, n, G);
    if (id >= 0) atomicAdd(&hist[id], 1);
  }
  wave_sync();
  for (int g = lane; g < G; g += 64) counts[(int64_t)g * tiles + t] = hist[g];
}

// each block: one group's counts over the tiles, to exclusive sums
__global__ __launch_bounds__(256) void route_scan_kernel(
    int* __restrict__ counts, int tiles, int* __restrict__ totals) {
  __shared__ int sums[4];
  int* c = counts + (int64_t)blockIdx.x * tiles;
  int carry = 0;
  for (int base = 0; base < tiles; base += blockDim.x) {
    const int i = base + threadIdx.x;
    const int v = i < tiles ? c[i] : 0;
    int all;
    const int at = carry + block_exclusive(v, sums, &all);
    if (i < tiles) c[i] = at;
    carry += all;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

template <typename IdT>
__global__ __launch_bounds__(64) void route_place_kernel(
    const IdT* __restrict__ ids, int64_t n, int G, int bits, int tile,
    int tiles, const int* __restrict__ counts, const int* __restrict__ totals,
    int64_t* __restrict__ offsets, int* __restrict__ position,
    int* __restrict__ source) {
  extern __shared__ int next[];
  const int lane = threadIdx.x, t = blockIdx.x;
  // every wave sums up the groups' totals by itself: less than a launch
  int carry = 0;
#pragma unroll 4
  for (int base = 0; base < G; base += 64) {
    const int g = base + lane;
    const int v = g < G ? totals[g] : 0;
    const int before = g < G ? counts[(int64_t)g * tiles + t] : 0;
    int inc = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(inc, d);
      if (lane >= d) inc += o;
    }
    const int at = carry + inc - v;
    if (g < G) {
      next[g] = at + before;
      if (t == 0) offsets[g] = at;
    }
    carry += __shfl(inc, 63);
  }
  if (t == 0 && lane == 0) offsets[G] = carry;
  wave_sync();
  const int64_t lo = (int64_t)t * tile, hi = min(n, lo + tile);
  place_tile(ids, lo, hi, G, bits, next, position, source);
  for (int64_t p = carry + (int64_t)t * 64 + lane; p < n;
       p += (int64_t)tiles * 64)
    source[p] = -1;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> route_rows(at::Tensor ids,
                                                          int64_t groups) {
  TORCH_CHECK(ids.is_cuda(), "route_rows: ids must be on GPU");
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt,
              "route_rows: int64 or int32 ids expected");
  TORCH_CHECK(groups >= 1 && groups <= kRouteMaxGroups,
              "route_rows: 1 to ", kRouteMaxGroups, " groups, got ", groups);
  const int64_t n = ids.numel();
  TORCH_CHECK(n < (int64_t)INT32_MAX, "route_rows: too many slots");
  c10::DeviceGuard guard(ids.device());
  auto idc = ids.contiguous();
  auto i32 = ids.options().dtype(at::kInt);
  auto offsets = at::empty({groups + 1}, ids.options().dtype(at::kLong));
  auto position = at::empty(ids.sizes(), i32);
  auto source = at::empty({n}, i32);
  const int G = (int)groups;
  int bits = 0;
  while ((1 << bits) < G) ++bits;
  auto stream = stream_of_current();
  // counters a block: 64 KiB of LDS with the scan's few, one set a wave
  const int fit = std::max(1, (kRouteMaxGroups - 16) / G);
  auto go = [&](auto* idp) {
    using IdT = std::remove_const_t<std::remove_pointer_t<decltype(idp)>>;
    if (n <= 8192 && G <= 4096) {
      const int waves = (int)std::max<int64_t>(
          1, std::min<int64_t>({16, fit, ceil_div(n, 64)}));
      const int tile = (int)ceil_div(ceil_div(n, waves), 64) * 64;
      hipLaunchKernelGGL((route_small_kernel<IdT>), dim3(1), dim3(64 * waves),
                         (size_t)waves * G * sizeof(int), stream, idp, (int)n,
                         G, bits, tile, offsets.data_ptr<int64_t>(),
                         position.data_ptr<int>(), source.data_ptr<int>());
      return;
    }
    // a tile's G counters are written and read once more: a tile of G/4 slots
    // keeps them at a few bytes a slot; at least 256 slots, and no more tiles
    // than fill the chip
    const int64_t want =
        std::max<int64_t>({256, G / 4, ceil_div(n, 8192)});
    const int tile = (int)ceil_div(want, 64) * 64;
    // (one tile where there is no slot: it writes the offsets)
    const int tiles = (int)std::max<int64_t>(1, ceil_div(n, tile));
    auto counts = at::empty({(int64_t)G * tiles + G}, i32);
    int* cp = counts.data_ptr<int>();
    int* totals = cp + (int64_t)G * tiles;
    const size_t lds = (size_t)G * sizeof(int);
    hipLaunchKernelGGL((route_count_kernel<IdT>), dim3(tiles), dim3(64), lds,
                       stream, idp, n, G, tile, tiles, cp);
    hipLaunchKernelGGL(route_scan_kernel, dim3(G),
                       dim3(tiles <= 64 ? 64 : 256), 0, stream, cp, tiles,
                       totals);
    hipLaunchKernelGGL((route_place_kernel<IdT>), dim3(tiles), dim3(64), lds,
                       stream, idp, n, G, bits, tile, tiles, cp, totals,
                       offsets.data_ptr<int64_t>(), position.data_ptr<int>(),
                       source.data_ptr<int>());
  };
  if (ids.scalar_type() == at::kLong)
    go(idc.data_ptr<int64_t>());
  else
    go(idc.data_ptr<int>());
  DOA_CHECK_HIP(hipGetLastError());
  return {offsets, position, source};
}

// ---------------------------------------------------------------------------
// The row kernels: 2^sh lanes a row, 16 bytes a lane where rows allow it.
// Bound by memory. They go over the rows before sorting, so that each of those
// is read (or written) once whatever k, and the sorted rows once each. 262144
// rows of 512 in bf16 with k = 2: copy out 137 us (5.9 TB/s), weighted sum 167 us
// (4.8 TB/s), its gradient 263 us (5.1 TB/s).
// ---------------------------------------------------------------------------

// a slot's row: not that of a dropped one, and never outside the sorted rows
__device__ inline bool inside(int p, int64_t n) { return p >= 0 && p < n; }

// rows behind the last group
template <typename T, int V>
__device__ inline void zero_tail(T* out, int64_t end, int64_t n, int D,
                                 int sh) {
  const int lane = threadIdx.x & ((1 << sh) - 1);
  Vec<T, V> z;
#pragma unroll
  for (int i = 0; i < V; ++i) z.v[i] = (T)0.f;
  for (int64_t p = max((int64_t)0, end) +
                   (((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> sh);
       p < n; p += ((int64_t)gridDim.x * blockDim.x) >> sh)
    for (int c = lane * V; c < D; c += V << sh)
      *reinterpret_cast<Vec<T, V>*>(out + p * D + c) = z;
}

// out[position[t, j]] = x[t]: x is read once, whatever k
template <typename T, int V>
__global__ __launch_bounds__(256) void dispatch_rows_kernel(
    const T* __restrict__ x, int64_t xs, const int* __restrict__ position,
    const int64_t* __restrict__ offsets_end, T* __restrict__ out, int64_t rows,
    int k, int D, int sh) {
  const int lane = threadIdx.x & ((1 << sh) - 1);
  const int64_t step = ((int64_t)gridDim.x * blockDim.x) >> sh;
  for (int64_t t = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> sh;
       t < rows; t += step)
    for (int c = lane * V; c < D; c += V << sh) {
      const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(x + t * xs + c);
      for (int j = 0; j < k; ++j) {
        const int p = position[t * k + j];
        if (inside(p, rows * k))
          *reinterpret_cast<Vec<T, V>*>(out + (int64_t)p * D + c) = v;
      }
    }
  zero_tail<T, V>(out, *offsets_end, rows * k, D, sh);
}

// out[t] = sum_j w[t, j] y[position[t, j]], summed in fp32 in the order of j
template <typename T, int V>
__global__ __launch_bounds__(256) void combine_rows_kernel(
    const T* __restrict__ y, int64_t ys, const int* __restrict__ position,
    const float* __restrict__ w, T* __restrict__ out, int64_t rows, int k,
    int D, int sh) {
  const int lane = threadIdx.x & ((1 << sh) - 1);
  const int64_t step = ((int64_t)gridDim.x * blockDim.x) >> sh;
  for (int64_t t = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> sh;
       t < rows; t += step)
    for (int c = lane * V; c < D; c += V << sh) {
      float acc[V];
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = 0.f;
      for (int j = 0; j < k; ++j) {
        const int p = position[t * k + j];
        if (!inside(p, rows * k)) continue;
        const float wj = w ? w[t * k + j] : 1.f;
        const Vec<T, V> v =
            *reinterpret_cast<const Vec<T, V>*>(y + (int64_t)p * ys + c);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += wj * (float)v.v[i];
      }
      Vec<T, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) o.v[i] = (T)acc[i];
      *reinterpret_cast<Vec<T, V>*>(out + t * D + c) = o;
    }
}

// dy[position[t, j]] = w[t, j] g[t];  dw[t, j] = <g[t], y[position[t, j]]>
template <typename T, int V>
__global__ __launch_bounds__(256) void combine_rows_bwd_kernel(
    const T* __restrict__ g, int64_t gs, const T* __restrict__ y, int64_t ys,
    const int* __restrict__ position, const int64_t* __restrict__ offsets_end,
    const float* __restrict__ w, T* __restrict__ dy, float* __restrict__ dw,
    int64_t rows, int k, int D, int sh) {
  const int lane = threadIdx.x & ((1 << sh) - 1);
  const int64_t step = ((int64_t)gridDim.x * blockDim.x) >> sh;
  // whole waves walk the rows, so that the shuffles find their lanes
  for (int64_t t0 = ((int64_t)blockIdx.x * blockDim.x + (threadIdx.x & ~63)) >> sh;
       t0 < rows; t0 += step) {
    const int64_t t = t0 + ((threadIdx.x & 63) >> sh);
    const bool live = t < rows;
    for (int j = 0; j < k; ++j) {
      const int p = live ? position[t * k + j] : -1;
      float part = 0.f;
      if (inside(p, rows * k)) {
        const float wj = w ? w[t * k + j] : 1.f;
        for (int c = lane * V; c < D; c += V << sh) {
          const Vec<T, V> gv =
              *reinterpret_cast<const Vec<T, V>*>(g + t * gs + c);
          if (dw) {
            const Vec<T, V> yv =
                *reinterpret_cast<const Vec<T, V>*>(y + (int64_t)p * ys + c);
#pragma unroll
            for (int i = 0; i < V; ++i)
              part += (float)gv.v[i] * (float)yv.v[i];
          }
          if (dy) {
            Vec<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = (T)(wj * (float)gv.v[i]);
            *reinterpret_cast<Vec<T, V>*>(dy + (int64_t)p * D + c) = o;
          }
        }
      }
      if (dw) {
        for (int d = 1; d < (1 << sh); d <<= 1) part += __shfl_xor(part, d);
        if (live && lane == 0) dw[t * k + j] = part;
      }
    }
  }
  if (dy) zero_tail<T, V>(dy, *offsets_end, rows * k, D, sh);
}

// lanes a row: the power of two that covers a row's vectors, at most a wave
static int row_shift(int64_t vecs) {
  int sh = 0;
  while (sh < 6 && (1 << sh) < vecs) ++sh;
  return sh;
}

#define DOA_ROW_VEC(VEC, ...)                                   \
  [&] {                                                         \
    constexpr int most = 16 / sizeof(T);                        \
    switch (VEC) {                                              \
      case most: { constexpr int V = most; __VA_ARGS__(); break; }          \
      case most / 2: { constexpr int V = most / 2; __VA_ARGS__(); break; }  \
      case most / 4: { constexpr int V = most / 4; __VA_ARGS__(); break; }  \
      default: { constexpr int V = 1; __VA_ARGS__(); }          \
    }                                                           \
  }()

static at::Tensor row_contiguous(const at::Tensor& t) {
  return (t.size(1) <= 1 || t.stride(1) == 1) && t.stride(0) >= 0
             ? t
             : t.contiguous();
}

static void check_plan(const at::Tensor& position, const char* what) {
  TORCH_CHECK(position.dim() == 2 && position.scalar_type() == at::kInt &&
                  position.is_contiguous(),
              what, ": the plan's contiguous int32 positions expected");
}
static void check_plan(const at::Tensor& position, const at::Tensor& offsets,
                       const char* what) {
  check_plan(position, what);
  TORCH_CHECK(offsets.dim() == 1 && offsets.scalar_type() == at::kLong &&
                  offsets.numel() >= 1 && offsets.is_contiguous() &&
                  offsets.device() == position.device(),
              what, ": the plan's contiguous int64 offsets expected");
}

static void check_rows(const at::Tensor& t, const at::Tensor& position,
                       int64_t rows, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == position.device() && t.dim() == 2 &&
                  t.size(0) == rows,
              what, ": [", rows, ", D] rows on the plan's device expected");
  // columns are counted in 32 bits, a wave's step beyond the last one too
  TORCH_CHECK(t.size(1) < (1 << 30), what, ": rows of fewer than 2^30 elements "
              "expected, got ", t.size(1));
}

static const float* weights_ptr(const c10::optional<at::Tensor>& w,
                                const at::Tensor& position, const char* what) {
  if (!w.has_value()) return nullptr;
  TORCH_CHECK(w->scalar_type() == at::kFloat && w->is_contiguous() &&
                  w->sizes() == position.sizes() &&
                  w->device() == position.device(),
              what, ": contiguous fp32 weights of the plan's shape expected");
  return w->data_ptr<float>();
}

at::Tensor dispatch_rows(at::Tensor x, at::Tensor position,
                         at::Tensor offsets) {
  check_plan(position, offsets, "dispatch_rows");
  const int64_t rows = position.size(0), k = position.size(1);
  check_rows(x, position, rows, "dispatch_rows");
  c10::DeviceGuard guard(x.device());
  auto xc = row_contiguous(x);
  const int64_t D = x.size(1);
  auto out = at::empty({rows * k, D}, x.options());
  if (out.numel() == 0) return out;
  DOA_FLOAT_TYPES(x.scalar_type(), "dispatch_rows", [&] {
    const int vec = row_vec(xc.data_ptr(), D, xc.stride(0), sizeof(T));
    const int sh = row_shift(ceil_div(D, vec));
    DOA_ROW_VEC(vec, [&] {
      hipLaunchKernelGGL((dispatch_rows_kernel<T, V>),
                         dim3(grid_for(rows << sh, 256, 1 << 20)), dim3(256), 0,
                         stream_of_current(), (const T*)xc.data_ptr(),
                         xc.stride(0), position.data_ptr<int>(),
                         offsets.data_ptr<int64_t>() + offsets.numel() - 1,
                         (T*)out.data_ptr(), rows, (int)k, (int)D, sh);
    });
  });
  DOA_CHECK_HIP(hipGetLastError());
  return out;
}

at::Tensor combine_rows(at::Tensor y, at::Tensor position,
                        c10::optional<at::Tensor> weights) {
  check_plan(position, "combine_rows");
  const int64_t rows = position.size(0), k = position.size(1);
  check_rows(y, position, rows * k, "combine_rows");
  const float* wp = weights_ptr(weights, position, "combine_rows");
  c10::DeviceGuard guard(y.device());
  auto yc = row_contiguous(y);
  const int64_t D = y.size(1);
  auto out = at::empty({rows, D}, y.options());
  if (out.numel() == 0) return out;
  DOA_FLOAT_TYPES(y.scalar_type(), "combine_rows", [&] {
    const int vec = row_vec(yc.data_ptr(), D, yc.stride(0), sizeof(T));
    const int sh = row_shift(ceil_div(D, vec));
    DOA_ROW_VEC(vec, [&] {
      hipLaunchKernelGGL((combine_rows_kernel<T, V>),
                         dim3(grid_for(rows << sh, 256, 1 << 20)), dim3(256), 0,
                         stream_of_current(), (const T*)yc.data_ptr(),
                         yc.stride(0), position.data_ptr<int>(), wp,
                         (T*)out.data_ptr(), rows, (int)k, (int)D, sh);
    });
  });
  DOA_CHECK_HIP(hipGetLastError());
  return out;
}

std::tuple<at::Tensor, at::Tensor> combine_rows_bwd(
    at::Tensor gout, c10::optional<at::Tensor> y, at::Tensor position,
    at::Tensor offsets, c10::optional<at::Tensor> weights, bool want_y) {
  check_plan(position, offsets, "combine_rows");
  const int64_t rows = position.size(0), k = position.size(1);
  const bool want_w = y.has_value();
  check_rows(gout, position, rows, "combine_rows");
  at::Tensor yc;
  if (want_w) {
    check_rows(*y, position, rows * k, "combine_rows");
    TORCH_CHECK(gout.scalar_type() == y->scalar_type() &&
                    gout.size(1) == y->size(1),
                "combine_rows: the gradient's rows differ from the rows");
    yc = row_contiguous(*y);
  }
  const float* wp = weights_ptr(weights, position, "combine_rows");
  c10::DeviceGuard guard(gout.device());
  auto gc = row_contiguous(gout);
  const int64_t D = gout.size(1);
  at::Tensor dy, dw;
  if (want_y) dy = at::empty({rows * k, D}, gout.options());
  if (want_w) dw = at::empty({rows, k}, gout.options().dtype(at::kFloat));
  if (D == 0 && want_w) dw.zero_();
  if (rows * k * D == 0 || !(want_y || want_w)) return {dy, dw};
  DOA_FLOAT_TYPES(gout.scalar_type(), "combine_rows", [&] {
    int vec = row_vec(gc.data_ptr(), D, gc.stride(0), sizeof(T));
    if (want_w)
      vec = std::min(vec, row_vec(yc.data_ptr(), D, yc.stride(0), sizeof(T)));
    const int sh = row_shift(ceil_div(D, vec));
    DOA_ROW_VEC(vec, [&] {
      hipLaunchKernelGGL((combine_rows_bwd_kernel<T, V>),
                         dim3(grid_for(rows << sh, 256, 1 << 20)), dim3(256), 0,
                         stream_of_current(), (const T*)gc.data_ptr(),
                         gc.stride(0),
                         want_w ? (const T*)yc.data_ptr() : nullptr,
                         want_w ? yc.stride(0) : 0, position.data_ptr<int>(),
                         offsets.data_ptr<int64_t>() + offsets.numel() - 1, wp,
                         want_y ? (T*)dy.data_ptr() : nullptr,
                         want_w ? dw.data_ptr<float>() : nullptr, rows, (int)k,
                         (int)D, sh);
    });
  });
  DOA_CHECK_HIP(hipGetLastError());
  return {dy, dw};
}

}  // namespace doa
