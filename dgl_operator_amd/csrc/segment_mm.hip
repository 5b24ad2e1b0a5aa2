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

// --- tiles in LDS -----------------------------------------------------------
// A step covers BK = 128 bytes of depth. An operand whose depth is contiguous
// ("row" tiles, [rows][BK]) is read as it is: lane l takes the 16 bytes of row
// l & 15 at depth (l >> 4) * 16 bytes. One whose depth is the outer index
// ("col" tiles, [BK][cols]) is read through the transposing LDS read: within 16
// lanes, lane s gives the address of 4 columns at depth s >> 2, and lane i gets
// column i at the 4 depths. Both come out as 8 halves (4 floats) of one row at
// depths (l >> 4) * 8 .. + 8, what the matrix instruction wants.
//
// 16-byte chunks are swizzled so that neither read meets a bank twice: row
// tiles by key(r) = (r ^ r >> 3) & 7 over the row's 8 chunks, col tiles by the
// depth over 32 bytes (halves, two depth quads a read) or 64 (floats).

constexpr int kStepBytes = 128;

template <typename T, bool COL, int CHUNKS>
__device__ inline int swizzle(int chunk, int outer) {
  if constexpr (!COL) return chunk ^ ((outer ^ (outer >> 3)) & 7);
  if constexpr (sizeof(T) == 2 && CHUNKS >= 16)
    return chunk ^ (((outer & 3) | ((outer >> 1) & 4)) << 1);
  if constexpr (sizeof(T) == 2)
    return chunk ^ (((outer ^ (outer >> 3)) & 1) << 1 | (outer & 2) << 1);
  return chunk ^ (((outer >> 2) & 3) << 2);
}

// one operand's tile: SIDE rows (or columns) by BK of depth
template <typename T, bool COL, int SIDE, int THREADS>
struct Tile {
  static constexpr int E = 16 / sizeof(T);                  // a chunk
  static constexpr int BK = kStepBytes / sizeof(T);
  static constexpr int CHUNKS = COL ? SIDE / E : BK / E;    // an outer index
  static constexpr int BYTES = SIDE * kStepBytes;
  static constexpr int PER = BYTES / 16 / THREADS;          // chunks a thread
  static_assert(PER * THREADS * 16 == BYTES, "tile and threads do not match");
  static_assert(!COL || CHUNKS >= (sizeof(T) == 2 ? 8 : 16), "swizzle");

  // Where the thread's chunks lie from the tile's corner, in bytes; kOut for
  // those beyond the `side` rows there are.
  static constexpr uint32_t kOut = 0x80000000u;
  static __device__ void place(int64_t ld, int side, uint32_t* at) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int id = i * THREADS + threadIdx.x, o = id / CHUNKS;
      const int c = swizzle<T, COL, CHUNKS>(id % CHUNKS, o) * E;
      at[i] = (COL ? c : o) < side ? (uint32_t)((o * ld + c) * sizeof(T)) : kOut;
    }
  }
  // Whole aligned chunks straight to LDS; those beyond the operand are out of
  // the buffer's range and arrive as zeros. Written out because the compiler
  // orders every transposing LDS read behind all such loads in flight; here
  // only the wait before the barrier that publishes the step does.
  static __device__ void load(const T* p, const uint32_t* at, int64_t depth,
                              char* lds) {
    const uint64_t base = reinterpret_cast<uint64_t>(p);
    const Chunk rsrc = {
        (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)base),
        (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(base >> 32)) & 0xffffu,
        0x7fffffffu, 0x00020000u};
    // the wave's part of the tile: 64 chunks in a row
    const uint32_t to = __builtin_amdgcn_readfirstlane(
        (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds +
        (threadIdx.x >> 6) * 1024);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      uint32_t v = at[i];
      if (depth < BK) {
        const int id = i * THREADS + threadIdx.x, o = id / CHUNKS;
        const int k = COL ? o : swizzle<T, COL, CHUNKS>(id % CHUNKS, o) * E;
        if (k >= depth) v = kOut;
      }
      asm volatile(
          "s_mov_b32 m0, %0\n\t"
          "s_nop 0\n\t"
          "buffer_load_dwordx4 %1, %2, 0 offen lds"
          :
          : "s"(to + i * THREADS * 16), "v"(v), "s"(rsrc)
          : "memory", "m0");
    }
  }
  // the same through registers, element by element where a chunk is cut
  static __device__ void fetch(const T* p, int64_t ld, int side, int64_t depth,
                               Chunk* to) {
    const int O = COL ? (int)min((int64_t)BK, depth) : side;
    const int I = COL ? side : (int)min((int64_t)BK, depth);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int id = i * THREADS + threadIdx.x, o = id / CHUNKS;
      const int c = swizzle<T, COL, CHUNKS>(id % CHUNKS, o) * E;
      const T* src = p + o * ld + c;
      union { Chunk q; T v[E]; } u;
      u.q = Chunk{0, 0, 0, 0};
      if (o < O && c + E <= I) {
        u.q = *reinterpret_cast<const LooseChunk*>(src);
      } else if (o < O) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c + e < I) u.v[e] = src[e];
      }
      to[i] = u.q;
    }
  }
  static __device__ void put(const Chunk* from, char* lds) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      *reinterpret_cast<Chunk*>(lds + (i * THREADS + threadIdx.x) * 16) = from[i];
  }

  // the 16 x (4 E) fragment of rows s0.. at depth chunk step kk (0, 1)
  using Frag = __attribute__((__vector_size__(16))) T;
  static __device__ Frag frag(const char* lds, int s0, int kk) {
    const int lane = threadIdx.x & 63, q = lane >> 4, s = lane & 15;
    if constexpr (!COL) {
      const int r = s0 + s;
      return *reinterpret_cast<const Frag*>(
          lds + r * kStepBytes + swizzle<T, false, CHUNKS>(kk * 4 + q, r) * 16);
    } else if constexpr (sizeof(T) == 2) {
      using S4 = short __attribute__((ext_vector_type(4)));
      const int col = s0 + (s & 3) * 4;
      union { S4 h[2]; Frag f; } u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = kk * 32 + q * 8 + h * 4 + (s >> 2);
        const char* a = lds + k * (SIDE * 2) +
                        swizzle<T, true, CHUNKS>(col / 8, k) * 16 + (col & 4) * 2;
        u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) S4*)a);
      }
      return u.f;
    } else {
      Frag f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = kk * 16 + q * 4 + i, col = s0 + s;
        f[i] = *reinterpret_cast<const T*>(
            lds + k * (SIDE * 4) + swizzle<T, true, CHUNKS>(col / 4, k) * 16 +
            (col & 3) * 4);
      }
      return f;
    }
  }
};

template <typename T, typename Frag>
__device__ inline f32x4 mma(Frag a, Frag b, f32x4 c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  } else if constexpr (std::is_same_v<T, __bf16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
}

// four neighbours at once, at any element unless ALIGNED
template <bool ALIGNED, typename O>
__device__ inline void store4(O* p, const Vec<O, 4>& v) {
  using U = uint32_t __attribute__((ext_vector_type(sizeof(O))));
  typedef U L __attribute__((aligned(sizeof(O))));
  using P = std::conditional_t<ALIGNED, U, L>;
  *reinterpret_cast<P*>(p) = __builtin_bit_cast(U, v);
}

// c[m][n] = sum_k a(m, k) b(k, n) for one tile of BM x BN. AC, BC: that
// operand's depth is its outer index. WM x WN waves. WHOLE: every row of both
// starts on 16 bytes and is whole chunks long.
template <typename T, typename O, bool AC, bool BC, bool WHOLE, int BM, int BN,
          int WM, int WN>
__device__ inline void tile_product(const T* a, int64_t lda, int M, const T* b,
                                    int64_t ldb, int N, int64_t K, O* c,
                                    int64_t ldc) {
  constexpr int THREADS = 64 * WM * WN;
  using TA = Tile<T, AC, BM, THREADS>;
  using TB = Tile<T, BC, BN, THREADS>;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int BK = TA::BK;
  __shared__ __align__(16) char lds[2][TA::BYTES + TB::BYTES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  f32x4 acc[FM][FN] = {};
  const int64_t step_a = AC ? BK * lda : BK, step_b = BC ? BK * ldb : BK;
  auto multiply = [&](const char* la, const char* lb) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      typename TA::Frag fa[FM];
      typename TB::Frag fb[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[i] = TA::frag(la, wm + i * 16, kk);
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[j] = TB::frag(lb, wn + j * 16, kk);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          // b first: a lane then holds 4 neighbouring columns of one row
          acc[i][j] = mma<T>(fb[j], fa[i], acc[i][j]);
    }
  };
  int now = 0;
  if constexpr (WHOLE) {
    uint32_t pa[TA::PER], pb[TB::PER];
    TA::place(lda, M, pa);
    TB::place(ldb, N, pb);
    if (K > 0) {
      TA::load(a, pa, K, lds[0]);
      TB::load(b, pb, K, lds[0] + TA::BYTES);
    }
    for (int64_t left = K; left > 0; left -= BK, now ^= 1) {
      // this step has arrived, and the last one's readers are done
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (left > BK) {  // the next step travels while this one multiplies
        a += step_a;
        b += step_b;
        TA::load(a, pa, left - BK, lds[now ^ 1]);
        TB::load(b, pb, left - BK, lds[now ^ 1] + TA::BYTES);
      }
      multiply(lds[now], lds[now] + TA::BYTES);
    }
  } else {
    Chunk ra[TA::PER], rb[TB::PER];
    if (K > 0) {
      TA::fetch(a, lda, M, K, ra);
      TB::fetch(b, ldb, N, K, rb);
      TA::put(ra, lds[0]);
      TB::put(rb, lds[0] + TA::BYTES);
    }
    for (int64_t left = K; left > 0; left -= BK, now ^= 1) {
      __syncthreads();
      if (left > BK) {
        a += step_a;
        b += step_b;
        TA::fetch(a, lda, M, left - BK, ra);
        TB::fetch(b, ldb, N, left - BK, rb);
      }
      multiply(lds[now], lds[now] + TA::BYTES);
      if (left > BK) {
        TA::put(ra, lds[now ^ 1]);
        TB::put(rb, lds[now ^ 1] + TA::BYTES);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = wm + i * 16 + (lane & 15);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = wn + j * 16 + (lane >> 4) * 4;
      if (m >= M) continue;
      Vec<O, 4> o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o.v[r] = (O)acc[i][j][r];
      if constexpr (WHOLE) {
        if (n < N) store4<true>(c + m * ldc + n, o);
      } else if (n + 4 <= N) {
        store4<false>(c + m * ldc + n, o);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < N) c[m * ldc + n + r] = o.v[r];
      }
    }
  }
}

__device__ inline int64_t offset_at(const int64_t* offsets, int g,
                                    int64_t rows) {
  const int64_t o = offsets[g];
  return o < 0 ? 0 : o > rows ? rows : o;  // never outside the rows
}

// blocks go round robin over the 8 XCDs: neighbours in the work's order share
// an XCD's L2 when block b does the work (b % 8) * (blocks / 8) + b / 8
__device__ inline int64_t xcd_order(int64_t b, int64_t blocks) {
  const int64_t whole = blocks >> 3;
  return (b >> 3) < whole ? (b & 7) * whole + (b >> 3) : b;
}

template <typename T, bool WC, bool WHOLE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void segment_mm_kernel(
    const T* __restrict__ x, int64_t xs, const T* __restrict__ w, int64_t wg,
    int64_t wl, const int64_t* __restrict__ offsets, T* __restrict__ y,
    int64_t rows, int G, int K, int N, int tiles_n) {
  // rows of no group
  const int64_t first = offset_at(offsets, 0, rows);
  const int64_t end = max(first, offset_at(offsets, G, rows));
  const int64_t outside = (first + rows - end) * N;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < outside;
       i += (int64_t)gridDim.x * blockDim.x)
    y[i < first * N ? i : i + (end - first) * N] = (T)0.f;
  const int64_t work = xcd_order(blockIdx.x, gridDim.x);
  const int64_t v = work / tiles_n;
  int lo = 0, hi = G;  // the last g with start(g) <= v
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offset_at(offsets, mid, rows) / BM + mid <= v) lo = mid; else hi = mid;
  }
  const int64_t begin = offset_at(offsets, lo, rows);
  const int64_t r0 = begin + (v - begin / BM - lo) * BM;
  const int64_t stop = offset_at(offsets, lo + 1, rows);
  if (r0 < begin || r0 >= stop) return;
  const int n0 = (int)(work % tiles_n) * BN;
  tile_product<T, T, false, WC, WHOLE, BM, BN, WM, WN>(
      x + r0 * xs, xs, (int)min((int64_t)BM, stop - r0),
      w + lo * wg + n0 * (WC ? 1 : wl), wl, min(BN, N - n0), K,
      y + r0 * N + n0, N);
}

// dW tiles; the group's rows in `splits` parts, each to its own plane of `out`
template <typename T, typename O, bool WHOLE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void segment_mm_wgrad_kernel(
    const T* __restrict__ x, int64_t xs, const T* __restrict__ g, int64_t gs,
    const int64_t* __restrict__ offsets, O* __restrict__ out, int64_t rows,
    int G, int K, int N, int tiles_k, int tiles_n, int splits) {
  int64_t work = xcd_order(blockIdx.x, gridDim.x);
  const int n0 = (int)(work % tiles_n) * BN;
  work /= tiles_n;
  const int k0 = (int)(work % tiles_k) * BM;
  work /= tiles_k;
  const int part = (int)(work % splits);
  const int e = (int)(work / splits);
  const int64_t begin = offset_at(offsets, e, rows);
  const int64_t len = max((int64_t)0, offset_at(offsets, e + 1, rows) - begin);
  constexpr int BK = kStepBytes / sizeof(T);
  const int64_t each = (len + (int64_t)splits * BK - 1) / (splits * BK) * BK;
  const int64_t from = min(len, part * each), to = min(len, from + each);
  tile_product<T, O, true, true, WHOLE, BM, BN, WM, WN>(
      x + (begin + from) * xs + k0, xs, min(BM, K - k0),
      g + (begin + from) * gs + n0, gs, min(BN, N - n0), to - from,
      out + (((int64_t)part * G + e) * K + k0) * N + n0, N);
}

// the parts' sum, in their order
template <typename T>
__global__ __launch_bounds__(256) void sum_parts_kernel(
    const float* __restrict__ parts, T* __restrict__ out, int64_t n,
    int splits) {
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n;
       i += (int64_t)gridDim.x * 1024) {
    if (i + 4 <= n) {
      float s[4] = {};
      for (int p = 0; p < splits; ++p) {
        union { Chunk q; float v[4]; } u;
        u.q = *reinterpret_cast<const LooseChunk*>(parts + p * n + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += u.v[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) out[i + e] = (T)s[e];
    } else {
      for (int64_t j = i; j < n; ++j) {
        float s = 0.f;
        for (int p = 0; p < splits; ++p) s += parts[p * n + j];
        out[j] = (T)s;
      }
    }
  }
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

// whether a tile of rows can be read in whole aligned chunks, from byte offsets
// below 2^31
template <typename T>
static bool whole_rows(const at::Tensor& t, int64_t width) {
  constexpr int E = 16 / sizeof(T);
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
         width % E == 0 && t.stride(0) % E == 0 && t.stride(0) < (1 << 20);
}
template <typename T>
static bool whole_weight(const at::Tensor& w, int64_t outer) {
  constexpr int E = 16 / sizeof(T);
  return reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0 &&
         outer % E == 0 && w.stride(0) % E == 0 && outer < (1 << 20);
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
  auto wt = transposed ? weight.transpose(1, 2) : weight;
  const int64_t K = wt.size(1), N = wt.size(2);
  TORCH_CHECK(x.size(1) == K, "segment_mm: rows of ", K, " expected, got ",
              x.size(1));
  TORCH_CHECK(K < (1 << 30) && N < (1 << 30), "segment_mm: too wide");
  c10::DeviceGuard guard(x.device());
  auto xc = mm_rows(x);
  const int64_t R = x.size(0);
  auto y = at::empty({R, N}, x.options());
  if (R * N == 0) return y;
  // one of the weight's two inner strides has to be 1
  const bool n_inner = N <= 1 ? wt.stride(1) != 1 || K <= 1 : wt.stride(2) == 1;
  if (!n_inner && !(K <= 1 || wt.stride(1) == 1)) wt = wt.contiguous();
  const bool wc = N <= 1 ? n_inner : wt.stride(2) == 1;
  const int64_t wl = wt.stride(wc ? 1 : 2);
  DOA_FLOAT_TYPES(x.scalar_type(), "segment_mm", [&] {
    auto go = [&](auto kernel, int BM, int BN, int threads) {
      const int64_t tn = ceil_div(N, BN), blocks = (R / BM + G) * tn;
      TORCH_CHECK(blocks < INT32_MAX, "segment_mm: too many tiles");
      hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0,
                         stream_of_current(), (const T*)xc.data_ptr(),
                         xc.stride(0), (const T*)wt.data_ptr(), wt.stride(0),
                         wl, offsets.data_ptr<int64_t>(), (T*)y.data_ptr(), R,
                         (int)G, (int)K, (int)N, (int)tn);
    };
    // whole aligned chunks of 16 bytes go straight to LDS
    const bool whole = whole_rows<T>(xc, K) && N % (16 / sizeof(T)) == 0 &&
                       K % (16 / sizeof(T)) == 0 && whole_weight<T>(wt, wl);
    auto pick = [&](auto wcv, auto wv) {
      constexpr bool WC = decltype(wcv)::value, W = decltype(wv)::value;
      // few rows a group: a tile of 32 rows leaves less of it empty and reads
      // the weights over more blocks
      if (R <= 48 * G)
        go(segment_mm_kernel<T, WC, W, 32, 64, 1, 4>, 32, 64, 256);
      else
        go(segment_mm_kernel<T, WC, W, 128, 128, 2, 2>, 128, 128, 256);
    };
    if (wc)
      whole ? pick(std::true_type{}, std::true_type{})
            : pick(std::true_type{}, std::false_type{});
    else
      whole ? pick(std::false_type{}, std::true_type{})
            : pick(std::false_type{}, std::false_type{});
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
  TORCH_CHECK(x.size(1) < (1 << 30) && grad.size(1) < (1 << 30),
              "segment_mm: too wide");
  c10::DeviceGuard guard(x.device());
  auto xc = mm_rows(x);
  auto gc = mm_rows(grad);
  const int64_t K = x.size(1), N = grad.size(1), R = x.size(0);
  auto dw = at::empty({G, K, N}, x.options());
  if (dw.numel() == 0) return dw;
  constexpr int B = 128;
  const int64_t tk = ceil_div(K, B), tn = ceil_div(N, B), tiles = G * tk * tn;
  // few tiles over long groups: parts of at least 512 rows, about 1024 blocks
  const int64_t splits = std::max<int64_t>(
      1, std::min<int64_t>({ceil_div(1024, tiles), R / G / 512, 64}));
  TORCH_CHECK(tiles * splits < INT32_MAX, "segment_mm: too many tiles");
  DOA_FLOAT_TYPES(x.scalar_type(), "segment_mm", [&] {
    const bool whole = whole_rows<T>(xc, K) && whole_rows<T>(gc, N);
    auto go = [&](auto* out) {
      using O = std::remove_pointer_t<decltype(out)>;
      auto kernel = whole ? segment_mm_wgrad_kernel<T, O, true, B, B, 2, 2>
                          : segment_mm_wgrad_kernel<T, O, false, B, B, 2, 2>;
      hipLaunchKernelGGL(kernel, dim3(tiles * splits), dim3(256), 0,
                         stream_of_current(), (const T*)xc.data_ptr(),
                         xc.stride(0), (const T*)gc.data_ptr(), gc.stride(0),
                         offsets.data_ptr<int64_t>(), out, R, (int)G, (int)K,
                         (int)N, (int)tk, (int)tn, (int)splits);
    };
    if (splits == 1) {
      go((T*)dw.data_ptr());
    } else {
      auto parts = at::empty({splits * dw.numel()},
                             x.options().dtype(at::kFloat));
      go(parts.data_ptr<float>());
      hipLaunchKernelGGL((sum_parts_kernel<T>),
                         dim3(grid_for(ceil_div(dw.numel(), 4), 256, 8192)),
                         dim3(256), 0, stream_of_current(),
                         parts.data_ptr<float>(), (T*)dw.data_ptr(),
                         dw.numel(), (int)splits);
    }
  });
  DOA_CHECK_HIP(hipGetLastError());
  return dw;
}

}  // namespace doa
