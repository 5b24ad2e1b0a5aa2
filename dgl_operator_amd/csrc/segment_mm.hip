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
//
// Measured on one MI355X (a large copy 4.8 TB/s, a large bf16 product 1230 and
// fp32 153 TFLOP/s), each product by itself, ten calls back to back:
//   262144 rows, 8 x 512 x 1024, bf16   y 339, dx 304, dW 278 us (0.81, 0.90, 0.99
//       PFLOP/s; the first calls after a pause 390, 360, 326). The matrix
//       instructions alone take 196 us, the loads alone 189; 537 MB of y to
//       write, and L2, keep the two from hiding each other whole. One weight for
//       all rows in the library: y 358, dx 236 us.
//   65536 rows, 1345 x 400 x 400, bf16   133, 142, 177 us: 430 MB of weights to
//       read or write each time, 112 us of copying.
//   53504 rows, 16 x 100 x 256, fp32    39, 41, 49 us against 18 of matrix rate;
//       partial tiles (100 of 112, groups' last rows) are a fifth, the first
//       loads and the last blocks of so short a kernel most of the rest.
//   186248 rows, 415 x 618 x 19, bf16 (unaligned)   106, 57, 147 us against 52 of
//       copying: through registers, one step ahead.
//   16 rows, 8 x 256 x 512, bf16   5 us, a few rows a group: latency.

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
// tiles by (r >> 1) & 7 over a row's 8 chunks, or -(r >> 2) & 3 over 4 (16 lanes
// of a 16-byte read meet in rows 0-3, 12-15 of one depth and 4-11 of the next),
// col tiles by the depth over 32 bytes (halves, two depth quads a read) or 64
// (floats).

constexpr int kStepBytes = 128;

template <typename T, bool COL, int CHUNKS>
__device__ inline int swizzle(int chunk, int outer) {
  if constexpr (!COL && CHUNKS == 4) return chunk ^ (-(outer >> 2) & 3);
  if constexpr (!COL) return chunk ^ ((outer >> 1) & 7);
  if constexpr (sizeof(T) == 2 && CHUNKS >= 16)
    return chunk ^ (((outer & 3) | ((outer >> 1) & 4)) << 1);
  if constexpr (sizeof(T) == 2)
    return chunk ^ (((outer ^ (outer >> 3)) & 1) << 1 | (outer & 2) << 1);
  return chunk ^ (((outer >> 2) & 3) << 2);
}

// the thread's index, in a way that what depends on it is computed where it is
// used: kept across a loop it would cost the accumulators their registers
__device__ inline int thread_here() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// one operand's tile: SIDE rows (or columns) by BK of depth
template <typename T, bool COL, int SIDE, int THREADS, int STEP = kStepBytes>
struct Tile {
  static constexpr int E = 16 / sizeof(T);                  // a chunk
  static constexpr int BK = STEP / sizeof(T);
  static constexpr int CHUNKS = COL ? SIDE / E : BK / E;    // an outer index
  static constexpr int BYTES = SIDE * STEP;
  static constexpr int PER = BYTES / 16 / THREADS;          // chunks a thread
  static_assert(PER * THREADS * 16 == BYTES, "tile and threads do not match");
  static_assert(!COL || CHUNKS >= (sizeof(T) == 2 ? 8 : 16), "swizzle");

  // Where the thread's chunks lie from the tile's corner, in bytes; kOut for
  // those beyond the `side` rows there are.
  static constexpr uint32_t kOut = 0x80000000u;
  static __device__ void place(int64_t ld, int side, uint32_t* at) {
    const int thread = thread_here();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int id = i * THREADS + thread, o = id / CHUNKS;
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
    auto issue = [&](int i, uint32_t v) {
      asm volatile(
          "s_mov_b32 m0, %0\n\t"
          "s_nop 0\n\t"
          "buffer_load_dwordx4 %1, %2, 0 offen lds"
          :
          : "s"(to + i * THREADS * 16), "v"(v), "s"(rsrc)
          : "memory", "m0");
    };
    if (depth >= BK) {
#pragma unroll
      for (int i = 0; i < PER; ++i) issue(i, at[i]);
    } else {
      const int thread = thread_here();
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int id = i * THREADS + thread, o = id / CHUNKS;
        const int k = COL ? o : swizzle<T, COL, CHUNKS>(id % CHUNKS, o) * E;
        issue(i, k < depth ? at[i] : kOut);
      }
    }
  }
  // The same through registers, from any element's address: a chunk that the
  // operand's edge cuts is read whole and masked, unless that would leave its
  // memory, which ends at `end`.
  static __device__ void fetch(const T* p, int64_t ld, int side, int64_t depth,
                               const T* end, Chunk* to) {
    const int O = COL ? (int)min((int64_t)BK, depth) : side;
    const int I = COL ? side : (int)min((int64_t)BK, depth);
    using Bits = std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t>;
    constexpr int W = 4 / sizeof(T);  // elements a word
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int id = i * THREADS + threadIdx.x, o = id / CHUNKS;
      const int c = swizzle<T, COL, CHUNKS>(id % CHUNKS, o) * E;
      const int there = o < O ? I - c : 0;  // elements of the chunk there are
      const T* src = p + o * ld + c;
      Chunk q = {0, 0, 0, 0};
      if (there > 0) {
        if (src + E <= end) {
          q = *reinterpret_cast<const LooseChunk*>(src);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (e < there)
              q[e / W] |= (uint32_t)reinterpret_cast<const Bits*>(src)[e]
                          << (e % W * 16);
        }
        if (there < E) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int in = there - w * W;  // of this word
            q[w] &= in >= W ? ~0u : in == 1 && W == 2 ? 0xffffu : 0u;
          }
        }
      }
      to[i] = q;
    }
  }
  static __device__ void put(const Chunk* from, char* lds) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      *reinterpret_cast<Chunk*>(lds + (i * THREADS + threadIdx.x) * 16) = from[i];
  }

  // A wave's F fragments: 16 rows each from row s0 on, 4 E of depth at step kk.
  // A row tile's swizzle is the same 16 rows further on, a col tile's is not.
  using Frag = __attribute__((__vector_size__(16))) T;
  template <int F>
  struct Reader {
    int at[COL ? F : 1];
    __device__ explicit Reader(int s0) {
      const int lane = threadIdx.x & 63, q = lane >> 4, s = lane & 15;
      if constexpr (!COL) {
        at[0] = (s0 + s) * STEP + swizzle<T, false, CHUNKS>(q, s0 + s) * 16;
      } else {
        // halves: 4 columns at depth q * 8 + (s >> 2); floats: column s at q * 4
        const int k = sizeof(T) == 2 ? q * 8 + (s >> 2) : q * 4;
        const int off = sizeof(T) == 2 ? (s & 3) * 4 : s;
#pragma unroll
        for (int f = 0; f < F; ++f) {
          const int col = s0 + f * 16 + off;
          at[f] = k * (SIDE * (int)sizeof(T)) +
                  swizzle<T, true, CHUNKS>(col / E, k) * 16 +
                  col % E * (int)sizeof(T);
        }
      }
    }
    __device__ Frag get(const char* lds, int f, int kk) const {
      if constexpr (!COL) {
        return *reinterpret_cast<const Frag*>(
            lds + (at[0] ^ (kk * 64)) + f * 16 * STEP);
      } else if constexpr (sizeof(T) == 2) {
        using S4 = short __attribute__((ext_vector_type(4)));
        union { S4 h[2]; Frag f; } u;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) S4*)(
                  lds + at[f] + (kk * 32 + h * 4) * (SIDE * 2)));
        return u.f;
      } else {
        Frag r;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          r[i] = *reinterpret_cast<const T*>(
              lds + at[f] + (kk * 16 + i) * (SIDE * 4));
        return r;
      }
    }
  };
};

template <typename T, typename Frag>
__device__ inline f32x4 mma(Frag a, Frag b, f32x4 c, int q = 0) {
  if constexpr (sizeof(T) == 4)
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a[q], b[q], c, 0, 0, 0);
  else if constexpr (std::is_same_v<T, __bf16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A wave's 16 FM x 16 FN results: strips of 16 rows go through `room` (ROOM
// bytes of LDS, the wave's own) and out in whole lines of its columns; a row is
// padded by 16 bytes to keep the strip's writes off one bank.
template <typename T, typename O, bool WHOLE, int FM, int FN, int ROOM>
__device__ inline void store_tile(const f32x4 (&acc)[FM][FN], char* room, O* c,
                                  int64_t ldc, int M, int N) {
  constexpr int E = 16 / sizeof(O), ROW = FN * 16 * sizeof(O) + 16;
  constexpr int CHUNKS = FN * 16 / E;
  constexpr int FIT = ROOM / (16 * ROW), STRIPS = FIT < FM ? FIT : FM;
  static_assert(STRIPS >= 1, "no room for a strip");
#pragma unroll
  for (int i0 = 0; i0 < FM; i0 += STRIPS) {
    wave_sync();  // the last strips are out
    __builtin_amdgcn_sched_barrier(0);
    const int lane = thread_here() & 63;
#pragma unroll
    for (int i = i0; i < FM && i < i0 + STRIPS; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        Vec<O, 4> o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o.v[r] = (O)acc[i][j][r];
        *reinterpret_cast<Vec<O, 4>*>(
            room + ((i - i0) * 16 + (lane & 15)) * ROW +
            (j * 16 + (lane >> 4) * 4) * sizeof(O)) = o;
      }
    wave_sync();
#pragma unroll
    for (int i = i0; i < FM && i < i0 + STRIPS; ++i)
#pragma unroll
      for (int at = lane; at < 16 * CHUNKS; at += 64) {
        const int r = at / CHUNKS, n = at % CHUNKS * E, m = i * 16 + r;
        if (m >= M || n >= N) continue;
        union { Chunk q; O v[E]; } u;
        u.q = *reinterpret_cast<const Chunk*>(
            room + ((i - i0) * 16 + r) * ROW + at % CHUNKS * 16);
        O* to = c + m * ldc + n;
        if (n + E <= N) {
          if constexpr (WHOLE) *reinterpret_cast<Chunk*>(to) = u.q;
          else *reinterpret_cast<LooseChunk*>(to) = u.q;
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (n + e < N) to[e] = u.v[e];
        }
      }
  }
}

// two stages of both operands
constexpr int lds_bytes(int BM, int BN, int STEP) { return 2 * (BM + BN) * STEP; }

// c[m][n] = sum_k a(m, k) b(k, n) for one tile of BM x BN. AC, BC: that
// operand's depth is its outer index. WM x WN waves. WHOLE: every row of both
// starts on 16 bytes and is whole chunks long.
template <typename T, typename O, bool AC, bool BC, bool WHOLE, int BM, int BN,
          int WM, int WN, int STEP>
__device__ inline void tile_product(char* lds, const T* a, int64_t lda, int M,
                                    const T* end_a, const T* b, int64_t ldb,
                                    int N, const T* end_b, int64_t K, O* c,
                                    int64_t ldc) {
  constexpr int THREADS = 64 * WM * WN;
  using TA = Tile<T, AC, BM, THREADS, STEP>;
  using TB = Tile<T, BC, BN, THREADS, STEP>;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int BK = TA::BK;
  constexpr int STAGE = TA::BYTES + TB::BYTES;
  static_assert(2 * STAGE == lds_bytes(BM, BN, STEP), "LDS");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const typename TA::template Reader<FM> read_a(wm);
  const typename TB::template Reader<FN> read_b(wn);
  f32x4 acc[FM][FN] = {};
  const int64_t step_a = AC ? BK * lda : BK, step_b = BC ? BK * ldb : BK;
  auto multiply = [&](const char* la, const char* lb, int64_t left) {
#pragma unroll
    for (int kk = 0; kk < STEP / 64; ++kk) {
      // fp32's matrix rate is worth a branch around zeros
      if (sizeof(T) == 4 && kk && left <= BK / 2) continue;
      typename TA::Frag fa[FM];
      typename TB::Frag fb[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[i] = read_a.get(la, i, kk);
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[j] = read_b.get(lb, j, kk);
      // b first: a lane then holds 4 neighbouring columns of one row. fp32's
      // four instructions a fragment go round the tiles, not on one of them
#pragma unroll
      for (int q = 0; q < (sizeof(T) == 4 ? 4 : 1); ++q)
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j)
            acc[i][j] = mma<T>(fb[j], fa[i], acc[i][j], q);
    }
  };
  int now = 0;
  if constexpr (WHOLE) {
    uint32_t pa[TA::PER], pb[TB::PER];
    TA::place(lda, M, pa);
    TB::place(ldb, N, pb);
    if (K > 0) {
      TA::load(a, pa, K, lds);
      TB::load(b, pb, K, lds + TA::BYTES);
    }
    for (int64_t left = K; left > 0; left -= BK, now ^= 1) {
      // this step has arrived, and the last one's readers are done
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (left > BK) {  // the next step travels while this one multiplies
        a += step_a;
        b += step_b;
        TA::load(a, pa, left - BK, lds + (now ^ 1) * STAGE);
        TB::load(b, pb, left - BK, lds + (now ^ 1) * STAGE + TA::BYTES);
      }
      multiply(lds + now * STAGE, lds + now * STAGE + TA::BYTES, left);
    }
  } else {
    Chunk ra[TA::PER], rb[TB::PER];
    if (K > 0) {
      TA::fetch(a, lda, M, K, end_a, ra);
      TB::fetch(b, ldb, N, K, end_b, rb);
      TA::put(ra, lds);
      TB::put(rb, lds + TA::BYTES);
    }
    for (int64_t left = K; left > 0; left -= BK, now ^= 1) {
      __syncthreads();
      if (left > BK) {
        a += step_a;
        b += step_b;
        TA::fetch(a, lda, M, left - BK, end_a, ra);
        TB::fetch(b, ldb, N, left - BK, end_b, rb);
      }
      multiply(lds + now * STAGE, lds + now * STAGE + TA::BYTES, left);
      if (left > BK) {
        TA::put(ra, lds + (now ^ 1) * STAGE);
        TB::put(rb, lds + (now ^ 1) * STAGE + TA::BYTES);
      }
    }
  }
  __syncthreads();  // every wave is done with the tiles
  constexpr int ROOM = 2 * STAGE / (WM * WN);
  store_tile<T, O, WHOLE, FM, FN, ROOM>(acc, lds + wave * ROOM,
                                        c + wm * ldc + wn, ldc, M - wm, N - wn);
}

// offsets never change under a kernel: scalar loads, whatever it writes
using ConstOffsets = const __attribute__((address_space(4))) int64_t*;

__device__ inline int offset_at(ConstOffsets offsets, int g, int rows) {
  const int64_t o = offsets[g];
  return o < 0 ? 0 : o > rows ? rows : (int)o;  // never outside the rows
}

// the tile of rows at virtual tile v: its group, first row and rows (0: none)
struct Span {
  int g, r0, many;
};
template <int BM>
__device__ inline Span find_span(ConstOffsets offsets, int v, int rows, int G) {
  int lo = 0, hi = G;  // the last g with start(g) <= v
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offset_at(offsets, mid, rows) / BM + mid <= v) lo = mid; else hi = mid;
  }
  const int begin = offset_at(offsets, lo, rows);
  const int stop = offset_at(offsets, lo + 1, rows);
  const int64_t r0 = begin + (int64_t)(v - begin / BM - lo) * BM;
  if (r0 < begin || r0 >= stop) return {lo, 0, 0};
  return {lo, (int)r0, min(BM, stop - (int)r0)};
}

template <typename T>
__device__ inline void zero_outside(ConstOffsets offsets, T* y, int rows, int G,
                                    int N) {
  const int64_t first = offset_at(offsets, 0, rows);
  const int64_t end = max((int)first, offset_at(offsets, G, rows));
  const int64_t outside = (first + rows - end) * N;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < outside;
       i += (int64_t)gridDim.x * blockDim.x)
    y[i < first * N ? i : i + (end - first) * N] = (T)0.f;
}

// blocks go round robin over the 8 XCDs: neighbours in the work's order share
// an XCD's L2 when block b does the work (b % 8) * (blocks / 8) + b / 8
__device__ inline int64_t xcd_order(int64_t b, int64_t blocks) {
  const int64_t whole = blocks >> 3;
  return (b >> 3) < whole ? (b & 7) * whole + (b >> 3) : b;
}

template <typename T, bool WC, bool WHOLE, int BM, int BN, int WM, int WN,
          int STEP, int WAVES>
__global__ __launch_bounds__(64 * WM * WN, WAVES) void segment_mm_kernel(
    const T* __restrict__ x, int64_t xs, const T* __restrict__ w, int64_t wg,
    int64_t wl, ConstOffsets offsets, T* __restrict__ y, int rows, int G, int K,
    int N, int tiles_n) {
  zero_outside(offsets, y, rows, G, N);
  const int work = (int)xcd_order(blockIdx.x, gridDim.x);
  __shared__ __align__(16) char lds[lds_bytes(BM, BN, STEP)];
  const Span s = find_span<BM>(offsets, work / tiles_n, rows, G);
  if (s.many == 0) return;
  const int n0 = work % tiles_n * BN;
  tile_product<T, T, false, WC, WHOLE, BM, BN, WM, WN, STEP>(
      lds, x + s.r0 * xs, xs, s.many, x + (rows - 1) * xs + K,
      w + s.g * wg + n0 * (WC ? 1 : wl), wl, min(BN, N - n0),
      w + (G - 1) * wg + ((WC ? K : N) - 1) * wl + (WC ? N : K), K,
      y + (int64_t)s.r0 * N + n0, N);
}

// ---------------------------------------------------------------------------
// Many rows a group, 16-bit types: one block of 8 waves a CU walks over tiles of
// 256 x 256: a smaller tile asks more of L2 than it gives (128 x 128 is 64 bytes
// a clock and CU at the matrix rate; y 437 and dx 353 us in the run where this was
// 352 and 315). Steps of 64 bytes of depth go round a ring of 4 LDS stages: one is
// multiplied from registers while the next is read into them and three more are
// on their way; the loads run on into the next tile while this one's results go
// out.
// ---------------------------------------------------------------------------
template <typename T, bool WC>
__global__ __launch_bounds__(512) void segment_mm_wide_kernel(
    const T* __restrict__ x, int64_t xs, const T* __restrict__ w, int64_t wg,
    int64_t wl, ConstOffsets offsets, T* __restrict__ y, int rows, int G, int K,
    int N, int tiles_n, int tiles) {
  constexpr int B = 256, STEP = 64, STAGES = 4;
  using TA = Tile<T, false, B, 512, STEP>;
  using TB = Tile<T, WC, B, 512, STEP>;
  constexpr int STAGE = TA::BYTES + TB::BYTES, BK = TA::BK;
  constexpr int FM = 8, FN = 4, ROOM = 16 * (FN * 16 * sizeof(T) + 16);
  __shared__ __align__(16) char lds[STAGES * STAGE + 8 * ROOM];
  zero_outside(offsets, y, rows, G, N);
  // an XCD's blocks walk side by side over its own stretch of the tiles
  const int xcd = blockIdx.x & 7, t_step = gridDim.x >> 3;
  const int t_end = (int)((int64_t)tiles * (xcd + 1) / 8);
  auto next = [&](int t) {  // the first tile from t on that has rows
    while (t < t_end && find_span<B>(offsets, t / tiles_n, rows, G).many == 0)
      t += t_step;
    return t;
  };
  int use_t = next((int)((int64_t)tiles * xcd / 8) + (blockIdx.x >> 3));
  if (use_t >= t_end) return;
  int load_t = use_t, load_left = K;
  const T* a;
  const T* b;
  uint32_t pa[TA::PER], pb[TB::PER];
  auto enter = [&](int t) {
    const Span s = find_span<B>(offsets, t / tiles_n, rows, G);
    const int n0 = t % tiles_n * B;
    a = x + s.r0 * xs;
    b = w + s.g * wg + n0 * (WC ? 1 : wl);
    TA::place(xs, s.many, pa);
    TB::place(wl, min(B, N - n0), pb);
  };
  enter(load_t);
  const int64_t step_b = WC ? BK * wl : BK;
  auto ahead = [&](char* stage) {
    TA::load(a, pa, load_left, stage);
    TB::load(b, pb, load_left, stage + TA::BYTES);
    a += BK;
    b += step_b;
    load_left -= BK;
    if (load_left > 0) return;
    load_left = K;
    load_t = load_t < t_end ? next(load_t + t_step) : t_end;
    if (load_t < t_end) {
      enter(load_t);
    } else {
      // behind the last tile the loads go on out of range, so that a wait's
      // count always means the same
      TA::place(xs, 0, pa);
      TB::place(wl, 0, pb);
    }
  };
#pragma unroll 1
  for (int i = 0; i < STAGES; ++i) ahead(lds + i * STAGE);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / 4 * 128, wn = wave % 4 * 64;
  const typename TA::template Reader<FM> read_a(wm);
  const typename TB::template Reader<FN> read_b(wn);
  static_assert(TA::PER + TB::PER == 4, "the waits count loads");
  typename TA::Frag fa[FM];
  typename TB::Frag fb[FN];
  asm volatile("s_waitcnt vmcnt(12)\n\ts_barrier" ::: "memory");
#pragma unroll
  for (int j = 0; j < FN; ++j) fb[j] = read_b.get(lds + TA::BYTES, j, 0);
#pragma unroll
  for (int i = 0; i < FM; ++i) fa[i] = read_a.get(lds, i, 0);
  int stage = 0;
  while (use_t < t_end) {
    f32x4 acc[FM][FN] = {};
#pragma unroll 1
    for (int left = K; left > 0; left -= BK) {
      // The fragments of this step are in registers, the next stage has arrived
      // and two are on their way; every wave has read this stage, which the
      // loads may fill again. The next step's fragments replace this one's as
      // these are used up.
      asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      ahead(lds + stage * STAGE);
      stage = (stage + 1) & (STAGES - 1);
      const char* la = lds + stage * STAGE;
      typename TB::Frag nb[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) nb[j] = read_b.get(la + TA::BYTES, j, 0);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = mma<T>(fb[j], fa[i], acc[i][j]);
        fa[i] = read_a.get(la, i, 0);
      }
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[j] = nb[j];
    }
    const Span s = find_span<B>(offsets, use_t / tiles_n, rows, G);
    const int n0 = use_t % tiles_n * B;
    store_tile<T, T, true, FM, FN, ROOM>(
        acc, lds + STAGES * STAGE + wave * ROOM,
        y + (int64_t)(s.r0 + wm) * N + n0 + wn, N, s.many - wm, N - n0 - wn);
    use_t = next(use_t + t_step);
  }
  // nothing may still be on its way into LDS when the block ends
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// dW over many rows a group, 16-bit types, the same ring. The rows of all groups
// are dealt evenly to teams, a team being one block for each 256 x 256 tile of
// a group's dW (they read the same rows, on one XCD where they fit). A block
// walks over its team's rows; where they hold a whole group its product goes
// straight to dW, where they begin or end inside one it goes to the team's
// first or second fp32 plane, and sum_teams_kernel adds those up.
struct Team {
  int begin, each;  // the first row of all, rows a team
};
__device__ inline Team team_rows(ConstOffsets offsets, int rows, int G,
                                 int teams) {
  const int first = offset_at(offsets, 0, rows);
  const int all = max(0, offset_at(offsets, G, rows) - first);
  return {first, max(32, ((all + teams - 1) / teams + 31) & ~31)};
}

// the last group that starts at or before row r
__device__ inline int group_at(ConstOffsets offsets, int r, int rows, int G) {
  int lo = 0, hi = G;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offset_at(offsets, mid, rows) <= r) lo = mid; else hi = mid;
  }
  return lo;
}

template <typename T>
__global__ __launch_bounds__(512) void segment_wgrad_wide_kernel(
    const T* __restrict__ x, int64_t xs, const T* __restrict__ g, int64_t gs,
    ConstOffsets offsets, T* __restrict__ dw, float* __restrict__ planes,
    int rows, int G, int K, int N, int tiles_n, int tiles, int teams) {
  constexpr int B = 256, STEP = 64, STAGES = 4;
  using TT = Tile<T, true, B, 512, STEP>;
  constexpr int STAGE = 2 * TT::BYTES, BK = TT::BK;
  constexpr int FM = 8, FN = 4, ROOM = 16 * (FN * 16 * sizeof(T) + 16);
  __shared__ __align__(16) char lds[STAGES * STAGE + 8 * ROOM];
  const int id = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const int team = id / tiles, tile = id % tiles;
  if (team >= teams) return;
  const int k0 = tile / tiles_n * B, n0 = tile % tiles_n * B;
  const Team tr = team_rows(offsets, rows, G, teams);
  const int from = tr.begin + (int)min((int64_t)team * tr.each, (int64_t)rows);
  const int to = (int)min((int64_t)from + tr.each,
                          (int64_t)offset_at(offsets, G, rows));
  if (from >= to) return;
  auto stop_of = [&](int e) { return min(to, offset_at(offsets, e + 1, rows)); };
  // the group that holds row r >= its start: the first from e on that ends later
  auto group_of = [&](int e, int r) {
    while (e < G - 1 && offset_at(offsets, e + 1, rows) <= r) ++e;
    return e;
  };
  const int lo = group_at(offsets, from, rows, G);
  int use_g = lo, use_r = from, load_g = lo, load_r = from;
  int load_stop = max(from + 1, stop_of(lo));
  uint32_t pa[TT::PER], pb[TT::PER];
  TT::place(xs, min(B, K - k0), pa);
  TT::place(gs, min(B, N - n0), pb);
  auto ahead = [&](char* stage) {
    const int depth = load_stop - load_r;  // 0 behind the last row: no loads
    TT::load(x + load_r * xs + k0, pa, depth, stage);
    TT::load(g + load_r * gs + n0, pb, depth, stage + TT::BYTES);
    load_r = min(load_stop, load_r + BK);
    if (load_r < load_stop || load_r >= to) return;
    load_g = group_of(load_g, load_r);
    load_stop = max(load_r + 1, stop_of(load_g));
  };
#pragma unroll 1
  for (int i = 0; i < STAGES; ++i) ahead(lds + i * STAGE);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / 4 * 128, wn = wave % 4 * 64;
  const typename TT::template Reader<FM> read_a(wm);
  const typename TT::template Reader<FN> read_b(wn);
  static_assert(2 * TT::PER == 4, "the waits count loads");
  typename TT::Frag fa[FM], fb[FN];
  asm volatile("s_waitcnt vmcnt(12)\n\ts_barrier" ::: "memory");
#pragma unroll
  for (int j = 0; j < FN; ++j) fb[j] = read_b.get(lds + TT::BYTES, j, 0);
#pragma unroll
  for (int i = 0; i < FM; ++i) fa[i] = read_a.get(lds, i, 0);
  int stage = 0;
  while (use_r < to) {
    f32x4 acc[FM][FN] = {};
    const int start = use_r, stop = max(use_r + 1, stop_of(use_g));
#pragma unroll 1
    for (int left = stop - start; left > 0; left -= BK) {
      asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      ahead(lds + stage * STAGE);
      stage = (stage + 1) & (STAGES - 1);
      const char* la = lds + stage * STAGE;
      typename TT::Frag nb[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) nb[j] = read_b.get(la + TT::BYTES, j, 0);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = mma<T>(fb[j], fa[i], acc[i][j]);
        fa[i] = read_a.get(la, i, 0);
      }
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[j] = nb[j];
    }
    const int M = K - k0 - wm, W = N - n0 - wn;
    const int64_t corner = (int64_t)(k0 + wm) * N + n0 + wn;
    const int g_start = offset_at(offsets, use_g, rows);
    const int g_stop = offset_at(offsets, use_g + 1, rows);
    if (start == g_start && stop == g_stop) {
      store_tile<T, T, true, FM, FN, ROOM>(
          acc, lds + STAGES * STAGE + wave * ROOM,
          dw + (int64_t)use_g * K * N + corner, N, M, W);
    } else {
      // begun in an earlier team: the first plane, else the second
      float* c = planes + (2 * (int64_t)team + (start == g_start)) * K * N + corner;
      const int lane = thread_here() & 63;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int m = i * 16 + (lane & 15), n = j * 16 + (lane >> 4) * 4;
          if (m < M && n < W)
            *reinterpret_cast<f32x4*>(c + (int64_t)m * N + n) = acc[i][j];
        }
    }
    use_r = stop;
    if (use_r < to) use_g = group_of(use_g, use_r);
  }
  // nothing may still be on its way into LDS when the block ends
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// Groups that several teams hold, and empty ones. A block has 64 lanes of up to
// 4 elements; each of its 4 waves sums a quarter of the teams in their order,
// and the quarters are added in theirs.
template <typename T>
__global__ __launch_bounds__(256) void sum_teams_kernel(
    const float* __restrict__ planes, ConstOffsets offsets, T* __restrict__ dw,
    int rows, int G, int64_t n, int teams) {
  __shared__ f32x4 part[4][64];
  const Team tr = team_rows(offsets, rows, G, teams);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int e = blockIdx.y; e < G; e += gridDim.y) {
    const int b = offset_at(offsets, e, rows), s = offset_at(offsets, e + 1, rows);
    // (clamped for offsets that fall: the planes are never left)
    const int t0 = min(teams - 1, max(0, b - tr.begin) / tr.each);
    const int t1 = min(teams - 1, max(0, s - 1 - tr.begin) / tr.each);
    if (s > b && t0 == t1) continue;  // whole in one team
    const int many = s > b ? t1 - t0 + 1 : 0, each = (many + 3) >> 2;
    const int from = t0 + min(many, wave * each);
    const int to = t0 + min(many, wave * each + each);
    for (int64_t i0 = (int64_t)blockIdx.x * 256; i0 < n;
         i0 += (int64_t)gridDim.x * 256) {
      const int64_t i = i0 + lane * 4;
      const bool whole = n % 4 == 0;  // planes then start on 16 bytes
      f32x4 sum = {};
      if (i < n) {
#pragma unroll 8
        for (int t = from; t < to; ++t) {
          const float* p = planes + (2 * (int64_t)t + (t == t0)) * n + i;
          if (whole) {
            sum += *reinterpret_cast<const f32x4*>(p);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (i + r < n) sum[r] += p[r];
          }
        }
      }
      part[wave][lane] = sum;
      __syncthreads();
      if (wave == 0 && i < n) {
        sum = ((part[0][lane] + part[1][lane]) + part[2][lane]) + part[3][lane];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (i + r < n) dw[e * n + i + r] = (T)sum[r];
      }
      __syncthreads();
    }
  }
}

// dW by a block for each group and tile: many groups
template <typename T, bool WHOLE, int BM, int BN, int WM, int WN, int STEP,
          int WAVES>
__global__ __launch_bounds__(64 * WM * WN, WAVES) void segment_wgrad_kernel(
    const T* __restrict__ x, int64_t xs, const T* __restrict__ g, int64_t gs,
    ConstOffsets offsets, T* __restrict__ dw, int rows, int K, int N,
    int tiles_k, int tiles_n) {
  __shared__ __align__(16) char lds[lds_bytes(BM, BN, STEP)];
  int work = (int)xcd_order(blockIdx.x, gridDim.x);
  const int n0 = work % tiles_n * BN;
  work /= tiles_n;
  const int k0 = work % tiles_k * BM, e = work / tiles_k;
  const int64_t begin = offset_at(offsets, e, rows);
  const int64_t len = offset_at(offsets, e + 1, rows) - begin;
  tile_product<T, T, true, true, WHOLE, BM, BN, WM, WN, STEP>(
      lds, x + begin * xs + k0, xs, min(BM, K - k0), x + (rows - 1) * xs + K,
      g + begin * gs + n0, gs, min(BN, N - n0), g + (rows - 1) * gs + N, len,
      dw + ((int64_t)e * K + k0) * N + n0, N);
}

// dW by teams, as segment_wgrad_wide_kernel: few groups with many rows
template <typename T, bool WHOLE, int BM, int BN, int WM, int WN, int STEP,
          int WAVES>
__global__ __launch_bounds__(64 * WM * WN, WAVES) void segment_wgrad_teams_kernel(
    const T* __restrict__ x, int64_t xs, const T* __restrict__ g, int64_t gs,
    ConstOffsets offsets, T* __restrict__ dw, float* __restrict__ planes,
    int rows, int G, int K, int N, int tiles_n, int tiles, int teams) {
  const int work = (int)xcd_order(blockIdx.x, gridDim.x);
  __shared__ __align__(16) char lds[lds_bytes(BM, BN, STEP)];
  const int team = work / tiles, tile = work % tiles;
  const int k0 = tile / tiles_n * BM, n0 = tile % tiles_n * BN;
  const Team tr = team_rows(offsets, rows, G, teams);
  const int from = tr.begin + (int)min((int64_t)team * tr.each, (int64_t)rows);
  const int to = (int)min((int64_t)from + tr.each,
                          (int64_t)offset_at(offsets, G, rows));
  if (from >= to) return;
  int e = group_at(offsets, from, rows, G);
  for (int r = from; r < to;) {
    while (e < G - 1 && offset_at(offsets, e + 1, rows) <= r) ++e;
    const int g_start = offset_at(offsets, e, rows);
    const int g_stop = offset_at(offsets, e + 1, rows);
    const int stop = max(r + 1, min(to, g_stop));
    const T* a = x + r * xs + k0;
    const T* b = g + r * gs + n0;
    const int64_t corner = (int64_t)k0 * N + n0;
    __syncthreads();  // the last product's LDS is free
    if (r == g_start && stop == g_stop)
      tile_product<T, T, true, true, WHOLE, BM, BN, WM, WN, STEP>(
          lds, a, xs, min(BM, K - k0), x + (rows - 1) * xs + K, b, gs, min(BN, N - n0), g + (rows - 1) * gs + N, stop - r,
          dw + (int64_t)e * K * N + corner, N);
    else
      tile_product<T, float, true, true, WHOLE, BM, BN, WM, WN, STEP>(
          lds, a, xs, min(BM, K - k0), x + (rows - 1) * xs + K, b, gs, min(BN, N - n0), g + (rows - 1) * gs + N, stop - r,
          planes + (2 * (int64_t)team + (r == g_start)) * K * N + corner, N);
    r = stop;
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
  TORCH_CHECK(groups < (1 << 30), what, ": too many groups");
}

// blocks of a kernel that fills the chip once: a multiple of the 8 XCDs
static int cu_count() {
  static const int cus = [] {
    hipDeviceProp_t p;
    DOA_CHECK_HIP(hipGetDeviceProperties(&p, 0));
    return std::max(8, p.multiProcessorCount / 8 * 8);
  }();
  return cus;
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
  TORCH_CHECK(R < (1 << 30), "segment_mm: too many rows");
  const auto op = (ConstOffsets)offsets.data_ptr<int64_t>();
  if (R * N == 0) return at::empty({R, N}, x.options());
  at::Tensor y;
  // one of the weight's two inner strides has to be 1
  const bool n_inner = N <= 1 ? wt.stride(1) != 1 || K <= 1 : wt.stride(2) == 1;
  if (!n_inner && !(K <= 1 || wt.stride(1) == 1)) wt = wt.contiguous();
  const bool wc = N <= 1 ? n_inner : wt.stride(2) == 1;
  const int64_t wl = wt.stride(wc ? 1 : 2);
  DOA_FLOAT_TYPES(x.scalar_type(), "segment_mm", [&] {
    auto go = [&](auto kernel, int BM, int BN, int threads) {
      const int64_t tn = ceil_div(N, BN), blocks = (R / BM + G) * tn;
      TORCH_CHECK(blocks <= kMostThreads / threads, "segment_mm: too many tiles");
      y = at::empty({R, N}, x.options());
      hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0,
                         stream_of_current(), (const T*)xc.data_ptr(),
                         xc.stride(0), (const T*)wt.data_ptr(), wt.stride(0),
                         wl, op, (T*)y.data_ptr(), (int)R, (int)G, (int)K,
                         (int)N, (int)tn);
    };
    // whole aligned chunks of 16 bytes go straight to LDS
    const bool whole = whole_rows<T>(xc, K) && N % (16 / sizeof(T)) == 0 &&
                       K % (16 / sizeof(T)) == 0 && whole_weight<T>(wt, wl);
    auto pick = [&](auto wcv, auto wv) {
      constexpr bool WC = decltype(wcv)::value, W = decltype(wv)::value;
      if constexpr (W && sizeof(T) == 2) {
        if (N >= 256 && R >= 512 * G && K > 0) {
          const int64_t tn = ceil_div(N, 256), tiles = (R / 256 + G) * tn;
          TORCH_CHECK(tiles < (1 << 30), "segment_mm: too many tiles");
          y = at::empty({R, N}, x.options());
          hipLaunchKernelGGL((segment_mm_wide_kernel<T, WC>), dim3(cu_count()),
                             dim3(512), 0, stream_of_current(),
                             (const T*)xc.data_ptr(), xc.stride(0),
                             (const T*)wt.data_ptr(), wt.stride(0), wl,
                             op, (T*)y.data_ptr(), (int)R, (int)G, (int)K, (int)N,
                             (int)tn, (int)tiles);
          return;
        }
      }
      // Few rows a group: a lower tile leaves less of it empty and spreads the
      // weights over more blocks; many: a higher one reads them less often. us
      // with tiles of 32, 64 and (16-bit) 128 rows, by rows a group:
      //   rows                   16            32            48            96
      //   bf16 1345 x 400 x 400  110 111 116   130 121 127   157 132 139   241 178 175
      //   bf16 256 x 512 x 512   26 27 32      27 28 32      31 28 34      44 35 35
      //   fp32 1345 x 400 x 400  209 275       246 300       307 337       501 503
      //   fp32 16 x 512 x 512    10 17         11 18         15 18         16 25
      // 48 lies between where 16-bit products of many groups change (about 20)
      // and fp32 ones (about 60). From 97 on (128 rows: 297 221 202, 54 41 37)
      // steps of 64 bytes let four blocks share a CU and hide each other's first
      // loads and stores (1345 groups of 195 rows 256 us, 277 with 128 bytes).
      if (R <= 48 * G)
        go(segment_mm_kernel<T, WC, W, 32, 64, 1, 4, 128, 2>, 32, 64, 256);
      else if constexpr (sizeof(T) == 4)
        go(segment_mm_kernel<T, WC, W, 64, 64, 2, 2, W ? 64 : 128, W ? 6 : 2>,
           64, 64, 256);
      else if (R <= 96 * G)
        go(segment_mm_kernel<T, WC, W, 64, 128, 2, 2, 128, 2>, 64, 128, 256);
      else
        go(segment_mm_kernel<T, WC, W, 128, 128, 2, 2, 64, W ? 4 : 2>, 128, 128,
           256);
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
  TORCH_CHECK(R < (1 << 30), "segment_mm: too many rows");
  if (G * K * N == 0) return at::empty({G, K, N}, x.options());
  at::Tensor dw;
  DOA_FLOAT_TYPES(x.scalar_type(), "segment_mm", [&] {
    const bool whole = whole_rows<T>(xc, K) && whole_rows<T>(gc, N);
    const T* xp = (const T*)xc.data_ptr();
    const T* gp = (const T*)gc.data_ptr();
    const auto op = (ConstOffsets)offsets.data_ptr<int64_t>();
    const auto stream = stream_of_current();
    const int cus = cu_count();
    at::Tensor planes;
    auto by_teams = [&](auto kernel, int blocks, int threads, int BN,
                        int64_t tiles, int teams) {
      dw = at::empty({G, K, N}, x.options());
      planes = at::empty({2 * teams * K * N}, x.options().dtype(at::kFloat));
      hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0, stream, xp,
                         xc.stride(0), gp, gc.stride(0), op, (T*)dw.data_ptr(),
                         planes.data_ptr<float>(), (int)R, (int)G, (int)K,
                         (int)N, (int)ceil_div(N, BN), (int)tiles, teams);
      hipLaunchKernelGGL((sum_teams_kernel<T>),
                         dim3(grid_for(K * N, 256, 4096),
                              (unsigned)std::min<int64_t>(G, 1024)),
                         dim3(256), 0, stream, planes.data_ptr<float>(), op,
                         (T*)dw.data_ptr(), (int)R, (int)G, K * N, teams);
    };
    if constexpr (sizeof(T) == 2) {
      const int64_t tiles = ceil_div(K, 256) * ceil_div(N, 256);
      // its 256 x 256 tiles want 1024 rows a block to be worth their planes
      if (whole && K >= 128 && N >= 128 && R >= 512 * G && tiles <= cus &&
          R / (cus / tiles) >= 1024) {
        by_teams(segment_wgrad_wide_kernel<T>, cus, 512, 256, tiles,
                 (int)(cus / tiles));
        return;
      }
    }
    auto pick = [&](auto wv) {
      constexpr bool W = decltype(wv)::value;
      constexpr int B = W && sizeof(T) == 2 ? 128 : 64;
      const int64_t tk = ceil_div(K, B), tn = ceil_div(N, B), tiles = tk * tn;
      // Teams where groups are long and, with their tiles, few: their lengths
      // differ, and the longest would be waited for. A team has rows enough to
      // read as much as its plane costs (8 bytes an element, written and read);
      // as many blocks as the chip holds, two a CU or four of the small tiles.
      const int64_t blocks = (B == 64 ? 4 : 2) * cus;
      const int64_t each =
          std::max<int64_t>(B == 64 ? 512 : 256, 2 * K * N / (K + N));
      const int64_t teams =
          std::min(ceil_div(blocks, tiles), ceil_div(R, each));
      if (teams > 1 && R >= 256 * G && tiles * G < 8 * blocks) {
        by_teams(segment_wgrad_teams_kernel<T, W, B, B, 2, 2, 128, 2>,
                 (int)(teams * tiles), 256, B, tiles, (int)teams);
        return;
      }
      TORCH_CHECK(tiles <= kMostThreads / 256 / G, "segment_mm: too many tiles");
      dw = at::empty({G, K, N}, x.options());
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(tiles * G), dim3(256), 0, stream, xp,
                           xc.stride(0), gp, gc.stride(0), op,
                           (T*)dw.data_ptr(), (int)R, (int)K, (int)N, (int)tk,
                           (int)tn);
      };
      // short groups are a step or two: more blocks a CU hide their ends (400 x
      // 400 for 1345 groups in bf16, 49 rows a group: 174 us, and 233 with steps
      // of 128 bytes; 437 rows a group of 256 x 512: 223 and 185)
      if constexpr (W && sizeof(T) == 2) {
        if (R <= 256 * G) {
          go(segment_wgrad_kernel<T, W, B, B, 2, 2, 64, 4>);
          return;
        }
      }
      go(segment_wgrad_kernel<T, W, B, B, 2, 2, 128, 2>);
    };
    whole ? pick(std::true_type{}) : pick(std::false_type{});
  });
  DOA_CHECK_HIP(hipGetLastError());
  return dw;
}

}  // namespace doa
