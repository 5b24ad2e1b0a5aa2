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
//
// e^x is 2^(x log2 e) with the product rounded to fp32: off by |x| 2^-24 of
// itself, beside as much from the rounding of z - m, where its terms weigh e^-|x|.
// expf left the results no nearer (entropies of 14951 classes within 1.3e-6 of 64
// bits with both, fp32 gradients within 3.5e-8 of their size) and took longer:
// 2449029 x 47 with the five best 135 us instead of 122, 4096 x 14951 53 instead
// of 41, their gradients 153 instead of 135 and 59 instead of 51.
//
// Measured on one MI355X (a large copy 4.8 TB/s): 2449029 x 47 in fp16 with the
// five best 114 us (91 of copying; ~24 vector instructions a logit are 70 of
// them), 1024 x 14951 in bf16 with the ten best 17-20 us and its gradient 21 us
// (the chain of one row's steps, twice a CU at a time; 6 and 13 us of copying),
// 8 x 14951 in fp32 7 us, 1000 x 47 4.4 us. Further from the copy's time where
// lanes keep long lists, 100000 x 100 with the ten best: bf16 26 us (7), fp32 65
// (11); and where a row is short for its block, 20000 x 2000 in bf16 68 us (17),
// 600 x 115412 in bf16 65 us (29).

#include "vec.h"

namespace doa {

constexpr int kTopMost = 32;

using f32x4 = __attribute__((__vector_size__(4 * sizeof(float)))) float;

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

// what a row's sums say
struct RowStat {
  float base, logs;
  bool none;
  __device__ RowStat(float m, float s) {
    none = s == 0.f;
    base = m == -INFINITY ? 0.f : m;
    logs = none ? 0.f : logf(s);
  }
  __device__ float log_p(float z) const { return (z - base) - logs; }
  __device__ void write(int64_t row, float a, float s, float* ent,
                        float* stats) const {
    ent[row] = none ? 0.f : logs - a / s;
    stats[2 * row] = base;
    stats[2 * row + 1] = none ? INFINITY : logs;  // the mark of an empty row
  }
  __device__ float answer(float z) const { return none ? -INFINITY : log_p(z); }
};

// one term of s and a; -inf is 0 in both, NaN spoils both
__device__ inline void add_term(float z, float base, float& s, float& a) {
  const float d = z - base;
  const float e = __expf(d);
  s += e;
  a += fmaxf(d, -1e30f) * e;
}

template <typename T>
__device__ inline void write_answer(const T* zr, const RowStat& st, int64_t row,
                                    const int64_t* target, int64_t ignore,
                                    int C, float* lp) {
  const int64_t t = target[row];
  lp[row] = t == ignore ? 0.f
                        : (t >= 0 && t < C) ? st.answer((float)zr[t]) : NAN;
}

// ---------------------------------------------------------------------------
// Short rows: L lanes a row, 64 / L rows a wave. A wave copies its rows to LDS
// (16 bytes a lane, whatever the rows' alignment), each lane walks its part of
// one row and keeps the K best keys sorted in registers: an insertion is one
// median a slot for 16-bit logits, whose value and index fit one word.
// Lanes start at different places of their rows where an even length would
// send them to the same banks; the keys hold the index, so order is free.
// ---------------------------------------------------------------------------
template <typename T>
struct SmallKey;
template <>
struct SmallKey<float> {
  using type = uint64_t;
  static __device__ uint64_t make(float z, int j) { return top_key(z, j); }
  static __device__ uint64_t quick(float z, int j) {  // not for NaN
    const int32_t b = (int32_t)__float_as_uint(z + 0.f);
    return (uint64_t)(uint32_t)(b ^ (b >> 31 | INT32_MIN)) << 32 | (uint32_t)~j;
  }
  static __device__ int index(uint64_t k) { return key_index(k); }
  static __device__ float value(uint64_t k) { return key_value(k); }
  // x into the falling list; the last one drops out
  template <int K>
  static __device__ void insert(uint64_t (&list)[K], uint64_t x) {
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const uint64_t o = list[i];
      const bool c = x > o;
      list[i] = c ? x : o;
      x = c ? o : x;
    }
  }
};
template <typename T>
struct SmallKey {  // 16-bit types: the index has 16 bits too
  using type = uint32_t;
  static __device__ uint32_t make(T v, int j) {
    uint32_t b = __builtin_bit_cast(uint16_t, v);
    if ((b & 0x7fffu) == 0) b = 0;
    if (v != v) b = 0x7fffu;
    b = (b & 0x8000u) ? ~b & 0xffffu : b | 0x8000u;
    return b << 16 | (0xffffu - j);
  }
  static __device__ uint32_t quick(T v, int j) {  // not for NaN
    // -0 + 0 is +0; the sign turns the order of the negative round
    const int32_t b =
        (int32_t)__builtin_bit_cast(uint16_t, (T)(v + (T)0.f)) << 16;
    const uint32_t o = b ^ (b >> 31 | INT32_MIN);
    return (o & 0xffff0000u) | (0xffffu - j);
  }
  static __device__ int index(uint32_t k) { return 0xffff - (k & 0xffffu); }
  static __device__ float value(uint32_t k) {
    const uint32_t b = k >> 16;
    return (float)__builtin_bit_cast(
        T, (uint16_t)((b & 0x8000u) ? b & 0x7fffu : ~b));
  }
  template <int K>
  static __device__ void insert(uint32_t (&list)[K], uint32_t x) {
#pragma unroll
    for (int i = K - 1; i > 0; --i) {  // median of x and two neighbours
      const uint32_t hi = list[i - 1], lo = list[i];
      list[i] = max(min(hi, lo), min(max(hi, lo), x));
    }
    list[0] = max(list[0], x);
  }
};

template <typename K>
__device__ inline K shuffle_key(K k, int d) {
  if constexpr (sizeof(K) == 4) return __shfl_xor((int)k, d);
  else return (K)__shfl_xor((unsigned long long)k, d);
}

template <typename T, int L, int K>
__global__ __launch_bounds__(256) void log_probs_short_kernel(
    const T* __restrict__ z, int64_t zs, const int64_t* __restrict__ target,
    int64_t ignore, int64_t rows, int C, int k, float* __restrict__ lp,
    float* __restrict__ ent, float* __restrict__ top_lp,
    int64_t* __restrict__ top_idx, float* __restrict__ stats, int wave_bytes) {
  extern __shared__ __align__(16) char lds[];
  constexpr int RW = 64 / L;  // rows a wave
  using Key = SmallKey<T>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row0 = ((int64_t)blockIdx.x * 4 + wave) * RW;
  if (row0 >= rows) return;
  char* mine = lds + wave * wave_bytes;
  T* tile = reinterpret_cast<T*>(mine);
  const int many = (int)min((int64_t)RW, rows - row0);
  const T* src = z + row0 * zs;
  if (zs == C) {
    constexpr int E = 16 / sizeof(T);
    const int n = many * C, whole = n / E;
    for (int i = lane; i < whole; i += 64)
      reinterpret_cast<Chunk*>(mine)[i] =
          *reinterpret_cast<const LooseChunk*>(src + i * E);
    for (int i = whole * E + lane; i < n; i += 64) tile[i] = src[i];
  } else {
    for (int r = 0; r < many; ++r)
      for (int j = lane; j < C; j += 64) tile[r * C + j] = src[r * zs + j];
  }
  wave_sync();
  const int r = lane / L, part = lane % L;
  const bool live = r < many;
  const T* zr = tile + (live ? r : 0) * C;
  // my elements: part, part + L, ... begun at a place of my own where rows of
  // even length would start on the same banks
  const int count = (C - part + L - 1) / L;
  const int begin = (C & 1) || count < 1 ? 0 : r % count;
  // (element by element: wider reads would straddle the rows' odd alignment)
  using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
  const auto* zb =
      (const volatile __attribute__((address_space(3))) Bits*)zr;
  auto at = [&](int j) { return __builtin_bit_cast(T, (Bits)zb[j]); };
  auto walk = [&](auto visit) {
    if (C & 1) {
#pragma unroll 4
      for (int i = 0; i < count; ++i) visit(at(i * L + part), i * L + part);
    } else {
#pragma unroll 4
      for (int i = begin; i < count; ++i) visit(at(i * L + part), i * L + part);
#pragma unroll 4
      for (int i = 0; i < begin; ++i) visit(at(i * L + part), i * L + part);
    }
  };
  constexpr int S = K > 0 ? K : 1;
  typename Key::type best[S];
  auto find_best = [&](auto make) {
#pragma unroll
    for (int i = 0; i < S; ++i) best[i] = 0;
    walk([&](T v, int j) { Key::template insert<S>(best, make(v, j)); });
#pragma unroll
    for (int d = 1; d < L; d <<= 1) {
      typename Key::type other[S];
#pragma unroll
      for (int i = 0; i < S; ++i) other[i] = shuffle_key(best[i], d);
      if constexpr ((S & (S - 1)) == 0) {
        // one list against the other turned round leaves the K best, first
        // rising then falling: log K exchanges sort them
#pragma unroll
        for (int i = 0; i < S; ++i) best[i] = max(best[i], other[S - 1 - i]);
#pragma unroll
        for (int h = S / 2; h > 0; h /= 2)
#pragma unroll
          for (int i = 0; i < S; ++i)
            if (!(i & h)) {
              const auto x = best[i], y = best[i + h];
              best[i] = max(x, y);
              best[i + h] = min(x, y);
            }
      } else {
#pragma unroll
        for (int i = 0; i < S; ++i) Key::template insert<S>(best, other[i]);
      }
    }
  };
  float m = -INFINITY;
  if constexpr (K > 0) {
    find_best([](T v, int j) { return Key::quick(v, j); });
    m = Key::value(best[0]);
  } else {
    walk([&](T v, int) { m = fmaxf(m, (float)v); });
#pragma unroll
    for (int d = 1; d < L; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  }
  const float base = m == -INFINITY ? 0.f : m;
  float s = 0.f, a = 0.f;
  walk([&](T v, int) { add_term((float)v, base, s, a); });
#pragma unroll
  for (int d = 1; d < L; d <<= 1) {
    s += __shfl_xor(s, d);
    a += __shfl_xor(a, d);
  }
  if constexpr (K > 0) {
    // a NaN has spoiled its row's sum and may have lost its place
    if (__ballot(s != s)) {
      find_best([](T v, int j) { return Key::make(v, j); });
      m = Key::value(best[0]);
    }
  }
  if (!live || part != 0) return;
  const int64_t row = row0 + r;
  const RowStat st(m, s);
  st.write(row, a, s, ent, stats);
  if (target) write_answer(zr, st, row, target, ignore, C, lp);
  if constexpr (K > 0) {
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (i < k) {
        top_idx[row * k + i] = Key::index(best[i]);
        top_lp[row * k + i] = st.log_p(Key::value(best[i]));
      }
  }
}

// ---------------------------------------------------------------------------
// Long rows: a block holds a row's logits in registers, PER a thread, and reads
// them once; rows longer than that are split over blocks and joined.
//
// The best k: the 64 lanes' maxima (over the block's waves) give a threshold,
// the k-th largest of them, that at least k logits reach; what reaches it is
// collected (about k of them) and ranked by counting. Where ties or masks let
// too many through, k rounds of a block maximum find them one by one.
// ---------------------------------------------------------------------------
constexpr int kCap = 512;   // collected candidates

template <int NT>
struct LongShared {
  float lane_max[NT / 64][64];
  float sums[2][NT / 64];
  uint64_t keys[kCap];
  uint64_t round[NT / 64];
  float threshold;
  int count;
};

// a thread's part of a row as it was read
template <typename T, int PER>
struct Logits {
  static constexpr int E = 16 / sizeof(T);
  union Part { Chunk q; T e[E]; };
  Part part[PER / E];
  __device__ float at(int i, int e) const { return (float)part[i].e[e]; }
  // what was made of the logits is made again when it is wanted: kept, it would
  // cost the registers of the other blocks on the CU
  __device__ void anew() {
#pragma unroll
    for (int i = 0; i < PER / E; ++i) asm volatile("" : "+v"(part[i].q));
  }
};

// the k largest of the block's keys, falling, each given to emit(rank, key)
template <typename T, int NT, int PER, typename Emit>
__device__ inline void best_of_block(Logits<T, PER>& v, const T* zr, int c0,
                                     int c1, int k, LongShared<NT>& sh,
                                     Emit emit) {
  constexpr int E = Logits<T, PER>::E;
  const float t = sh.threshold;
  v.anew();
#pragma unroll
  for (int i = 0; i < PER / E; ++i) {
    const int j = c0 + (i * NT + (int)threadIdx.x) * E;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (!(v.at(i, e) < t) && j + e < c1) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kCap) sh.keys[at] = top_key(v.at(i, e), j + e);
      }
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
  const int count = sh.count;
  if (count <= kCap) {
    for (int i = threadIdx.x; i < count; i += NT) {
      const uint64_t key = sh.keys[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += sh.keys[j] > key;
      if (rank < k) emit(rank, key);
    }
    // fewer than k logits in this part of the row
    for (int i = count + threadIdx.x; i < k; i += NT) emit(i, 0);
    return;
  }
  uint64_t last = ~0ull;
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
    // (from memory again: rare, and registers would cost a block on the CU)
    for (int j = c0 + threadIdx.x; j < c1; j += NT) {
      const uint64_t key = top_key((float)zr[j], j);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t o = shuffle_key(best, d);
      best = o > best ? o : best;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.round[threadIdx.x >> 6] = best;
    __syncthreads();
    for (int w = 0; w < NT / 64; ++w) best = max(best, sh.round[w]);
    if (threadIdx.x == 0) emit(r, best);
    last = best;
  }
}

// the value that k of a wave's 64 values reach (-inf: fewer than k are above)
__device__ inline float kth_of_wave(float v, int k) {
  int reach = 0;
#pragma unroll 8
  for (int i = 0; i < 64; ++i) {
    const float o = __uint_as_float(
        __builtin_amdgcn_readlane(__float_as_uint(v), i));
    reach += o >= v;
  }
  float t = reach >= k ? v : -INFINITY;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) t = fmaxf(t, __shfl_xor(t, d));
  return t;
}

// (64 registers: two blocks of 1024 threads a CU)
template <typename T, int NT, int PER>
__global__ __launch_bounds__(NT, 8) void log_probs_long_kernel(
    const T* __restrict__ z, int64_t zs, const int64_t* __restrict__ target,
    int64_t ignore, int C, int k, int splits, int chunk,
    float* __restrict__ lp, float* __restrict__ ent,
    float* __restrict__ top_lp, int64_t* __restrict__ top_idx,
    float* __restrict__ stats, float* __restrict__ part_sums,
    uint64_t* __restrict__ part_keys) {
  __shared__ LongShared<NT> sh;
  constexpr int E = 16 / sizeof(T);
  const int64_t row = blockIdx.x / splits;
  const int part = blockIdx.x % splits;
  const int c0 = part * chunk, c1 = min(C, c0 + chunk);
  const T* zr = z + row * zs;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Logits<T, PER> v;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER / E; ++i) {
    const int j = c0 + (i * NT + threadIdx.x) * E;
    if (j + E <= c1) {
      v.part[i].q = *reinterpret_cast<const LooseChunk*>(zr + j);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        v.part[i].e[e] = j + e < c1 ? zr[j + e] : (T)-INFINITY;
    }
  }
#pragma unroll
  for (int i = 0; i < PER / E; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(m, v.at(i, e));
  sh.lane_max[wave][lane] = m;
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) m = fmaxf(m, sh.lane_max[w][lane]);
  if (k > 0 && wave == 0) {
    const float t = kth_of_wave(m, k);
    if (lane == 0) sh.threshold = t;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  const float base = m == -INFINITY ? 0.f : m;
  float s = 0.f, a = 0.f;
  v.anew();
#pragma unroll
  for (int i = 0; i < PER / E; ++i) {
#pragma unroll
    for (int e = 0; e < E; ++e) add_term(v.at(i, e), base, s, a);
    __builtin_amdgcn_sched_barrier(0);  // not all exponentials at once
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    s += __shfl_xor(s, d);
    a += __shfl_xor(a, d);
  }
  if (lane == 0) {
    sh.sums[0][wave] = s;
    sh.sums[1][wave] = a;
  }
  __syncthreads();
  s = a = 0.f;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    s += sh.sums[0][w];
    a += sh.sums[1][w];
  }
  if (splits > 1) {
    if (threadIdx.x == 0) {
      float* o = part_sums + (int64_t)blockIdx.x * 3;
      o[0] = m;
      o[1] = s;
      o[2] = a;
    }
    if (k > 0)
      best_of_block<T, NT, PER>(v, zr, c0, c1, k, sh, [&](int r, uint64_t key) {
        part_keys[(int64_t)blockIdx.x * k + r] = key;
      });
    return;
  }
  const RowStat st(m, s);
  if (threadIdx.x == 0) {
    st.write(row, a, s, ent, stats);
    if (target) write_answer(zr, st, row, target, ignore, C, lp);
  }
  if (k > 0)
    best_of_block<T, NT, PER>(v, zr, c0, c1, k, sh, [&](int r, uint64_t key) {
      top_idx[row * k + r] = key_index(key);
      top_lp[row * k + r] = st.log_p(key_value(key));
    });
}

// the parts of one row joined: a block a row
template <typename T>
__global__ __launch_bounds__(256) void log_probs_join_kernel(
    const T* __restrict__ z, int64_t zs, const int64_t* __restrict__ target,
    int64_t ignore, int C, int k, int splits,
    const float* __restrict__ part_sums, const uint64_t* __restrict__ part_keys,
    float* __restrict__ lp, float* __restrict__ ent,
    float* __restrict__ top_lp, int64_t* __restrict__ top_idx,
    float* __restrict__ stats) {
  __shared__ uint64_t keys[kCap], round[4];
  __shared__ float tmp[4];
  const int64_t row = blockIdx.x;
  const float* ps = part_sums + row * splits * 3;
  auto over_block = [&](float v, auto op) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = op(v, __shfl_xor(v, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    return op(op(tmp[0], tmp[1]), op(tmp[2], tmp[3]));
  };
  float m = -INFINITY;
  for (int p = threadIdx.x; p < splits; p += 256) m = fmaxf(m, ps[3 * p]);
  m = over_block(m, [](float x, float y) { return fmaxf(x, y); });
  const float base = m == -INFINITY ? 0.f : m;
  float s = 0.f, a = 0.f;
  for (int p = threadIdx.x; p < splits; p += 256) {
    // sums over a base of their own: e^(z - m_p) -> e^(z - m)
    const float mp = ps[3 * p];
    // (a part that lies far below has e = 0; its d times its sum, a part's length
    // at most, must not pass the largest float there)
    const float d = (mp == -INFINITY ? 0.f : mp) - base;
    const float e = ps[3 * p + 1] == 0.f ? 0.f : __expf(d);
    s += ps[3 * p + 1] * e;
    a += (ps[3 * p + 2] + fmaxf(d, -1e30f) * ps[3 * p + 1]) * e;
  }
  s = over_block(s, [](float x, float y) { return x + y; });
  a = over_block(a, [](float x, float y) { return x + y; });
  const RowStat st(m, s);
  if (threadIdx.x == 0) {
    st.write(row, a, s, ent, stats);
    if (target) write_answer(z + row * zs, st, row, target, ignore, C, lp);
  }
  const uint64_t* pk = part_keys + row * splits * k;
  const int64_t count = (int64_t)splits * k;
  auto emit = [&](int r, uint64_t key) {
    top_idx[row * k + r] = key_index(key);
    top_lp[row * k + r] = st.log_p(key_value(key));
  };
  if (count <= kCap) {
    for (int i = threadIdx.x; i < count; i += 256) keys[i] = pk[i];
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += 256) {
      const uint64_t key = keys[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += keys[j] > key;
      if (key && rank < k) emit(rank, key);
    }
    return;
  }
  uint64_t last = ~0ull;
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
    for (int64_t i = threadIdx.x; i < count; i += 256) {
      const uint64_t key = pk[i];
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t o = shuffle_key(best, d);
      best = o > best ? o : best;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) round[threadIdx.x >> 6] = best;
    __syncthreads();
    for (int w = 0; w < 4; ++w) best = max(best, round[w]);
    if (threadIdx.x == 0) emit(r, best);
    last = best;
  }
}

// ---------------------------------------------------------------------------
// dz_j = g_lp [j = t] + sum_i g_i [j = idx_i]
//        - p_j (g_lp + sum_i g_i + g_H (log p_j + H))
// A block makes a tile in LDS, in fp32: several whole rows or a part of a long
// one. The common term comes first, then the alternatives' own (different
// places), then the target's, and the tile is rounded once on its way out.
// ---------------------------------------------------------------------------
constexpr int kTileElems = 4096;
constexpr int kTileRows = 64;

struct RowPull {
  float base, logs, pull, gh, ent;
};

template <typename T>
__global__ __launch_bounds__(256) void log_probs_bwd_kernel(
    const T* __restrict__ z, int64_t zs, const int64_t* __restrict__ target,
    int64_t ignore, const int64_t* __restrict__ top_idx,
    const float* __restrict__ stats, const float* __restrict__ ent,
    const float* __restrict__ g_lp, const float* __restrict__ g_ent,
    const float* __restrict__ g_top, int64_t rows, int C, int k,
    int tile_rows, int col_tiles, uint64_t magic, T* __restrict__ dz) {
  __shared__ __align__(16) float tile[kTileElems];
  __shared__ RowPull info[kTileRows];
  __shared__ float own[kTileRows * kTopMost];
  constexpr int E = 16 / sizeof(T), PER = kTileElems / (256 * E);
  const int64_t row0 = blockIdx.x / col_tiles * (int64_t)tile_rows;
  const int c0 = blockIdx.x % col_tiles * kTileElems;
  const int many = (int)min((int64_t)tile_rows, rows - row0);
  const int W = min(kTileElems, C - c0);  // = C where a tile has many rows
  const int n = many * W;
  // all loads first: what the tile needs and the logits themselves
  const T* src = z + row0 * zs + c0;
  const bool flat = zs == W || many == 1;
  union Part { Chunk q; T e[E]; };
  Part part[PER];
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int i = (p * 256 + threadIdx.x) * E;
    if (flat && i + E <= n) {
      part[p].q = *reinterpret_cast<const LooseChunk*>(src + i);
    } else if (i < n) {
      // i / W by a product: exact for i below 2^12
      int r = (int)((i * magic) >> 32), c = i - r * W;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        part[p].e[e] = i + e < n ? src[r * zs + c] : (T)0.f;
        if (++c == W) c = 0, ++r;
      }
    }
  }
  const int tops = g_top ? many * k : 0;
  for (int i = threadIdx.x; i < tops; i += 256) own[i] = g_top[row0 * k + i];
  int64_t t = -1;
  float gl = 0.f;
  RowPull p{};
  if (threadIdx.x < many) {
    const int64_t row = row0 + threadIdx.x;
    p = {stats[2 * row], stats[2 * row + 1], 0.f, g_ent ? g_ent[row] : 0.f,
         ent[row]};
    if (target && g_lp) {
      t = target[row];
      gl = t == ignore ? 0.f : (t >= 0 && t < C) ? g_lp[row] : NAN;
    }
  }
  const int first_top =
      threadIdx.x < tops ? (int)(top_idx[row0 * k + threadIdx.x] - c0) : -1;
  __syncthreads();
  if (threadIdx.x < many) {
    p.pull = gl;
    if (g_top)
      for (int i = 0; i < k; ++i) p.pull += own[threadIdx.x * k + i];
    info[threadIdx.x] = p;
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int i = (q * 256 + threadIdx.x) * E;
    if (i >= n) break;
    int r = (int)((i * magic) >> 32), c = i - r * W;
    union { f32x4 v[E / 4]; float e[E]; } g;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const RowPull& u = info[r];
      const float l = ((float)part[q].e[e] - u.base) - u.logs;
      // (e^-128 is 0 in fp32: from there on l must not spoil the product, however
      // large gh is)
      const float v = -__expf(l) * (u.pull + u.gh * (fmaxf(l, -128.f) + u.ent));
      g.e[e] = u.logs == INFINITY ? 0.f : v;
      // (behind the last row: any row there is)
      if (++c == W) c = 0, r = min(r + 1, many - 1);
    }
#pragma unroll
    for (int e = 0; e < E / 4; ++e)
      *reinterpret_cast<f32x4*>(tile + i + 4 * e) = g.v[e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tops; i += 256) {
    const int r = i / k;
    const int j = i == (int)threadIdx.x ? first_top
                                        : (int)(top_idx[row0 * k + i] - c0);
    if (j >= 0 && j < W && info[r].logs != INFINITY) tile[r * W + j] += own[i];
  }
  __syncthreads();
  if (threadIdx.x < many && t >= c0 && t < c0 + W && t != ignore &&
      p.logs != INFINITY)
    tile[threadIdx.x * W + (int)(t - c0)] += gl;
  __syncthreads();
  T* out = dz + row0 * C + c0;  // rows of a tile follow each other
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int i = (q * 256 + threadIdx.x) * E;
    if (i >= n) break;
    union { f32x4 v[E / 4]; float e[E]; } g;
#pragma unroll
    for (int e = 0; e < E / 4; ++e)
      g.v[e] = *reinterpret_cast<const f32x4*>(tile + i + 4 * e);
    Part u;
#pragma unroll
    for (int e = 0; e < E; ++e) u.e[e] = (T)g.e[e];
    if (i + E <= n) {
      *reinterpret_cast<LooseChunk*>(out + i) = u.q;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e < n) out[i + e] = u.e[e];
    }
  }
}

// more rows than one grid has threads for go out in launches of `most` rows, one
// behind the other on the stream
template <typename Launch>
static void by_grids(int64_t rows, int64_t most, Launch launch) {
  for (int64_t r0 = 0; r0 < rows; r0 += most)
    launch(r0, std::min(most, rows - r0));
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
  TORCH_CHECK(C >= 1 && C <= (1 << 30), "log_probs: 1 to 2^30 classes");
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
  if (rows == 0) return {lp, ent, top_lp, top_idx, stats};
  auto stream = stream_of_current();
  DOA_FLOAT_TYPES(logits.scalar_type(), "log_probs", [&] {
    const int64_t zs = zc.stride(0);
    // rows r0 .. r0 + n of everything there is a row of
    struct Rows {
      const T* z;
      const int64_t* target;
      float *lp, *ent, *top_lp;
      int64_t* top_idx;
      float* stats;
    };
    auto rows_from = [&](int64_t r0) {
      return Rows{(const T*)zc.data_ptr() + r0 * zs,
                  target.has_value() ? target->data_ptr<int64_t>() + r0 : nullptr,
                  lp.defined() ? lp.data_ptr<float>() + r0 : nullptr,
                  ent.data_ptr<float>() + r0, top_lp.data_ptr<float>() + r0 * k,
                  top_idx.data_ptr<int64_t>() + r0 * k,
                  stats.data_ptr<float>() + r0 * 2};
    };
    const int64_t row_bytes = C * sizeof(T);
    if (row_bytes <= 2048) {
      // lanes a row: as many as keep a wave's rows at 8 KiB of LDS, more where
      // there are too few rows for 1024 waves
      int L = row_bytes <= 128 ? 1 : row_bytes <= 512 ? 4 : 16;
      while (L < 16 && rows * L < 64 * 1024) L *= 4;
      const int wave_bytes = (int)ceil_div(64 / L * row_bytes, 16) * 16;
      const int64_t per_block = 4 * (64 / L);
      auto go = [&](auto lv, auto kv) {
        by_grids(rows, kMostThreads / 256 * per_block, [&](int64_t r0, int64_t n) {
          const Rows r = rows_from(r0);
          hipLaunchKernelGGL(
              (log_probs_short_kernel<T, decltype(lv)::value,
                                      decltype(kv)::value>),
              dim3(ceil_div(n, per_block)), dim3(256), 4 * wave_bytes, stream,
              r.z, zs, r.target, ignore, n, (int)C, (int)k, r.lp, r.ent,
              r.top_lp, r.top_idx, r.stats, wave_bytes);
        });
      };
      // Registers for the next such number of keys; each number is a kernel that
      // takes long to compile. 2449029 x 47 in fp16: none 60 us, 1 71, 2 81, 5 115,
      // 6 138, 10 239, 16 422, 32 998 (copying 61, 67, 73, 91, 97, 122, 159, 257).
      auto slots = [&](auto lv) {
        if (k == 0) go(lv, std::integral_constant<int, 0>{});
        else if (k == 1) go(lv, std::integral_constant<int, 1>{});
        else if (k <= 5) go(lv, std::integral_constant<int, 5>{});
        else if (k <= 10) go(lv, std::integral_constant<int, 10>{});
        else if (k <= 16) go(lv, std::integral_constant<int, 16>{});
        else go(lv, std::integral_constant<int, kTopMost>{});
      };
      if (L == 1) slots(std::integral_constant<int, 1>{});
      else if (L == 4) slots(std::integral_constant<int, 4>{});
      else slots(std::integral_constant<int, 16>{});
      return;
    }
    auto go = [&](auto nv, auto pv) {
      constexpr int NT = decltype(nv)::value, PER = decltype(pv)::value;
      constexpr int most = NT * PER;
      const int64_t splits = ceil_div(C, most);
      const int chunk = (int)ceil_div(ceil_div(C, splits), 16) * 16;
      const int64_t grid = kMostThreads / (NT * splits);
      at::Tensor sums, keys;
      if (splits > 1) {
        const int64_t parts = std::min(rows, grid) * splits;
        sums = at::empty({parts * 3}, f32);
        keys = at::empty({parts * k}, top_idx.options());
      }
      float* sp = splits > 1 ? sums.data_ptr<float>() : nullptr;
      uint64_t* kp =
          splits > 1 ? (uint64_t*)keys.data_ptr<int64_t>() : nullptr;
      by_grids(rows, grid, [&](int64_t r0, int64_t n) {
        const Rows r = rows_from(r0);
        hipLaunchKernelGGL((log_probs_long_kernel<T, NT, PER>), dim3(n * splits),
                           dim3(NT), 0, stream, r.z, zs, r.target, ignore, (int)C,
                           (int)k, (int)splits, chunk, r.lp, r.ent, r.top_lp,
                           r.top_idx, r.stats, sp, kp);
        if (splits > 1)
          hipLaunchKernelGGL((log_probs_join_kernel<T>), dim3(n), dim3(256), 0,
                             stream, r.z, zs, r.target, ignore, (int)C, (int)k,
                             (int)splits, sp, kp, r.lp, r.ent, r.top_lp,
                             r.top_idx, r.stats);
      });
    };
    constexpr std::integral_constant<int, 16> per;
    if (C <= 256 * 16) go(std::integral_constant<int, 256>{}, per);
    else go(std::integral_constant<int, 1024>{}, per);
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
  if (rows == 0) return dz;
  const int64_t W = std::min<int64_t>(C, kTileElems);
  const int64_t col_tiles = ceil_div(C, kTileElems);
  // rows a tile: what fits, but at least 1024 tiles where there are the rows
  const int64_t tile_rows = std::max<int64_t>(
      1, std::min<int64_t>({kTileRows, kTileElems / W, ceil_div(rows, 1024)}));
  const uint64_t magic = ((uint64_t)1 << 32) / W + 1;
  DOA_FLOAT_TYPES(logits.scalar_type(), "log_probs", [&] {
    by_grids(rows, kMostThreads / 256 / col_tiles * tile_rows,
             [&](int64_t r0, int64_t n) {
      hipLaunchKernelGGL(
          (log_probs_bwd_kernel<T>), dim3(ceil_div(n, tile_rows) * col_tiles),
          dim3(256), 0, stream_of_current(),
          (const T*)zc.data_ptr() + r0 * zc.stride(0), zc.stride(0),
          target.has_value() ? target->data_ptr<int64_t>() + r0 : nullptr,
          ignore, top_idx.data_ptr<int64_t>() + r0 * k,
          stats.data_ptr<float>() + r0 * 2, ent.data_ptr<float>() + r0,
          gp[0] ? gp[0] + r0 : nullptr, gp[1] ? gp[1] + r0 : nullptr,
          gp[2] ? gp[2] + r0 * k : nullptr, n, (int)C, (int)k, (int)tile_rows,
          (int)col_tiles, magic, (T*)dz.data_ptr() + r0 * C);
    });
  });
  DOA_CHECK_HIP(hipGetLastError());
  return dz;
}

}  // namespace doa
