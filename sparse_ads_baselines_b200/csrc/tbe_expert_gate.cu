// The router's gate: the k largest logits of every row with their softmax weights, and its gradient.
//
// Forward, per row l[0..E):   chosen = the k largest, ties to the lowest index, descending
//   e_j = exp(l_j - max l);   w_s = e_s / sum over the chosen   (renormalize)
//                             w_s = e_s / sum over all           (otherwise)
// A logit of -inf is a switched-off expert: it is never chosen, its slot gets id -1 and weight 0, so a
// row with nothing left is (-1, 0) throughout.  NaN ranks above everything and makes the row's weights
// NaN, as the formula does; the ids stay distinct and in range.
//
// A row belongs to a group of G = 2^g lanes (several rows per warp when E is small), each lane holds V
// of its logits as sort keys that carry the value's order and the column: the larger key is the larger
// logit, or the lower column of equal ones.  16-bit logits fit value and column into 32 bits, so a warp
// finds a maximum in one redux; 32-bit ones take 64-bit keys and two.
//
// The k largest lie in the k lanes with the largest maxima.  With a warp per row those lanes are found
// first, by k rounds over the lanes' maxima alone; their values are dealt to all lanes, C = k V / 32 each
// (2 or 4), and k rounds over those give the choices.  Groups of fewer lanes, and a k V above 128, run the
// rounds over all keys: sorted in runs of eight (a 19-comparator network), a round compares the runs' heads
// and pops one.  The backward takes the gate's own weights and ids; only the whole-row softmax reads the logits
// again and recomputes the row's maximum and sum.
//
// Bound by instruction issue (78 % of the slots), not by HBM.  65536 rows of 256 bf16 logits, k = 8, are
// 33.5 MB (5 us) and take 25 us: 33 us with rounds over the sorted runs of all keys, 30 with the best lanes
// first, 25 with four rows per warp (29 with the whole row's softmax).  fp32: 45 us (48).  Rows that are no multiple
// of 16 bytes take one element per load: 60 bf16 experts, k = 4, 11.3 us against 9.2 for 64, 100 21.4 against 17.2
// for 96 or 104.  One row: 2.4 us, about an empty kernel's time.  The fp64 variants with 128-bit keys spill (64 to
// 92 bytes) in a warp per row.
#include "tbe_elem.cuh"

namespace tbe {
namespace {

constexpr int kGateThreads = 256;
constexpr int64_t kManyRows = 16384;  // rows from which a warp takes several
constexpr int kGateMaxExperts = 1024;
constexpr int kGateMaxK = 32;

// ---------------------------------------------------------------- sort keys
// Order-preserving integers, ascending with the value, -0 equal to +0, every NaN above +inf.  alive() tells a
// candidate from -inf, which is also what lies outside the row; 0 is a key that was taken.
template <typename T>
struct Key;

// Two 16-bit values at a time.  Adding +0 turns -0 into +0 and every NaN into the canonical 0x7fff.
template <typename T>
struct Key16 {
  using type = uint32_t;
  __device__ static __forceinline__ void pair(uint32_t x, int col0, int col1, type* key) {
    const uint32_t sign = (x >> 15) & 0x00010001u;
    const uint32_t o = x ^ (0x80008000u | (sign * 0x7fffu));  // all bits of a negative, the top bit of the others
    key[0] = __byte_perm(o, static_cast<uint32_t>(0xffff - col0), 0x1054);
    key[1] = __byte_perm(o, static_cast<uint32_t>(0xffff - col1), 0x3254);
  }
  __device__ static __forceinline__ uint16_t bits(type k) {
    const uint32_t o = k >> 16;
    return static_cast<uint16_t>((o & 0x8000u) ? (o & 0x7fffu) : ~o);
  }
  __device__ static __forceinline__ int col(type k) { return 0xffff - static_cast<int>(k & 0xffffu); }
};
template <>
struct Key<__half> : Key16<__half> {
  __device__ static __forceinline__ void of(const __half* v, int c0, int c1, type* key) {
    const __half2 x = __hadd2(__halves2half2(v[0], v[1]), __half2half2(__ushort_as_half(0)));
    uint32_t u;
    memcpy(&u, &x, 4);
    pair(u, c0, c1, key);
  }
  __device__ static __forceinline__ bool alive(type k) { return k > 0x03ffffffu; }  // above -inf in every column
  __device__ static __forceinline__ float value(type k) { return __half2float(__ushort_as_half(bits(k))); }
};
template <>
struct Key<__nv_bfloat16> : Key16<__nv_bfloat16> {
  __device__ static __forceinline__ void of(const __nv_bfloat16* v, int c0, int c1, type* key) {
    const __nv_bfloat162 x = __hadd2(__halves2bfloat162(v[0], v[1]), __bfloat162bfloat162(__ushort_as_bfloat16(0)));
    uint32_t u;
    memcpy(&u, &x, 4);
    pair(u, c0, c1, key);
  }
  __device__ static __forceinline__ bool alive(type k) { return k > 0x007fffffu; }
  __device__ static __forceinline__ float value(type k) { return __bfloat162float(__ushort_as_bfloat16(bits(k))); }
};
template <>
struct Key<float> {
  using type = unsigned long long;
  __device__ static __forceinline__ type one(float v, int c) {
    const uint32_t b = __float_as_uint(__fadd_rn(v, 0.f));  // as above
    const uint32_t o = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
    return (static_cast<type>(o) << 32) | static_cast<uint32_t>(0xffff - c);
  }
  __device__ static __forceinline__ void of(const float* v, int c0, int c1, type* key) {
    key[0] = one(v[0], c0);
    key[1] = one(v[1], c1);
  }
  __device__ static __forceinline__ bool alive(type k) { return static_cast<uint32_t>(k >> 32) > 0x007fffffu; }
  __device__ static __forceinline__ float value(type k) {
    const uint32_t o = static_cast<uint32_t>(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
  }
  __device__ static __forceinline__ int col(type k) { return 0xffff - static_cast<int>(k & 0xffffu); }
};
template <>
struct Key<double> {
  using type = unsigned __int128;
  __device__ static __forceinline__ void of(const double* v, int c0, int c1, type* key) {
    key[0] = one(v[0], c0);
    key[1] = one(v[1], c1);
  }
  __device__ static __forceinline__ bool alive(type k) { return k != 0; }
  __device__ static __forceinline__ type one(double v, int c) {
    if (v == -INFINITY) return 0;
    unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v));
    if (b == 0x8000000000000000ull) b = 0;
    unsigned long long o = (b >> 63) ? ~b : (b | 0x8000000000000000ull);
    if (isnan(v)) o = ~0ull;
    return (static_cast<type>(o) << 64) | static_cast<unsigned long long>(0xffff - c);
  }
  __device__ static __forceinline__ double value(type k) {
    const unsigned long long o = static_cast<unsigned long long>(k >> 64);
    return __longlong_as_double(static_cast<long long>((o >> 63) ? (o & 0x7fffffffffffffffull) : ~o));
  }
  __device__ static __forceinline__ int col(type k) { return 0xffff - static_cast<int>(static_cast<uint32_t>(k) & 0xffffu); }
};

// Maximum over the 2^glog lanes of a group; every lane of the warp takes part.
__device__ __forceinline__ uint32_t group_max(uint32_t v, int glog) {
  if (glog == 5) return __reduce_max_sync(kFullMask, v);
  for (int m = 1; m < (1 << glog); m <<= 1) v = max(v, __shfl_xor_sync(kFullMask, v, m));
  return v;
}
__device__ __forceinline__ unsigned long long group_max(unsigned long long v, int glog) {
  if (glog == 5) {
    const uint32_t hi = static_cast<uint32_t>(v >> 32);
    const uint32_t top = __reduce_max_sync(kFullMask, hi);
    const uint32_t low = __reduce_max_sync(kFullMask, hi == top ? static_cast<uint32_t>(v) : 0u);
    return (static_cast<unsigned long long>(top) << 32) | low;
  }
  for (int m = 1; m < (1 << glog); m <<= 1) {
    const unsigned long long o = __shfl_xor_sync(kFullMask, v, m);
    v = o > v ? o : v;
  }
  return v;
}
__device__ __forceinline__ unsigned __int128 group_max(unsigned __int128 v, int glog) {
  for (int m = 1; m < (1 << glog); m <<= 1) {
    const unsigned long long hi = __shfl_xor_sync(kFullMask, static_cast<unsigned long long>(v >> 64), m);
    const unsigned long long lo = __shfl_xor_sync(kFullMask, static_cast<unsigned long long>(v), m);
    const unsigned __int128 o = (static_cast<unsigned __int128>(hi) << 64) | lo;
    v = o > v ? o : v;
  }
  return v;
}

template <typename K>
__device__ __forceinline__ K shuffle(K v, int from) {
  if constexpr (sizeof(K) == 16) {
    const unsigned long long hi = __shfl_sync(kFullMask, static_cast<unsigned long long>(v >> 64), from);
    const unsigned long long lo = __shfl_sync(kFullMask, static_cast<unsigned long long>(v), from);
    return (static_cast<K>(hi) << 64) | lo;
  } else {
    return __shfl_sync(kFullMask, v, from);
  }
}

// Eight keys, largest first (Batcher's odd-even merge network, 19 comparators).
template <typename K>
__device__ __forceinline__ void order2(K& a, K& b) {
  const bool swap = b > a;
  const K hi = swap ? b : a;
  b = swap ? a : b;
  a = hi;
}
template <>
__device__ __forceinline__ void order2<uint32_t>(uint32_t& a, uint32_t& b) {
  const uint32_t hi = max(a, b);
  b = min(a, b);
  a = hi;
}
template <typename K>
__device__ __forceinline__ void sort8(K* k) {
  order2(k[0], k[1]), order2(k[2], k[3]), order2(k[4], k[5]), order2(k[6], k[7]);
  order2(k[0], k[2]), order2(k[1], k[3]), order2(k[4], k[6]), order2(k[5], k[7]);
  order2(k[1], k[2]), order2(k[5], k[6]);
  order2(k[0], k[4]), order2(k[1], k[5]), order2(k[2], k[6]), order2(k[3], k[7]);
  order2(k[2], k[4]), order2(k[3], k[5]);
  order2(k[1], k[2]), order2(k[3], k[4]), order2(k[5], k[6]);
}

// Rounds over C keys per lane in descending order: the k largest of the group, the s-th in lane s.
// first(m) is called with the largest.
template <int C, typename K, typename F>
__device__ __forceinline__ K take_largest(K* key, int k, int sub, int glog, F first) {
  constexpr int RUN = C < 8 ? C : 8;  // the keys come in sorted runs
  K mine = 0;
  for (int s = 0; s < k; ++s) {
    K m = key[0];
#pragma unroll
    for (int r = RUN; r < C; r += RUN) m = key[r] > m ? key[r] : m;
    m = group_max(m, glog);
    if (s == 0) first(m);
    if (sub == s) mine = m;
#pragma unroll
    for (int r = 0; r < C; r += RUN) {
      const bool pop = key[r] == m;
#pragma unroll
      for (int i = r; i < r + RUN - 1; ++i) key[i] = pop ? key[i + 1] : key[i];
      key[r + RUN - 1] = pop ? K(0) : key[r + RUN - 1];
    }
  }
  return mine;
}

// A warp per row: the keys of the k lanes with the largest maxima, dealt to the lanes through `room`
// (32 * C keys of shared memory), then the rounds over those.
template <int V, int C, typename K, typename F>
__device__ __forceinline__ K take_from_best_lanes(const K* key, int k, int lane, K* room, F first) {
  K best = key[0];
#pragma unroll
  for (int i = 1; i < V; ++i) best = key[i] > best ? key[i] : best;
  int rank = -1, lanes = 0;
  for (int s = 0; s < k; ++s) {
    const K m = group_max(best, 5);
    if (s == 0) first(m);
    if (m == K(0)) break;  // (the whole warp) no candidate is left
    lanes = s + 1;
    if (best == m) {  // keys differ: one lane
      rank = s;
      best = 0;
    }
  }
  // lanes * V keys are written, in 16-byte stores; a lane behind them has nothing
  struct alignas(16) Some {
    K key[V];
  } all;
  struct alignas(C * sizeof(K) < 16 ? C * sizeof(K) : 16) Few {
    K key[C];
  } mine;
#pragma unroll
  for (int i = 0; i < V; ++i) all.key[i] = key[i];
  if (rank >= 0) reinterpret_cast<Some*>(room)[rank] = all;
  __syncwarp();
  mine = reinterpret_cast<const Few*>(room)[lane];
  K few[C];
#pragma unroll
  for (int i = 0; i < C; ++i) few[i] = lane * C < lanes * V ? mine.key[i] : K(0);
  order2(few[0], few[1]);
  if (C == 4) order2(few[2], few[3]), order2(few[0], few[2]), order2(few[1], few[3]), order2(few[1], few[2]);
  return take_largest<C>(few, k, lane, 5, [](K) {});
}

// Column of a lane's i-th value: vectors of VE neighbouring columns, dealt to the lanes in turn.
template <int VE>
__device__ __forceinline__ int column(int i, int sub, int glog) {
  return (((i / VE) << glog) + sub) * VE + i % VE;
}

// The row's values in the lane's registers, -inf outside the row.
template <typename T, int V, int VE>
__device__ __forceinline__ void load_row(const T* row, bool live, int E, int sub, int glog, T* v) {
  const T none = from_acc<T>(-INFINITY);
#pragma unroll
  for (int i = 0; i < V; i += VE) {
    const int c = column<VE>(i, sub, glog);
    if (live && c < E) {  // E % VE == 0: a vector lies inside the row or outside it
      const Raw<VE * sizeof(T)> r = ld_stream<VE * sizeof(T)>(row + c);
      memcpy(v + i, &r, sizeof(r));
    } else {
#pragma unroll
      for (int j = 0; j < VE; ++j) v[i + j] = none;
    }
  }
}

struct GateArgs {
  const void* logits;
  int64_t stride;
  void* weights;
  int32_t* experts;
  int64_t N;
  int E, k, glog;
  bool renormalize;
  const void* grad_weights;  // backward only
  void* grad_logits;
};

// WARP: a warp per row (a.glog is 5), known at compile time.
template <typename T, int V, int VE, bool WARP>
__global__ void __launch_bounds__(kGateThreads) gate_kernel(GateArgs a) {
  using A = typename Acc<T>::type;
  using K = typename Key<T>::type;
  const int lane = threadIdx.x & 31, glog = WARP ? 5 : a.glog, sub = lane & ((1 << glog) - 1);
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * (kGateThreads >> 5) + (threadIdx.x >> 5);
  const int64_t row = (warp << (5 - glog)) + (lane >> glog);
  const bool live = row < a.N;
  T v[V];
  load_row<T, V, VE>(static_cast<const T*>(a.logits) + row * a.stride, live, a.E, sub, glog, v);
  K key[V];
#pragma unroll
  for (int i = 0; i < V; i += 2) Key<T>::of(v + i, column<VE>(i, sub, glog), column<VE>(i + 1, sub, glog), key + i);
  A top = 0, sum = 0;
  auto first = [&](K m) {
    top = Key<T>::alive(m) ? Key<T>::value(m) : A(0);
    if (!a.renormalize) {
#pragma unroll
      for (int i = 0; i < V; ++i) sum += exp(to_acc<T>(v[i]) - top);  // -inf adds 0
    }
  };
  __shared__ __align__(16) K room[kGateThreads / 32][128];
  K mine;  // the s-th largest, in lane s of the group (k <= G)
  if (WARP && a.k * V <= 64) {
    mine = take_from_best_lanes<V, 2>(key, a.k, lane, room[threadIdx.x >> 5], first);
  } else if (WARP && a.k * V <= 128) {
    mine = take_from_best_lanes<V, 4>(key, a.k, lane, room[threadIdx.x >> 5], first);
  } else {
#pragma unroll
    for (int r = 0; r < V; r += 8) sort8(key + r);
    mine = take_largest<V>(key, a.k, sub, glog, first);
  }
  const bool chosen = sub < a.k && Key<T>::alive(mine);
  const A e = chosen ? exp(Key<T>::value(mine) - top) : A(0);
  if (a.renormalize) sum = e;
  if (WARP) {
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) sum += __shfl_xor_sync(kFullMask, sum, m);
  } else {
    sum = group_sum(sum, glog);
  }
  if (live && sub < a.k) {
    const int64_t at = row * a.k + sub;
    a.experts[at] = chosen ? Key<T>::col(mine) : -1;
    static_cast<A*>(a.weights)[at] = chosen ? e / sum : A(0);
  }
}

// R rows per warp, one after the other, so that what comes after the choice -- exponentials, sums, divisions,
// stores -- is done once for all of them: lane r * (32 / R) + s ends up with the s-th choice of the r-th row.
// Needs k <= 32 / R and k V <= 128.  For 16-bit logits, from 16384 rows: 8.5 us against 8.8 there, 25 against
// 30 at 65536, slower below (too few warps); with fp32's 64-bit keys it needs 80 registers and loses
// (15.8 against 14.2 us at 16384 rows).
template <typename T, int V, int VE, int R>
__global__ void __launch_bounds__(kGateThreads) gate_rows_kernel(GateArgs a) {
  using A = typename Acc<T>::type;
  using K = typename Key<T>::type;
  constexpr int W = 32 / R;
  __shared__ __align__(16) K room[kGateThreads / 32][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, slot = lane % W;
  const int64_t row0 = (static_cast<int64_t>(blockIdx.x) * (kGateThreads >> 5) + warp) * R;
  T v[R][V];
#pragma unroll
  for (int r = 0; r < R; ++r)
    load_row<T, V, VE>(static_cast<const T*>(a.logits) + (row0 + r) * a.stride, row0 + r < a.N, a.E, lane, 5, v[r]);
  K mine = 0;
  A top = 0, sum = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    K key[V];
#pragma unroll
    for (int i = 0; i < V; i += 2) Key<T>::of(v[r] + i, column<VE>(i, lane, 5), column<VE>(i + 1, lane, 5), key + i);
    A row_top = 0, row_sum = 0;
    auto first = [&](K m) {
      row_top = Key<T>::alive(m) ? Key<T>::value(m) : A(0);
      if (!a.renormalize) {
#pragma unroll
        for (int i = 0; i < V; ++i) row_sum += exp(to_acc<T>(v[r][i]) - row_top);  // -inf adds 0
#pragma unroll
        for (int m2 = 1; m2 < 32; m2 <<= 1) row_sum += __shfl_xor_sync(kFullMask, row_sum, m2);
      }
    };
    K got = a.k * V <= 64 ? take_from_best_lanes<V, 2>(key, a.k, lane, room[warp], first)
                          : take_from_best_lanes<V, 4>(key, a.k, lane, room[warp], first);
    __syncwarp();  // `room` is read; the next row may write it
    got = shuffle(got, slot);
    if (lane / W == r) {
      mine = got;
      top = row_top;
      sum = row_sum;
    }
  }
  const bool chosen = slot < a.k && Key<T>::alive(mine);
  const A e = chosen ? exp(Key<T>::value(mine) - top) : A(0);
  if (a.renormalize) {
    sum = e;
#pragma unroll
    for (int m = 1; m < W; m <<= 1) sum += __shfl_xor_sync(kFullMask, sum, m);
  }
  const int64_t row = row0 + lane / W;
  if (row < a.N && slot < a.k) {
    const int64_t at = row * a.k + slot;
    a.experts[at] = chosen ? Key<T>::col(mine) : -1;
    static_cast<A*>(a.weights)[at] = chosen ? e / sum : A(0);
  }
}

// The gradient of renormalized weights, which is zero but on the chosen columns: R rows per warp are filled
// with zeros in wide stores and then, behind a barrier of the warp, written to by the lanes that hold the
// slots.  The weights sum to 1, so g_s - c is taken as sum_j w_j (g_s - g_j), which keeps its digits when one
// weight is nearly 1 and c nearly that slot's g.  65536 rows of 256 bf16, k = 8 (33.5 MB written, 5 us): 9 us, 13 us for assembling the rows in
// shared memory first.
template <typename T, int VE, int R>
__global__ void __launch_bounds__(kGateThreads) gate_backward_chosen_kernel(GateArgs a) {
  using A = typename Acc<T>::type;
  constexpr int W = 32 / R;
  const int lane = threadIdx.x & 31, slot = lane % W;
  const int64_t row0 = (static_cast<int64_t>(blockIdx.x) * (kGateThreads >> 5) + (threadIdx.x >> 5)) * R;
  const int64_t row = row0 + lane / W;
  A w = 0, g = 0;
  int col = -1;
  if (row < a.N && slot < a.k) {
    const int64_t at = row * a.k + slot;
    col = a.experts[at];  // (three independent loads)
    w = static_cast<const A*>(a.weights)[at];
    g = static_cast<const A*>(a.grad_weights)[at];
    if (col < 0 || col >= a.E) {
      col = -1;
      w = g = A(0);
    }
  }
  T* out = static_cast<T*>(a.grad_logits);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (row0 + r >= a.N) break;
    for (int c = lane * VE; c < a.E; c += 32 * VE) st_row<VE * sizeof(T)>(out + (row0 + r) * a.E + c, raw_none<VE * sizeof(T)>());
  }
  A d = 0;
  for (int s = 0; s < a.k; ++s) {
    const A ws = __shfl_sync(kFullMask, w, lane - slot + s), gs = __shfl_sync(kFullMask, g, lane - slot + s);
    d += ws * (g - gs);
  }
  __syncwarp();
  if (col >= 0) out[row * a.E + col] = from_acc<T>(w * d);
}

// Gradient of the logits, with c = sum_s w_s g_s:
//   renormalize: dl = w_s (g_s - c) on the chosen, 0 elsewhere;   otherwise: dl_j = p_j (g_j [chosen] - c).
// This kernel is the second; gate_backward_chosen_kernel is the first.  A chosen column's g_s - c is taken as
//   sum_j w_j (g_s - g_j) + r g_s,   r = the mass of the columns that were not chosen, summed from their own p,
// which keeps its digits when one weight is nearly 1 and c nearly that slot's g (and as it stands where c is further
// from g than half of it: a relative rms error of 6e-8 instead of 10e-8 for ordinary rows).  The slots' lanes mark
// their columns in the owners' masks; the owners store -p_j c everywhere in wide stores and then, behind a barrier of
// the warp, the slots' lanes w_s times the sum above on the chosen columns.  Bound by instruction issue: 65536 rows of
// 256, k = 8: 33.4 us in bf16, 35.3 in fp32 (8192 rows of 1000 fp32: 14.8); with a division per column, the columns' factors
// read back from shared memory and the logits loaded behind the slots 41.6, 44.3 and 25.5, and 31.6, 35.1 and 19.5
// before the rest's mass was summed at all.
template <typename T, int V, int VE>
__global__ void __launch_bounds__(kGateThreads) gate_backward_kernel(GateArgs a) {
  using A = typename Acc<T>::type;
  __shared__ uint32_t marks[kGateThreads];
  const int lane = threadIdx.x & 31, glog = a.glog, sub = lane & ((1 << glog) - 1);
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * (kGateThreads >> 5) + (threadIdx.x >> 5);
  const int64_t row = (warp << (5 - glog)) + (lane >> glog);
  const bool live = row < a.N;
  struct Slot {
    A w, g;
  };
  __shared__ Slot slots[kGateThreads];
  marks[threadIdx.x] = 0;
  T v[V];
  load_row<T, V, VE>(static_cast<const T*>(a.logits) + row * a.stride, live, a.E, sub, glog, v);

  A w = 0, g = 0;
  int col = -1;
  if (live && sub < a.k) {
    const int64_t at = row * a.k + sub;
    col = a.experts[at];  // (three independent loads)
    w = static_cast<const A*>(a.weights)[at];
    g = static_cast<const A*>(a.grad_weights)[at];
    if (col < 0 || col >= a.E) {
      col = -1;
      w = g = A(0);
    }
  }
  slots[threadIdx.x] = {w, g};
  __syncwarp();
  if (col >= 0) {  // the inverse of column()
    const int vec = col / VE, owner = vec & ((1 << glog) - 1), i = (vec >> glog) * VE + col % VE;
    atomicOr(&marks[threadIdx.x - sub + owner], 1u << i);
  }
  __syncwarp();
  const uint32_t picked = marks[threadIdx.x];  // of this lane's columns
  A c = 0, diff = 0;
  for (int s = 0; s < a.k; ++s) {
    const Slot other = slots[threadIdx.x - sub + s];
    c += other.w * other.g;
    diff += other.w * (g - other.g);
  }

  T* out = static_cast<T*>(a.grad_logits) + row * a.E;
  A p[V], top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    p[i] = to_acc<T>(v[i]);
    top = p[i] > top ? p[i] : top;
    nan |= isnan(p[i]);
  }
  for (int m = 1; m < (1 << glog); m <<= 1) {
    const A o = __shfl_xor_sync(kFullMask, top, m);
    top = o > top ? o : top;
  }
  const bool none = top == -INFINITY;
  A sum = nan ? A(NAN) : A(0), rest = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    p[i] = p[i] == -INFINITY ? A(0) : exp(p[i] - top);
    sum += p[i];
    rest += ((picked >> i) & 1u) ? A(0) : p[i];
  }
  sum = group_sum(sum, glog);
  rest = group_sum(rest, glog);
  const bool nothing = none && !isnan(sum);  // every logit is -inf: p[i] is 0
  rest = nothing ? A(0) : rest / sum;
  const A spread = nothing ? A(0) : (A(0) - c) / sum;  // two divisions a row instead of one a column
#pragma unroll
  for (int i = 0; i < V; i += VE) {
    const int col0 = column<VE>(i, sub, glog);
    if (!live || col0 >= a.E) continue;
    A d[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) d[j] = p[i + j] * spread;
    st_row<VE * sizeof(T)>(out + col0, narrow<T, VE * sizeof(T)>(d));
  }
  __syncwarp();
  if (col >= 0) {
    const A direct = g - c;  // the fewer roundings, where little cancels
    out[col] = from_acc<T>(w * (fabs(direct) >= A(0.5) * fabs(g) ? direct : diff + rest * g));
  }
}

int64_t blocks_for(int64_t rows, int64_t rows_per_block) { return (rows + rows_per_block - 1) / rows_per_block; }

template <typename T, int V, int VE>
int launch_gate(const GateArgs& a, bool backward, cudaStream_t stream) {
  const unsigned blocks = static_cast<unsigned>(blocks_for(a.N, kGateThreads >> a.glog));
  if (!backward) {
    constexpr int R = V == 8 ? 4 : 2;
    KernelTimer timer("gate_kernel", stream);
    bool many = false;
    if constexpr (sizeof(T) == 2) {
      many = a.glog == 5 && a.k * R <= 32 && a.k * V <= 128 && a.N >= kManyRows;
      if (many)
        gate_rows_kernel<T, V, VE, R>
            <<<static_cast<unsigned>(blocks_for(a.N, (kGateThreads >> 5) * R)), kGateThreads, 0, stream>>>(a);
    }
    if (many) {
    } else if (a.glog == 5) gate_kernel<T, V, VE, true><<<blocks, kGateThreads, 0, stream>>>(a);
    else if constexpr (V == 8) gate_kernel<T, V, VE, false><<<blocks, kGateThreads, 0, stream>>>(a);
  } else {
    KernelTimer timer("gate_backward_kernel", stream);
    gate_backward_kernel<T, V, VE><<<blocks, kGateThreads, 0, stream>>>(a);
  }
  TBE_CHECK_LAUNCH(backward ? "gate_backward_kernel" : "gate_kernel");
  return TBE_OK;
}

template <typename T, int VE, int R>
int launch_backward_chosen(const GateArgs& a, cudaStream_t stream) {
  {
    KernelTimer timer("gate_backward_chosen_kernel", stream);
    gate_backward_chosen_kernel<T, VE, R>
        <<<static_cast<unsigned>(blocks_for(a.N, (kGateThreads >> 5) * R)), kGateThreads, 0, stream>>>(a);
  }
  TBE_CHECK_LAUNCH("gate_backward_chosen_kernel");
  return TBE_OK;
}

template <typename T, int VE>
int launch_gate_width(const GateArgs& a, bool backward, cudaStream_t stream) {
  if (backward && a.renormalize)
    return a.k <= 8 ? launch_backward_chosen<T, VE, 4>(a, stream) : launch_backward_chosen<T, VE, 1>(a, stream);
  const int per_lane = (a.E + (1 << a.glog) - 1) >> a.glog;
  if (per_lane <= 8) return launch_gate<T, 8, VE>(a, backward, stream);
  if (per_lane <= 16) return launch_gate<T, 16, VE>(a, backward, stream);
  return launch_gate<T, 32, VE>(a, backward, stream);
}

template <typename T>
int launch_gate_type(const GateArgs& a, bool backward, cudaStream_t stream) {
  // 16-byte loads where every row starts on 16 bytes and ends on a vector; else one value at a time
  constexpr int VE = 16 / sizeof(T);
  const uint64_t bits = addr_bits(a.logits) | addr_bits(a.grad_logits) |
                        (a.N > 1 ? static_cast<uint64_t>(a.stride) * sizeof(T) : 0);
  if (bits % 16 == 0 && a.E % VE == 0) return launch_gate_width<T, VE>(a, backward, stream);
  return launch_gate_width<T, 1>(a, backward, stream);
}

int run_gate(const char* who, GateArgs a, int dtype, bool backward, cudaStream_t stream) {
  const bool reads_logits = !(backward && a.renormalize);
  if (!reads_logits) {  // nor do they decide anything
    a.logits = nullptr;
    a.stride = 0;
  }
  TBE_REQUIRE(a.N < (1ll << 31), "%s: N must be below 2^31", who);
  TBE_REQUIRE(a.N >= 0 && a.E > 0 && a.E <= kGateMaxExperts, "%s: the number of experts must be 1..%d", who,
              kGateMaxExperts);
  TBE_REQUIRE(a.k > 0 && a.k <= a.E && a.k <= kGateMaxK, "%s: k must be 1..min(E, %d)", who, kGateMaxK);
  TBE_REQUIRE(known_dtype(dtype), "%s: bad dtype %d", who, dtype);
  TBE_REQUIRE(a.N <= 1 || a.stride >= 0, "%s: negative row stride", who);
  if (a.N == 0) return TBE_OK;
  TBE_REQUIRE((a.logits || !reads_logits) && a.weights && a.experts, "%s: null pointer argument", who);
  TBE_REQUIRE(!backward || (a.grad_weights && a.grad_logits), "%s: null pointer argument", who);
  TBE_REQUIRE(aligned_to(any_elem_size(dtype), a.logits, a.grad_logits) &&
                  aligned_to(acc_size(dtype), a.weights, a.grad_weights) && aligned_to(4, a.experts),
              "%s: a pointer is not aligned to its elements", who);
  // lanes per row: eight values each (the narrowest group reads 16-bit rows as whole vectors), and a lane
  // for every slot
  a.glog = 0;
  while (a.glog < 5 && ((8 << a.glog) < a.E || (1 << a.glog) < a.k)) ++a.glog;
  switch (dtype) {
    case TBE_F16: return launch_gate_type<__half>(a, backward, stream);
    case TBE_BF16: return launch_gate_type<__nv_bfloat16>(a, backward, stream);
    case TBE_F32: return launch_gate_type<float>(a, backward, stream);
    default: return launch_gate_type<double>(a, backward, stream);
  }
}

}  // namespace
}  // namespace tbe

extern "C" int tbe_expert_gate(const void* logits, int64_t row_stride, void* weights, int32_t* experts, int64_t N,
                               int64_t E, int64_t k, int dtype, int renormalize, void* stream) {
  using namespace tbe;
  TBE_REQUIRE(E > 0 && E <= kGateMaxExperts && k > 0 && k <= kGateMaxK,
              "tbe_expert_gate: E must be 1..%d and k 1..%d", kGateMaxExperts, kGateMaxK);
  GateArgs a{logits, row_stride, weights, experts, N, static_cast<int>(E), static_cast<int>(k), 0, renormalize != 0,
             nullptr, nullptr};
  return run_gate("tbe_expert_gate", a, dtype, false, static_cast<cudaStream_t>(stream));
}

extern "C" int tbe_expert_gate_backward(const void* grad_weights, const void* logits, int64_t row_stride,
                                        const void* weights, const int32_t* experts, void* grad_logits, int64_t N,
                                        int64_t E, int64_t k, int dtype, int renormalize, void* stream) {
  using namespace tbe;
  TBE_REQUIRE(E > 0 && E <= kGateMaxExperts && k > 0 && k <= kGateMaxK,
              "tbe_expert_gate_backward: E must be 1..%d and k 1..%d", kGateMaxExperts, kGateMaxK);
  GateArgs a{logits, row_stride, const_cast<void*>(weights), const_cast<int32_t*>(experts), N, static_cast<int>(E),
             static_cast<int>(k), 0, renormalize != 0, grad_weights, grad_logits};
  return run_gate("tbe_expert_gate_backward", a, dtype, true, static_cast<cudaStream_t>(stream));
}
