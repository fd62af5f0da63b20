// The 2-norm over a list of gradients, and the gradients scaled down to a largest norm.
//
//   n = sqrt(sum over all tensors of g^2);   c = min(1, max_norm / (n + eps));   g <- c * g
//
// A list is cut into chunks of kChunk elements, dealt to a grid that fills the GPU; every CTA sums its
// chunks' squares in fp64 into one partial, and the kernel that needs the norm adds the partials in their
// order, so the result is the same from run to run and no counter has to be cleared between calls.  The
// table of tensors travels in the kernel's parameters: no copy to the device, nothing to keep alive, and
// a captured graph holds it.  Lists that are too long for one launch take several.
//
// Bound by HBM.  The norm has to be known before the first element is scaled, so a list larger than L2 is
// read twice; the scaling pass runs through the chunks backwards, so that what the norm pass read last is
// still in L2.  In place and with c == 1 there is nothing to store and the second pass ends at once.
// 200 M bf16 elements: 68 us for the norm (400 MB, 5.9 TB/s) and 123 us for the scaling (800 MB, 6.5 TB/s);
// 300 M fp32 elements below the limit: 175 us (1.2 GB, 6.9 TB/s) and 3.
#include <cooperative_groups.h>

#include <algorithm>
#include <new>
#include <utility>

#include "tbe_elem.cuh"

namespace tbe {
namespace {

namespace cg = cooperative_groups;

constexpr int kClipThreads = 256;
constexpr int kClipBlocksPerSM = 8;   // norm pass (32 registers)
// Scaling pass (80 registers, four vectors in flight): all resident, or the sweep would not run backwards.
// 200 M bf16 elements: 123 us; five CTAs with two vectors 125, six with one 141.
constexpr int kScaleBlocksPerSM = 3;
// Elements a CTA takes at a time.  200 M bf16 elements in 120 tensors, norm + scaling: 8192 79 + 132 us,
// 16384 68 + 123, 32768 74 + 125, 65536 72 + 129.
constexpr int kChunk = 16384;
constexpr int kSmallChunk = 1024;  // elements per warp of the one-kernel form
constexpr int kSmallMost = 1 << 17;  // elements; see grad_clip_small_kernel
constexpr int kSmallCluster = 8;
// Tensors in a launch's parameter block, 29 bytes each.  40 tensors in a block for 64: 9.4 us of host time a
// call, in one for 1024 10.7.
constexpr int kSmallTable = 64;
constexpr int kLargeTable = 1024;

template <int CAP>
struct Table {
  const void* src[CAP];
  void* dst[CAP];
  int64_t n[CAP];
  int32_t first[CAP];  // first chunk of the tensor
  uint8_t dtype[CAP];
  int32_t count, chunks;
};

template <int CAP>
__device__ __forceinline__ int tensor_of(const Table<CAP>& t, int chunk) {
  int lo = 0, hi = t.count;  // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Sum of the squares of a vector.  fp32 and fp64 values are squared in fp64.  Sixteen-bit values are
// squared and summed over the vector in fp32 (eight terms, relative error 2^-21) unless a square leaves
// fp32's range, which only bfloat16 reaches; then in fp64 too.
template <typename T, int VB>
__device__ __forceinline__ double sum_squares(const Raw<VB>& r) {
  constexpr int N = VB / sizeof(T);
  typename Acc<T>::type e[N];
  expand<T, VB>(r, e);
  if constexpr (sizeof(T) == 2) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += e[i] * e[i];
    // in the range [1e-24, 1e38] no term that counts has lost digits; NaN and inf take the slow way and stay
    if (s >= 1e-24f && s <= 1e38f) return s;
  }
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) d += static_cast<double>(e[i]) * static_cast<double>(e[i]);
  return d;
}

// How the summing pass loads: ReadOnly where the kernel writes none of the tensors, Ordinary where it goes on to scale
// them (the read-only path is only for memory that nothing writes while the kernel runs).
struct ReadOnly {
  template <typename T>
  __device__ static __forceinline__ Raw<sizeof(T)> one(const T* p) {
    return ld_stream<sizeof(T)>(p);
  }
  __device__ static __forceinline__ Raw<16> vector(const void* p, uint64_t policy) { return ld_stream_hint<16>(p, policy); }
};
struct Ordinary {
  template <typename T>
  __device__ static __forceinline__ Raw<sizeof(T)> one(const T* p) {
    const T v = *p;
    Raw<sizeof(T)> r;
    memcpy(&r, &v, sizeof(T));
    return r;
  }
  __device__ static __forceinline__ Raw<16> vector(const void* p, uint64_t policy) { return ld_rw_hint<16>(p, policy); }
};

// By `threads` threads of which this one is `me`.
template <typename LOADS, typename T>
__device__ double chunk_squares(const T* p, int n, int me, int threads, uint64_t policy) {
  constexpr int NV = 16 / sizeof(T), U = 4;
  const int head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(T)));
  const int nvec = (n - head) / NV, tail = head + nvec * NV;
  double s = 0.0;
  for (int i = me; i < head; i += threads) s += sum_squares<T, sizeof(T)>(LOADS::one(p + i));
  for (int i = tail + me; i < n; i += threads) s += sum_squares<T, sizeof(T)>(LOADS::one(p + i));
  const T* q = p + head;
  for (int v = me; v < nvec; v += threads * U) {
    Raw<16> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = v + u * threads;
      r[u] = i < nvec ? LOADS::vector(q + static_cast<int64_t>(i) * NV, policy) : raw_none<16>();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) s += sum_squares<T, 16>(r[u]);
  }
  return s;
}

// Sum over the CTA in a fixed order; every thread gets it.
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kClipThreads / 32];
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) v += __shfl_xor_sync(kFullMask, v, m);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kClipThreads / 32; ++w) s += part[w];
  __syncthreads();
  return s;
}

// The elements of chunk c, in chunks of `chunk` elements: tensor, first element, number.
struct Piece {
  int tensor;
  int64_t at;
  int n;
};
template <int CAP>
__device__ __forceinline__ Piece piece_of(const Table<CAP>& t, int c, int chunk, int tensor) {
  Piece p;
  p.tensor = tensor;
  p.at = static_cast<int64_t>(c - t.first[p.tensor]) * chunk;
  const int64_t left = t.n[p.tensor] - p.at;
  p.n = static_cast<int>(left < chunk ? left : chunk);
  return p;
}

template <typename LOADS, int CAP>
__device__ __forceinline__ double piece_squares(const Table<CAP>& t, const Piece& p, int me, int threads, uint64_t policy) {
  const void* src = t.src[p.tensor];
  switch (t.dtype[p.tensor]) {
    case TBE_F16: return chunk_squares<LOADS>(static_cast<const __half*>(src) + p.at, p.n, me, threads, policy);
    case TBE_BF16: return chunk_squares<LOADS>(static_cast<const __nv_bfloat16*>(src) + p.at, p.n, me, threads, policy);
    case TBE_F32: return chunk_squares<LOADS>(static_cast<const float*>(src) + p.at, p.n, me, threads, policy);
    default: return chunk_squares<LOADS>(static_cast<const double*>(src) + p.at, p.n, me, threads, policy);
  }
}

// Chunks from `keep` on stay in L2 for the scaling pass, which begins with them; the others pass through.
template <int CAP>
__global__ void __launch_bounds__(kClipThreads) grad_norm_kernel(const __grid_constant__ Table<CAP> t, double* partial, int keep) {
  const uint64_t pass = l2_policy_evict_first(), stay = l2_policy_evict_normal();
  double s = 0.0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x)
    s += piece_squares<ReadOnly>(t, piece_of(t, c, kChunk, tensor_of(t, c)), threadIdx.x, kClipThreads, c < keep ? pass : stay);
  s = block_sum(s);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__device__ __forceinline__ double fold(const double* partial, int n) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kClipThreads) s += partial[i];
  return sqrt(block_sum(s));
}

__global__ void __launch_bounds__(kClipThreads) grad_norm_finish_kernel(const double* partial, int n, float* norm) {
  const double r = fold(partial, n);
  if (threadIdx.x == 0) *norm = static_cast<float>(r);
}

// The factor as a product of two in the accumulator's type, the second a power of two and 1 unless the first
// alone would be near the end of fp32's range: an element times a factor of 1e-50 need not be 0.
template <typename A>
struct Split {
  A a, b;
};
template <typename A>
__device__ __forceinline__ Split<A> split(double f) {
  if (sizeof(A) == 8 || !(f > 0.0 && f < 0x1p-60)) return {static_cast<A>(f), A(1)};
  const int m = min(126, -ilogb(f) / 2);  // both halves, and the product in between, stay in range
  return {static_cast<A>(ldexp(f, m)), static_cast<A>(ldexp(1.0, -m))};
}

template <int U, typename T>
__device__ void scale_chunk(const T* src, T* dst, int n, double c, int me, int threads, uint64_t policy) {
  using A = typename Acc<T>::type;
  constexpr int NV = 16 / sizeof(T);
  const Split<A> f = split<A>(c);
  const uintptr_t s = reinterpret_cast<uintptr_t>(src), d = reinterpret_cast<uintptr_t>(dst);
  if ((s ^ d) & 15) {  // no vector of one is a vector of the other (50 M bf16 elements: 185 us, 32 for aligned ones)
    for (int i = me; i < n; i += threads) dst[i] = from_acc<T>(to_acc<T>(src[i]) * f.a * f.b);
    return;
  }
  const int head = min(n, static_cast<int>((16 - (s & 15)) & 15) / static_cast<int>(sizeof(T)));
  const int nvec = (n - head) / NV, tail = head + nvec * NV;
  for (int i = me; i < head; i += threads) dst[i] = from_acc<T>(to_acc<T>(src[i]) * f.a * f.b);
  for (int i = tail + me; i < n; i += threads) dst[i] = from_acc<T>(to_acc<T>(src[i]) * f.a * f.b);
  for (int v = me; v < nvec; v += threads * U) {
    Raw<16> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = v + u * threads;
      if (i < nvec) r[u] = ld_rw_hint<16>(src + head + static_cast<int64_t>(i) * NV, policy);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = v + u * threads;
      if (i < nvec) {
        A x[NV];
        expand<T, 16>(r[u], x);
#pragma unroll
        for (int j = 0; j < NV; ++j) x[j] = x[j] * f.a * f.b;
        st_row_hint<16>(dst + head + static_cast<int64_t>(i) * NV, narrow<T, 16>(x), policy);
      }
    }
  }
}

template <int U, int CAP>
__device__ __forceinline__ void piece_scale(const Table<CAP>& t, const Piece& p, double f, int me, int threads, uint64_t policy) {
  const void* src = t.src[p.tensor];
  void* dst = t.dst[p.tensor];
  switch (t.dtype[p.tensor]) {
    case TBE_F16:
      return scale_chunk<U>(static_cast<const __half*>(src) + p.at, static_cast<__half*>(dst) + p.at, p.n, f, me, threads, policy);
    case TBE_BF16:
      return scale_chunk<U>(static_cast<const __nv_bfloat16*>(src) + p.at, static_cast<__nv_bfloat16*>(dst) + p.at, p.n, f, me,
                         threads, policy);
    case TBE_F32:
      return scale_chunk<U>(static_cast<const float*>(src) + p.at, static_cast<float*>(dst) + p.at, p.n, f, me, threads, policy);
    default:
      return scale_chunk<U>(static_cast<const double*>(src) + p.at, static_cast<double*>(dst) + p.at, p.n, f, me, threads, policy);
  }
}

__device__ __forceinline__ double factor(double norm, double max_norm, double eps) {
  const double f = max_norm / (norm + eps);
  return f > 1.0 ? 1.0 : f;  // NaN stays
}

template <int CAP>
__global__ void __launch_bounds__(kClipThreads, kScaleBlocksPerSM) grad_scale_kernel(const __grid_constant__ Table<CAP> t, const double* partial,
                                                                     int parts, double max_norm, double eps, bool in_place,
                                                                     float* norm) {
  const double n = fold(partial, parts);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
  const double f = factor(n, max_norm, eps);
  if (in_place && f == 1.0) return;
  const uint64_t pass = l2_policy_evict_first();
  for (int c = t.chunks - 1 - blockIdx.x; c >= 0; c -= gridDim.x)
    piece_scale<4>(t, piece_of(t, c, kChunk, tensor_of(t, c)), f, threadIdx.x, kClipThreads, pass);
}

// The tensor of every chunk of a short list: in a kernel of a few microseconds a search in the table is a
// chain of loads that all miss the constant cache.
template <int CAP>
struct Owners {
  uint16_t tensor[CAP + kSmallMost / kSmallChunk];
};

// A short list in one launch: a cluster of CTAs, a warp per kSmallChunk elements, the CTAs' sums exchanged
// through distributed shared memory between the two passes.  The second launch of the two-kernel form costs
// the host 4 us and the GPU a gap of about 1.5; on the GPU itself (one kernel / the two without the gap) 40 fp32
// tensors of 1000 elements in all take 5.0 / 5.7 us, of 65536 7.5 / 5.8, of 131072 7.2 / 5.7, of 262144 11.0 / 6.7.
// (1024 threads leave 64 registers; 32 bytes spill.)
template <int CAP>
__global__ void __launch_bounds__(1024) grad_clip_small_kernel(const __grid_constant__ Table<CAP> t,
                                                               const __grid_constant__ Owners<CAP> owners, bool scale,
                                                               double max_norm, double eps, bool in_place, float* norm) {
  __shared__ double part[32], own;
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = static_cast<int>(cluster.block_rank()) * 32 + warp, step = kSmallCluster * 32;
  const uint64_t policy = l2_policy_evict_normal();
  double s = 0.0;
  Piece own_piece{0, 0, 0};  // the first of this warp's pieces, which is all it has unless the list is long
  if (first < t.chunks) {
    own_piece = piece_of(t, first, kSmallChunk, owners.tensor[first]);
    s = piece_squares<Ordinary>(t, own_piece, lane, 32, policy);
  }
  for (int c = first + step; c < t.chunks; c += step)
    s += piece_squares<Ordinary>(t, piece_of(t, c, kSmallChunk, owners.tensor[c]), lane, 32, policy);
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) s += __shfl_xor_sync(kFullMask, s, m);
  if (lane == 0) part[warp] = s;
  __syncthreads();
  if (warp == 0) {
    s = part[lane];
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) s += __shfl_xor_sync(kFullMask, s, m);
    if (lane == 0) own = s;
  }
  cluster.sync();  // every CTA's sum is in place
  double total = 0.0;
#pragma unroll
  for (int r = 0; r < kSmallCluster; ++r) total += *cluster.map_shared_rank(&own, r);
  auto read = cluster.barrier_arrive();  // this CTA has read the others' sums
  const double n = sqrt(total);
  if (first == 0 && lane == 0) *norm = static_cast<float>(n);
  const double f = factor(n, max_norm, eps);
  if (scale && !(in_place && f == 1.0)) {
    if (first < t.chunks) piece_scale<2>(t, own_piece, f, lane, 32, policy);
    for (int c = first + step; c < t.chunks; c += step)
      piece_scale<2>(t, piece_of(t, c, kSmallChunk, owners.tensor[c]), f, lane, 32, policy);
  }
  cluster.barrier_wait(std::move(read));  // nobody reads a CTA's sum after it has left
}

// One launch's worth of the list: tensors [from, to), at most CAP of them, empty ones left out.
template <int CAP>
bool fill(Table<CAP>& t, const void* const* src, void* const* dst, const int64_t* n, const int32_t* dtype, int from, int to,
          int chunk) {
  t.count = 0;
  int64_t chunks = 0;
  for (int i = from; i < to; ++i) {
    if (n[i] == 0) continue;
    t.src[t.count] = src[i];
    t.dst[t.count] = dst ? dst[i] : nullptr;
    t.n[t.count] = n[i];
    t.first[t.count] = static_cast<int32_t>(chunks);
    t.dtype[t.count] = static_cast<uint8_t>(dtype[i]);
    ++t.count;
    chunks += (n[i] + chunk - 1) / chunk;
    if (chunks > 0x7fff0000) return false;
  }
  t.chunks = static_cast<int32_t>(chunks);
  return true;
}

// The chunk from which the rest of the list fits into half of L2.  (200 M bf16 elements, norm + scaling:
// 67 + 127 us with nothing kept, 68 + 122 with 63 MB, 71 + 120 with 126 MB, 79 + 120 with everything.)
template <int CAP>
int first_kept_chunk(const Table<CAP>& t) {
  int64_t room = device_l2_bytes() / 2;
  int c = t.chunks;
  for (int k = t.count - 1; k >= 0 && room > 0; --k) {
    const int64_t bytes = kChunk * static_cast<int64_t>(any_elem_size(t.dtype[k])), n = c - t.first[k];
    const int64_t fit = room / bytes;
    c -= static_cast<int>(n < fit ? n : fit);
    room = n <= fit ? room - n * bytes : 0;
  }
  return c;
}

int launch_grid(int64_t chunks, int blocks_per_sm) {
  const int64_t most = static_cast<int64_t>(device_sm_count()) * blocks_per_sm;
  return static_cast<int>(chunks < most ? (chunks > 0 ? chunks : 1) : most);
}

int check_list(const char* who, const void* const* src, const int64_t* n, const int32_t* dtype, int64_t count) {
  TBE_REQUIRE(count >= 0 && count < (1ll << 24), "%s: the number of tensors must be 0..2^24-1", who);
  TBE_REQUIRE(count == 0 || (src && n && dtype), "%s: null pointer argument", who);
  for (int64_t i = 0; i < count; ++i) {
    TBE_REQUIRE(known_dtype(dtype[i]), "%s: tensor %lld has bad dtype %d", who, static_cast<long long>(i), dtype[i]);
    TBE_REQUIRE(n[i] >= 0 && n[i] < (1ll << 44), "%s: tensor %lld has a bad size", who, static_cast<long long>(i));
    TBE_REQUIRE(n[i] == 0 || src[i], "%s: tensor %lld is a null pointer", who, static_cast<long long>(i));
    TBE_REQUIRE(addr_bits(src[i]) % any_elem_size(dtype[i]) == 0, "%s: tensor %lld is not aligned to its elements", who,
                static_cast<long long>(i));
  }
  return TBE_OK;
}

// Stores of one tensor must not meet loads or stores of another: the chunks run in no order.
struct Span {
  uint64_t begin, end;
  int64_t index;
};
int check_apart(const void* const* src, void* const* dst, const int64_t* n, const int32_t* dtype, int64_t count) {
  Span* spans = new (std::nothrow) Span[static_cast<size_t>(count) + 1];
  if (!spans) return fail(TBE_ERR_INVALID_ARGUMENT, "tbe_grad_clip: out of host memory");
  int64_t m = 0;
  for (int64_t i = 0; i < count; ++i)
    if (n[i] > 0) {
      const uint64_t b = addr_bits(dst[i]);
      spans[m++] = {b, b + static_cast<uint64_t>(n[i]) * any_elem_size(dtype[i]), i};
    }
  std::sort(spans, spans + m, [](const Span& x, const Span& y) { return x.begin < y.begin; });
  int64_t bad = -1;
  for (int64_t j = 1; j < m && bad < 0; ++j)
    if (spans[j].begin < spans[j - 1].end) bad = spans[j].index;
  for (int64_t i = 0; i < count && bad < 0; ++i) {
    if (n[i] == 0 || src[i] == dst[i]) continue;  // in place: the stores above are its loads
    const uint64_t b = addr_bits(src[i]), e = b + static_cast<uint64_t>(n[i]) * any_elem_size(dtype[i]);
    const Span* s = std::lower_bound(spans, spans + m, b, [](const Span& x, uint64_t v) { return x.end <= v; });
    if (s != spans + m && s->begin < e) bad = i;
  }
  delete[] spans;
  if (bad >= 0)
    return fail(TBE_ERR_INVALID_ARGUMENT, "tbe_grad_clip: tensor %lld shares memory with another one that is written",
                static_cast<long long>(bad));
  return TBE_OK;
}

template <int CAP>
int norm_launches(const void* const* src, const int64_t* n, const int32_t* dtype, int count, double* partial, int* parts,
                  cudaStream_t stream) {
  static_assert(sizeof(Table<CAP>) + 64 <= 32764, "the table does not fit into a kernel's parameters");
  *parts = 0;
  Table<CAP> t;
  int from = 0;
  do {
    const int to = count - from < CAP ? count : from + CAP;
    TBE_REQUIRE(fill(t, src, nullptr, n, dtype, from, to, kChunk), "tbe_grad_norm: too many elements");
    const int grid = launch_grid(t.chunks, kClipBlocksPerSM);
    {
      KernelTimer timer("grad_norm_kernel", stream);
      grad_norm_kernel<CAP><<<grid, kClipThreads, 0, stream>>>(t, partial + *parts, to == count ? first_kept_chunk(t) : t.chunks);
    }
    TBE_CHECK_LAUNCH("grad_norm_kernel");
    *parts += grid;
    from = to;
  } while (from < count);
  return TBE_OK;
}

template <int CAP>
int scale_launches(const void* const* src, void* const* dst, const int64_t* n, const int32_t* dtype, int count,
                   const double* partial, int parts, double max_norm, double eps, bool in_place, float* norm,
                   cudaStream_t stream) {
  Table<CAP> t;
  // backwards over the launches too
  int to = count;
  do {
    const int from = to > CAP ? (to - 1) / CAP * CAP : 0;
    TBE_REQUIRE(fill(t, src, dst, n, dtype, from, to, kChunk), "tbe_grad_clip: too many elements");
    {
      KernelTimer timer("grad_scale_kernel", stream);
      grad_scale_kernel<CAP><<<launch_grid(t.chunks, kScaleBlocksPerSM), kClipThreads, 0, stream>>>(t, partial, parts, max_norm, eps, in_place,
                                                                                 norm);
    }
    TBE_CHECK_LAUNCH("grad_scale_kernel");
    norm = nullptr;
    to = from;
  } while (to > 0);
  return TBE_OK;
}

// Whether the list is short enough for the one-kernel form.
bool is_small(const int64_t* n, int64_t count) {
  if (count > kLargeTable) return false;
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) total += n[i];
  return total <= kSmallMost;
}

template <int CAP>
int small_launch(const void* const* src, void* const* dst, const int64_t* n, const int32_t* dtype, int count, bool scale,
                 double max_norm, double eps, bool in_place, float* norm, cudaStream_t stream) {
  Table<CAP> t;
  Owners<CAP> owners;
  static_assert(sizeof(t) + sizeof(owners) + 64 <= 32764, "the tables do not fit into a kernel's parameters");
  fill(t, src, dst, n, dtype, 0, count, kSmallChunk);  // at most CAP + kSmallMost / kSmallChunk chunks
  for (int k = 0; k < t.count; ++k)
    for (int c = t.first[k]; c < (k + 1 < t.count ? t.first[k + 1] : t.chunks); ++c) owners.tensor[c] = static_cast<uint16_t>(k);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kSmallCluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(kSmallCluster);
  cfg.blockDim = dim3(1024);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  {
    KernelTimer timer("grad_clip_small_kernel", stream);
    TBE_CUDA_TRY(cudaLaunchKernelEx(&cfg, grad_clip_small_kernel<CAP>, t, owners, scale, max_norm, eps, in_place, norm));
  }
  TBE_CHECK_LAUNCH("grad_clip_small_kernel");
  return TBE_OK;
}
int run_small(const void* const* src, void* const* dst, const int64_t* n, const int32_t* dtype, int count, bool scale,
              double max_norm, double eps, bool in_place, float* norm, cudaStream_t stream) {
  return count <= kSmallTable
             ? small_launch<kSmallTable>(src, dst, n, dtype, count, scale, max_norm, eps, in_place, norm, stream)
             : small_launch<kLargeTable>(src, dst, n, dtype, count, scale, max_norm, eps, in_place, norm, stream);
}

int64_t launches_of(int64_t count) { return count <= kLargeTable ? 1 : (count + kLargeTable - 1) / kLargeTable; }

}  // namespace
}  // namespace tbe

extern "C" int64_t tbe_grad_norm_workspace_bytes(int64_t count) {
  using namespace tbe;
  if (count < 0 || count >= (1ll << 24))
    return fail(TBE_ERR_INVALID_ARGUMENT, "tbe_grad_norm_workspace_bytes: the number of tensors must be 0..2^24-1");
  return launches_of(count) * device_sm_count() * kClipBlocksPerSM * static_cast<int64_t>(sizeof(double));
}

namespace tbe {
namespace {
int check_workspace(const char* who, int64_t count, const void* workspace, int64_t workspace_bytes) {
  const int64_t need = tbe_grad_norm_workspace_bytes(count);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(TBE_ERR_WORKSPACE_TOO_SMALL, "%s: workspace of %lld bytes, %lld needed", who,
                static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  TBE_REQUIRE(addr_bits(workspace) % 8 == 0, "%s: the workspace must be 8-byte aligned", who);
  return TBE_OK;
}

int run_norm(const void* const* src, const int64_t* n, const int32_t* dtype, int64_t count, double* partial, int* parts,
             cudaStream_t stream) {
  return count <= kSmallTable ? norm_launches<kSmallTable>(src, n, dtype, static_cast<int>(count), partial, parts, stream)
                              : norm_launches<kLargeTable>(src, n, dtype, static_cast<int>(count), partial, parts, stream);
}
}  // namespace
}  // namespace tbe

extern "C" int tbe_grad_norm(const void* const* tensors, const int64_t* numels, const int32_t* dtypes, int64_t count,
                             float* norm, void* workspace, int64_t workspace_bytes, void* stream_v) {
  using namespace tbe;
  TBE_REQUIRE(norm, "tbe_grad_norm: null pointer argument");
  TBE_REQUIRE(aligned_to(4, norm), "tbe_grad_norm: norm is not aligned to its elements");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (const int rc = check_list("tbe_grad_norm", tensors, numels, dtypes, count)) return rc;
  if (const int rc = check_workspace("tbe_grad_norm", count, workspace, workspace_bytes)) return rc;
  if (is_small(numels, count))
    return run_small(tensors, nullptr, numels, dtypes, static_cast<int>(count), false, 0.0, 0.0, false, norm, stream);
  int parts = 0;
  if (const int rc = run_norm(tensors, numels, dtypes, count, static_cast<double*>(workspace), &parts, stream)) return rc;
  {
    KernelTimer timer("grad_norm_finish_kernel", stream);
    grad_norm_finish_kernel<<<1, kClipThreads, 0, stream>>>(static_cast<const double*>(workspace), parts, norm);
  }
  TBE_CHECK_LAUNCH("grad_norm_finish_kernel");
  return TBE_OK;
}

extern "C" int tbe_grad_clip(const void* const* tensors, void* const* outputs, const int64_t* numels, const int32_t* dtypes,
                             int64_t count, double max_norm, double eps, float* norm, void* workspace,
                             int64_t workspace_bytes, void* stream_v) {
  using namespace tbe;
  TBE_REQUIRE(norm && (count == 0 || outputs), "tbe_grad_clip: null pointer argument");
  TBE_REQUIRE(aligned_to(4, norm), "tbe_grad_clip: norm is not aligned to its elements");
  TBE_REQUIRE(max_norm >= 0.0 && eps >= 0.0, "tbe_grad_clip: max_norm and eps must not be negative");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (const int rc = check_list("tbe_grad_clip", tensors, numels, dtypes, count)) return rc;
  bool in_place = true;
  for (int64_t i = 0; i < count; ++i) {
    if (numels[i] == 0) continue;
    TBE_REQUIRE(outputs[i] && addr_bits(outputs[i]) % any_elem_size(dtypes[i]) == 0,
                "tbe_grad_clip: output %lld is null or not aligned to its elements", static_cast<long long>(i));
    in_place &= outputs[i] == tensors[i];
  }
  if (const int rc = check_apart(tensors, outputs, numels, dtypes, count)) return rc;
  if (const int rc = check_workspace("tbe_grad_clip", count, workspace, workspace_bytes)) return rc;
  if (is_small(numels, count))
    return run_small(tensors, outputs, numels, dtypes, static_cast<int>(count), true, max_norm, eps, in_place, norm, stream);
  int parts = 0;
  if (const int rc = run_norm(tensors, numels, dtypes, count, static_cast<double*>(workspace), &parts, stream)) return rc;
  const double* partial = static_cast<const double*>(workspace);
  return count <= kSmallTable ? scale_launches<kSmallTable>(tensors, outputs, numels, dtypes, static_cast<int>(count), partial,
                                                            parts, max_norm, eps, in_place, norm, stream)
                              : scale_launches<kLargeTable>(tensors, outputs, numels, dtypes, static_cast<int>(count), partial,
                                                            parts, max_norm, eps, in_place, norm, stream);
}
