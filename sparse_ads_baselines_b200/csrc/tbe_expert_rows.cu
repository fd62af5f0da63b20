// Samples sorted by expert and back.
//
//   plan      experts[N][k] -> a stable counting sort of the M = N*k choices by expert:
//             positions[t][s] = the row that choice (t, s) takes in expert order, order = its inverse,
//             offsets[E+1] = where every expert's rows begin.  Choices outside 0..E-1 sort behind all
//             experts; rows from offsets[E] ("kept") on belong to nobody.
//   dispatch  y[positions[t][s]] = x[t];  rows behind kept are zero
//   combine   out[t] = sum_s w[t][s] * y[positions[t][s]]   over the kept choices, slots ascending, fp32
//             sums (fp64 for fp64), rounded once.  Without weights it is also dispatch's gradient.
//   combine's gradient  dy[positions[t][s]] = w[t][s] * dout[t],  dw[t][s] = <dout[t], y[positions[t][s]]>
//
// Everything is indexed by sample, never by sorted row: a sample's row is read once and stored k times
// (or k rows are read and one stored), so the traffic is the algorithm's, no sum needs an atomic and the
// results do not depend on the order of anything.  A position outside the
// rows is skipped by every kernel, so a wrong plan cannot reach memory outside the tensors.
#include <cooperative_groups.h>

#include "tbe_elem.cuh"

namespace tbe {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int64_t kMaxEntries = 0x7fffffffll - 1024;  // 32-bit positions, and room for an index past the end
namespace cg = cooperative_groups;

// How many CTAs sort a plan, by its number of choices: one of 256 threads, one cluster of 1024-thread CTAs
// (totals exchanged through distributed shared memory), or a grid with a counting kernel in front (totals
// through global memory).  64 experts, us on the GPU (one / cluster / grid): 1024 choices 4.0 / 4.5 / 6.6,
// 2048 5.5 / 4.6 / 7.7, 65536 - / 10.2 / 12.8, 131072 - / 15.8 / 13.3, and a launch costs the host 4 us.
constexpr int kPlanOne = 1024;
constexpr int kPlanCluster = 8;
constexpr int kPlanClusterMost = 131072;
constexpr int64_t kFewVectors = 148 * 512;  // a quarter of the threads the GPU holds
constexpr int kPlanSlice = 8192;  // choices per CTA of the grid, at least
enum PlanMode { kOne, kCluster, kGrid };

// ---------------------------------------------------------------- plan
struct PlanArgs {
  const int32_t* experts;
  int32_t* offsets;
  int32_t* positions;
  int32_t* order;
  int32_t* counts;  // [ctas][E+1], two-kernel plan only
  int32_t M, E, slice;
  int32_t bits;  // of E + 1, the bin of a lane without a choice
};

__device__ __forceinline__ int bin_of(int32_t id, int E) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(E) ? id : E; }

// Exclusive prefix sum of v[0..n) in shared memory, by the whole CTA; n <= kMaxExperts + 1.
__device__ void block_exclusive_scan(int32_t* v, int n, int32_t* warp_sums) {
  const int per = (n + blockDim.x - 1) / blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int begin = min(static_cast<int>(threadIdx.x) * per, n), end = min(begin + per, n);
  int32_t own = 0;
  for (int i = begin; i < end; ++i) own += v[i];
  int32_t scan = own;
  for (int m = 1; m < 32; m <<= 1) {
    const int32_t o = __shfl_up_sync(kFullMask, scan, m);
    if (lane >= m) scan += o;
  }
  if (lane == 31) warp_sums[warp] = scan;
  __syncthreads();
  int32_t ws = lane < warp ? warp_sums[lane] : 0;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) ws += __shfl_xor_sync(kFullMask, ws, m);
  int32_t before = scan - own + ws;
  for (int i = begin; i < end; ++i) {
    const int32_t x = v[i];
    v[i] = before;
    before += x;
  }
  __syncthreads();
}

// One CTA sorts its slice: every warp counts a contiguous part per bin, the parts are prefix-summed warp
// by warp, and a second pass in the same order places each choice behind the earlier ones of its bin.
// The order is therefore the stable one, whatever the atomics of the counting did.  Bound by latency (loads,
// barriers) and by what a warp issues per 32 choices, not by its 12 bytes per choice.
//   shared: hist[warps][E+1], start[E+1], before[E+1], own[E+1], 32 words
template <int MODE>
__global__ void __launch_bounds__(1024) plan_place_kernel(PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  const int E1 = a.E + 1, warps = blockDim.x >> 5, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int32_t* hist = plan_smem;
  int32_t* start = hist + warps * E1;  // where a bin begins
  int32_t* before = start + E1;        // choices of the bin in the CTAs in front of this one
  int32_t* own = before + E1;          // choices of the bin in this CTA
  int32_t* warp_sums = own + E1;
  const int64_t s0 = static_cast<int64_t>(blockIdx.x) * a.slice;
  const int begin = static_cast<int>(s0 < a.M ? s0 : a.M), len = min(a.slice, a.M - begin);
  const int part = ((len + warps - 1) / warps + 31) & ~31;
  const int wb = begin + min(warp * part, len), we = begin + min((warp + 1) * part, len);

  for (int i = threadIdx.x; i < warps * E1 + 2 * E1; i += blockDim.x) hist[i] = 0;
  __syncthreads();
#pragma unroll 4
  for (int i = wb + lane; i < we; i += 32) atomicAdd(&hist[warp * E1 + bin_of(__ldg(a.experts + i), a.E)], 1);
  if (MODE == kGrid) {
    const int n = gridDim.x * E1, mine = blockIdx.x * E1;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int32_t c = __ldg(a.counts + i);
      const int b = i % E1;
      if (c) {
        atomicAdd(&start[b], c);
        if (i < mine) atomicAdd(&before[b], c);
      }
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < E1; b += blockDim.x) {
    int32_t run = 0;
    for (int w0 = 0; w0 < warps; w0 += 8) {  // (warps is a multiple of 8)
      int32_t c[8];
#pragma unroll
      for (int w = 0; w < 8; ++w) c[w] = hist[(w0 + w) * E1 + b];
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        hist[(w0 + w) * E1 + b] = run;
        run += c[w];
      }
    }
    if (MODE == kOne) start[b] = run;
    if (MODE == kCluster) own[b] = run;
  }
  if (MODE == kCluster) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();  // every CTA's own totals are in place
    const int rank = static_cast<int>(cluster.block_rank());
    for (int b = threadIdx.x; b < E1; b += blockDim.x) {
      int32_t total = 0, front = 0;
#pragma unroll
      for (int c = 0; c < kPlanCluster; ++c) {
        const int32_t t = cluster.map_shared_rank(own, c)[b];
        total += t;
        if (c < rank) front += t;
      }
      start[b] = total;
      before[b] = front;
    }
    cluster.sync();  // nobody's totals are read any more
  } else {
    __syncthreads();
  }
  block_exclusive_scan(start, E1, warp_sums);
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < E1; b += blockDim.x) a.offsets[b] = start[b];
  if (MODE != kOne) {
    __syncthreads();
    for (int b = threadIdx.x; b < E1; b += blockDim.x) start[b] += before[b];
    __syncthreads();
  }

  int32_t* next = hist + warp * E1;
  int32_t ahead = wb + lane < we ? __ldg(a.experts + wb + lane) : 0;
  for (int i0 = wb; i0 < we; i0 += 32) {
    const int i = i0 + lane;
    const bool on = i < we;
    const int b = on ? bin_of(ahead, a.E) : E1;
    if (i + 32 < we) ahead = __ldg(a.experts + i + 32);
    unsigned peers = kFullMask;  // the lanes of the same bin (32768 choices, 64 experts: 9.4 us with match.any, 7.4 so)
    for (int bit = 0; bit < a.bits; ++bit) {
      const bool set = (b >> bit) & 1;
      const unsigned with = __ballot_sync(kFullMask, set);
      peers &= set ? with : ~with;
    }
    const int rank = __popc(peers & ((1u << lane) - 1));
    const int32_t first = on ? next[b] : 0;
    __syncwarp();
    if (on && rank == 0) next[b] = first + __popc(peers);
    __syncwarp();
    if (on) {
      const int32_t p = start[b] + first + rank;
      a.positions[i] = p;
      a.order[p] = i;
    }
  }
}

__global__ void __launch_bounds__(1024) plan_count_kernel(PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  const int E1 = a.E + 1;
  const int64_t s0 = static_cast<int64_t>(blockIdx.x) * a.slice;
  const int begin = static_cast<int>(s0 < a.M ? s0 : a.M), end = begin + min(a.slice, a.M - begin);
  for (int b = threadIdx.x; b < E1; b += blockDim.x) plan_smem[b] = 0;
  __syncthreads();
  for (int i = begin + threadIdx.x; i < end; i += blockDim.x) atomicAdd(&plan_smem[bin_of(__ldg(a.experts + i), a.E)], 1);
  __syncthreads();
  for (int b = threadIdx.x; b < E1; b += blockDim.x) a.counts[static_cast<int64_t>(blockIdx.x) * E1 + b] = plan_smem[b];
}

struct PlanShape {
  PlanMode mode;
  int ctas, slice;
};
PlanShape plan_shape(int64_t M) {
  if (M <= kPlanOne) return {kOne, 1, static_cast<int>(M)};
  if (M <= kPlanClusterMost) return {kCluster, kPlanCluster, static_cast<int>((M + kPlanCluster - 1) / kPlanCluster)};
  int64_t ctas = (M + kPlanSlice - 1) / kPlanSlice;
  if (ctas > 148) ctas = 148;
  return {kGrid, static_cast<int>(ctas), static_cast<int>((M + ctas - 1) / ctas)};
}

// ---------------------------------------------------------------- rows
struct RowArgs {
  const char* x;       // dispatch: rows by sample; combine: rows by position
  int64_t x_stride;    // bytes
  const int32_t* positions;
  const int32_t* kept;  // offsets + E
  const void* weights;  // [N][k] in the accumulator type, or NULL
  char* out;
  int64_t row_bytes;  // stride of position-ordered and freshly written rows
  int32_t M;
  int k;
  uint32_t nvec, per_row, items;  // vectors per row, threads per row, threads of this launch
  FastDiv div;                    // by per_row
};

__device__ __forceinline__ uint32_t kept_rows(const int32_t* kept, int32_t M) {
  const int32_t n = __ldg(kept);
  return static_cast<uint32_t>(n < 0 ? 0 : n > M ? M : n);
}

// The U vectors of a thread: first, and the distance between them.  In a row of at least 32 U vectors (TILED) a
// warp takes 32 U neighbouring ones, so that the distance is known at compile time and all of a thread's accesses
// to a row are one address and constants; in a shorter row they lie a U-th of it apart.
template <int VB, int U, bool TILED>
struct Vectors {
  uint32_t first, apart;
  __device__ __forceinline__ Vectors(uint32_t place, uint32_t per_row)
      : first(TILED ? (place >> 5) * (32 * U) + (place & 31) : place), apart(TILED ? 32 : per_row) {}
  __device__ __forceinline__ uint32_t at(int u) const { return first + u * apart; }
  __device__ __forceinline__ int64_t offset(int u) const {
    return TILED ? static_cast<int64_t>(first) * VB + u * 32 * VB : static_cast<int64_t>(at(u)) * VB;
  }
};

// A thread takes U vectors of one sample's row, so that a warp's loads stay contiguous and the positions are
// looked up once for all of them: U independent loads, then k stores each.
// 2048 rows of 8192 fp16, k = 2: 16 us for 101 MB (6.3 TB/s).  Rows that are only aligned to 4 bytes are
// bound by the load-store unit: 5003 of 1001 fp32, k = 6: 26 us for 140 MB (5.4 TB/s; 29 without TILED); to 2 bytes:
// 8192 of 2047 bf16, k = 4: 40 us, 27 for 2048.
template <int VB, int U, bool TILED>
__global__ void __launch_bounds__(256) dispatch_kernel(RowArgs a) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= a.items) return;
  const uint32_t t = fastdiv(i, a.div), place = i - t * a.per_row;
  const Vectors<VB, U, TILED> v(place, a.per_row);
  const char* src = a.x + t * a.x_stride;
  Raw<VB> r[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (v.at(u) < a.nvec) r[u] = ld_stream<VB>(src + v.offset(u));
  const uint32_t kept = kept_rows(a.kept, a.M), M = static_cast<uint32_t>(a.M);
  const int32_t* pos = a.positions + static_cast<int64_t>(t) * a.k;
  for (int s = 0; s < a.k; ++s) {
    const uint32_t p = static_cast<uint32_t>(__ldg(pos + s));
    if (p >= M) continue;
    char* dst = a.out + p * a.row_bytes;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v.at(u) < a.nvec) st_row<VB>(dst + v.offset(u), p < kept ? r[u] : raw_none<VB>());
  }
}

// The same U vectors, summed over the sample's rows; KB * U row loads are in flight together, in 64 registers
// (four CTAs per SM), which do not hold all of them in 16-bit types with 16-byte vectors: (U, KB) = (2, 4) spills 96
// bytes where it is not TILED (k > 2, rows of fewer than 64 vectors: 65536 of 256 bf16, k = 8, 55 us for a floor of
// 46), (4, 1) 8 or 40.  8192 rows of 2048 bf16, us for (KB, U) = (1, 4) / (2, 1) / (2, 2) / (4, 1) / (4, 2) / (8, 1):
// k = 1 10.8 / 16.5 / 12.7 / 19.5 / 13.8 / 23.8, k = 2 15.9 / 18.9 / 15.5 / 22.4 / 16.6 / 25.7, k = 4 25.7 / 28.8 /
// 24.5 / 26.6 / 23.4 / 30.2, k = 8 45.9 / 49.0 / 43.3 / 44.4 / 41.7 / 42.6 (302 MB: 7.2 TB/s with L2's help).
template <typename T, int VB, int U, int KB, bool TILED>
__global__ void __launch_bounds__(256, 4) combine_kernel(RowArgs a) {
  using A = typename Acc<T>::type;
  constexpr int NE = VB / sizeof(T);
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= a.items) return;
  const uint32_t t = fastdiv(i, a.div), place = i - t * a.per_row;
  const Vectors<VB, U, TILED> v(place, a.per_row);
  const int64_t at = static_cast<int64_t>(t) * a.k;
  const uint32_t kept = kept_rows(a.kept, a.M);
  A acc[U][NE];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < NE; ++e) acc[u][e] = A(0);
  for (int s0 = 0; s0 < a.k; s0 += KB) {
    Raw<VB> r[KB][U];
    bool in[KB];
    A w[KB];
#pragma unroll
    for (int s = 0; s < KB; ++s) {
      const bool on = s0 + s < a.k;
      const uint32_t p = on ? static_cast<uint32_t>(__ldg(a.positions + at + s0 + s)) : 0xffffffffu;
      in[s] = p < kept;
      w[s] = in[s] && a.weights ? __ldg(static_cast<const A*>(a.weights) + at + s0 + s) : A(1);
      const char* src = a.x + p * a.x_stride;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (in[s] && v.at(u) < a.nvec) r[s][u] = ld_stream<VB>(src + v.offset(u));
    }
#pragma unroll
    for (int s = 0; s < KB; ++s) {
      if (!in[s]) continue;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        A e[NE];
        expand<T, VB>(r[s][u], e);
#pragma unroll
        for (int j = 0; j < NE; ++j) acc[u][j] += w[s] * e[j];
      }
    }
  }
  char* dst = a.out + t * a.row_bytes;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (v.at(u) < a.nvec) st_row<VB>(dst + v.offset(u), narrow<T, VB>(acc[u]));
}

struct GradArgs {
  const char* grad_out;  // [N], row stride go_stride bytes
  int64_t go_stride;
  const char* y;
  const int32_t* positions;
  const int32_t* kept;
  const void* weights;
  char* grad_y;        // or NULL
  void* grad_weights;  // or NULL
  int64_t row_bytes;
  int64_t N;
  int32_t M;
  int k;
  int nvec;
};

// G lanes per sample walk its row, U vectors at a time: the upstream row is held in registers while KB
// expert rows are read against it (dot products) and KB scaled copies are stored.  One pass for both
// gradients: 16384 rows of 2048 bf16, k = 8, read 604 MB and write 537 in 174 us (6.6 TB/s, the copy rate).
// G by the steps of a row, vectors / U (16 M bf16 elements in 16-byte vectors, k = 4; us with 8 / 32 / 128 lanes):
// 16 steps 28 / 40 / 91, 32 56 / 54 / 103, 96 68 / 52 / 53, 128 63 / 52 / 49.  KB by k (8192 x 2048 bf16; us with
// 2 / 4 / 8): k = 2 28.6 / 29.2 / 38, 4 54 / 48 / 53, 8 105 / 95 / 89; with vectors of 4 and 2 bytes, U = 4, eight
// rows would take 128 registers and more (4096 x 2047 bf16, k = 8: 80 us with 4, 106 with 8).
template <typename T, int VB, int U, int G, int KB>
__global__ void __launch_bounds__(G == 128 ? 128 : 256) combine_backward_kernel(GradArgs a) {
  using A = typename Acc<T>::type;
  constexpr int NE = VB / sizeof(T), kThreads = G == 128 ? 128 : 256;
  __shared__ A part[4][KB];
  const int sub = threadIdx.x % G;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + threadIdx.x / G;
  const bool live = t < a.N;
  const uint32_t kept = kept_rows(a.kept, a.M), M = static_cast<uint32_t>(a.M);
  const char* go = a.grad_out + (live ? t : 0) * a.go_stride;
  for (int s0 = 0; s0 < a.k; s0 += KB) {
    uint32_t p[KB];
    A w[KB], dot[KB];
#pragma unroll
    for (int s = 0; s < KB; ++s) {
      const bool on = live && s0 + s < a.k;
      p[s] = on ? static_cast<uint32_t>(__ldg(a.positions + t * a.k + s0 + s)) : 0xffffffffu;
      w[s] = on ? __ldg(static_cast<const A*>(a.weights) + t * a.k + s0 + s) : A(0);
      dot[s] = A(0);
    }
    for (int v0 = live ? sub : a.nvec; v0 < a.nvec; v0 += G * U) {
      Raw<VB> gr[U], r[KB][U];
#pragma unroll
      for (int u = 0; u < U; ++u) gr[u] = v0 + u * G < a.nvec ? ld_stream<VB>(go + static_cast<int64_t>(v0 + u * G) * VB) : raw_none<VB>();
      if (a.grad_weights) {
#pragma unroll
        for (int s = 0; s < KB; ++s)
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (p[s] < kept && v0 + u * G < a.nvec)
              r[s][u] = ld_stream<VB>(a.y + p[s] * a.row_bytes + static_cast<int64_t>(v0 + u * G) * VB);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (v0 + u * G >= a.nvec) break;
        const int64_t off = static_cast<int64_t>(v0 + u * G) * VB;
        A g[NE];
        expand<T, VB>(gr[u], g);
#pragma unroll
        for (int s = 0; s < KB; ++s) {
          if (a.grad_weights && p[s] < kept) {
            A e[NE];
            expand<T, VB>(r[s][u], e);
#pragma unroll
            for (int j = 0; j < NE; ++j) dot[s] += g[j] * e[j];
          }
          if (a.grad_y && p[s] < M) {
            A d[NE];
#pragma unroll
            for (int j = 0; j < NE; ++j) d[j] = p[s] < kept ? w[s] * g[j] : A(0);
            st_row<VB>(a.grad_y + p[s] * a.row_bytes + off, narrow<T, VB>(d));
          }
        }
      }
    }
    if (a.grad_weights) {
#pragma unroll
      for (int s = 0; s < KB; ++s)
#pragma unroll
        for (int m = 1; m < (G < 32 ? G : 32); m <<= 1) dot[s] += __shfl_xor_sync(kFullMask, dot[s], m);
      if (G == 128) {
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
          for (int s = 0; s < KB; ++s) part[threadIdx.x >> 5][s] = dot[s];
        }
        __syncthreads();
        if (threadIdx.x < KB && s0 + static_cast<int>(threadIdx.x) < a.k)
          static_cast<A*>(a.grad_weights)[t * a.k + s0 + threadIdx.x] =
              (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
        __syncthreads();
      } else if (live && sub == 0) {
#pragma unroll
        for (int s = 0; s < KB; ++s)
          if (s0 + s < a.k) static_cast<A*>(a.grad_weights)[t * a.k + s0 + s] = dot[s];
      }
    }
  }
}

// ---------------------------------------------------------------- launches
// 32-bit thread indices: a launch covers as many samples as fit below 2^32 threads.  body(first sample,
// arguments of the launch, blocks) launches one.
template <typename F>
int per_sample_launches(const char* name, RowArgs a, int64_t N, int vb, int u, cudaStream_t stream, F body) {
  a.nvec = static_cast<uint32_t>(a.row_bytes / vb);
  a.per_row = a.nvec >= 32u * u ? (a.nvec + 32 * u - 1) / (32 * u) * 32 : (a.nvec + u - 1) / u;
  a.div = make_fastdiv(a.per_row);
  const int64_t knob = g_row_threads.load(std::memory_order_relaxed), most = knob > 0 ? knob : 0xffffffffll - 4096;
  const int64_t step = most > a.per_row ? most / a.per_row : 1;  // per_row <= 2^28
  for (int64_t n0 = 0; n0 < N; n0 += step) {
    const int64_t n = N - n0 < step ? N - n0 : step;
    RowArgs b = a;
    b.positions = a.positions + n0 * a.k;
    b.items = static_cast<uint32_t>(n * a.per_row);
    {
      KernelTimer timer(name, stream);
      body(n0, b, static_cast<unsigned>((static_cast<int64_t>(b.items) + 255) / 256));
    }
    TBE_CHECK_LAUNCH(name);
  }
  return TBE_OK;
}

template <int VB>
int launch_dispatch(const RowArgs& a, int64_t N, cudaStream_t stream) {
  // 5003 rows of 1001 fp32 values, k = 6: 35 us with one vector a thread, 29 with two, 30 with four (not TILED)
  constexpr int U = VB == 2 ? 4 : 2;
  return per_sample_launches("dispatch_kernel", a, N, VB, U, stream, [&](int64_t n0, RowArgs b, unsigned blocks) {
    b.x = a.x + n0 * a.x_stride;
    (b.nvec >= 32u * U ? dispatch_kernel<VB, U, true> : dispatch_kernel<VB, U, false>)<<<blocks, 256, 0, stream>>>(b);
  });
}

template <typename T, int VB, int KB>
int launch_combine_k(const RowArgs& a, int64_t N, cudaStream_t stream) {
  using A = typename Acc<T>::type;
  // (the same rows: 43 us with one 4-byte vector a thread, 34 with two or four, 95 with eight)
  constexpr int U = KB == 8 ? 1 : KB == 1 || VB < 8 ? 4 : 2;
  return per_sample_launches("combine_kernel", a, N, VB, U, stream, [&](int64_t n0, RowArgs b, unsigned blocks) {
    b.weights = a.weights ? static_cast<const A*>(a.weights) + n0 * a.k : nullptr;
    b.out = a.out + n0 * a.row_bytes;
    (b.nvec >= 32u * U ? combine_kernel<T, VB, U, KB, true>
                       : combine_kernel<T, VB, U, KB, false>)<<<blocks, 256, 0, stream>>>(b);
  });
}

template <typename T, int VB>
int launch_combine(const RowArgs& a, int64_t N, cudaStream_t stream) {
  if constexpr (VB < static_cast<int>(sizeof(T))) {
    return fail(TBE_ERR_INVALID_ARGUMENT, "tbe_expert_combine: rows must be aligned to their element size");
  } else {
    // a call too small to fill the GPU waits for its loads: all of a sample's at once (8 rows of 2048 bf16,
    // k = 8: 2.3 us against 3.4)
    if (a.k > 4 && N * (a.row_bytes / VB) <= kFewVectors) return launch_combine_k<T, VB, 8>(a, N, stream);
    if (a.k == 1) return launch_combine_k<T, VB, 1>(a, N, stream);
    if (a.k == 2) return launch_combine_k<T, VB, 2>(a, N, stream);
    return launch_combine_k<T, VB, 4>(a, N, stream);
  }
}

template <typename T>
int launch_combine_type(const RowArgs& a, int vb, int64_t N, cudaStream_t stream) {
  switch (vb) {
    case 16: return launch_combine<T, 16>(a, N, stream);
    case 8: return launch_combine<T, 8>(a, N, stream);
    case 4: return launch_combine<T, 4>(a, N, stream);
    default: return launch_combine<T, 2>(a, N, stream);
  }
}

constexpr int backward_vectors(int vb) { return vb == 16 ? 1 : vb == 8 ? 2 : 4; }

template <typename T, int VB, int G, int KB>
int launch_backward_gk(const GradArgs& a, cudaStream_t stream) {
  constexpr int kThreads = G == 128 ? 128 : 256;
  const int64_t blocks = (a.N + kThreads / G - 1) / (kThreads / G);
  {
    KernelTimer timer("combine_backward_kernel", stream);
    combine_backward_kernel<T, VB, backward_vectors(VB), G, KB><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(a);
  }
  TBE_CHECK_LAUNCH("combine_backward_kernel");
  return TBE_OK;
}

template <typename T, int VB, int G>
int launch_backward_g(const GradArgs& a, cudaStream_t stream) {
  if (a.k <= 2) return launch_backward_gk<T, VB, G, 2>(a, stream);
  if (a.k <= 4 || VB < 8) return launch_backward_gk<T, VB, G, 4>(a, stream);
  return launch_backward_gk<T, VB, G, 8>(a, stream);
}

template <typename T, int VB>
int launch_backward(GradArgs a, cudaStream_t stream) {
  if constexpr (VB < static_cast<int>(sizeof(T))) {
    return fail(TBE_ERR_INVALID_ARGUMENT, "tbe_expert_combine_backward: rows must be aligned to their element size");
  } else {
    a.nvec = static_cast<int>(a.row_bytes / VB);
    const int steps = (a.nvec + backward_vectors(VB) - 1) / backward_vectors(VB);
    if (steps <= 16) return launch_backward_g<T, VB, 8>(a, stream);
    if (steps <= 96) return launch_backward_g<T, VB, 32>(a, stream);
    return launch_backward_g<T, VB, 128>(a, stream);
  }
}

template <typename T>
int launch_backward_type(const GradArgs& a, int vb, cudaStream_t stream) {
  switch (vb) {
    case 16: return launch_backward<T, 16>(a, stream);
    case 8: return launch_backward<T, 8>(a, stream);
    case 4: return launch_backward<T, 4>(a, stream);
    default: return launch_backward<T, 2>(a, stream);
  }
}

int check_rows(const char* who, int64_t N, int64_t k, int64_t D, int dtype) {
  TBE_REQUIRE(known_dtype(dtype), "%s: bad dtype %d", who, dtype);
  TBE_REQUIRE(N >= 0 && k > 0 && D > 0 && N <= kMaxEntries && k <= kMaxEntries && N * k <= kMaxEntries,
              "%s: N must be >= 0, k and D > 0, and N*k <= 2^31-1025", who);
  TBE_REQUIRE(D <= (1ll << 28), "%s: rows of more than 2^28 elements are not supported", who);
  return TBE_OK;
}

}  // namespace
}  // namespace tbe

extern "C" int64_t tbe_expert_plan_workspace_bytes(int64_t M, int64_t E) {
  using namespace tbe;
  if (M < 0 || M > kMaxEntries || E < 1 || E > kMaxExperts)
    return fail(TBE_ERR_INVALID_ARGUMENT, "tbe_expert_plan: M must be 0..2^31-1025 and E 1..%d", kMaxExperts);
  const PlanShape s = plan_shape(M);
  return s.mode == kGrid ? static_cast<int64_t>(s.ctas) * (E + 1) * 4 : 0;
}

extern "C" int tbe_expert_plan(const int32_t* experts, int32_t* offsets, int32_t* positions, int32_t* order, int64_t M,
                               int64_t E, void* workspace, int64_t workspace_bytes, void* stream_v) {
  using namespace tbe;
  const int64_t need = tbe_expert_plan_workspace_bytes(M, E);
  if (need < 0) return static_cast<int>(need);
  TBE_REQUIRE(offsets && (M == 0 || (experts && positions && order)), "tbe_expert_plan: null pointer argument");
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(TBE_ERR_WORKSPACE_TOO_SMALL, "tbe_expert_plan: workspace of %lld bytes, %lld needed",
                static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  TBE_REQUIRE(aligned_to(4, experts, offsets, positions, order, workspace),
              "tbe_expert_plan: a pointer is not aligned to its elements");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  const PlanShape s = plan_shape(M);
  int bits = 1;
  while (((E + 1) >> bits) != 0) ++bits;
  PlanArgs a{experts, offsets, positions, order, static_cast<int32_t*>(workspace), static_cast<int32_t>(M),
             static_cast<int32_t>(E), s.slice, bits};
  const int threads = s.mode == kOne ? 256 : 1024;
  const size_t shared = (static_cast<size_t>(threads / 32 + 3) * (E + 1) + 32) * 4;  // at most 144 KB
  auto place = s.mode == kOne ? plan_place_kernel<kOne> : s.mode == kCluster ? plan_place_kernel<kCluster> : plan_place_kernel<kGrid>;
  if (shared > 48 * 1024)
    TBE_CUDA_TRY(cudaFuncSetAttribute(place, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared)));
  if (s.mode == kGrid) {
    {
      KernelTimer timer("plan_count_kernel", stream);
      plan_count_kernel<<<s.ctas, 1024, (E + 1) * 4, stream>>>(a);
    }
    TBE_CHECK_LAUNCH("plan_count_kernel");
  }
  {
    KernelTimer timer("plan_place_kernel", stream);
    if (s.mode == kCluster) {
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = kPlanCluster;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(kPlanCluster);
      cfg.blockDim = dim3(static_cast<unsigned>(threads));
      cfg.dynamicSmemBytes = shared;
      cfg.stream = stream;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      TBE_CUDA_TRY(cudaLaunchKernelEx(&cfg, place, a));
    } else {
      place<<<s.ctas, threads, shared, stream>>>(a);
    }
  }
  TBE_CHECK_LAUNCH("plan_place_kernel");
  return TBE_OK;
}

extern "C" int tbe_expert_dispatch(const void* x, int64_t row_stride, const int32_t* positions, const int32_t* offsets,
                                   void* y, int64_t N, int64_t k, int64_t D, int64_t E, int dtype, void* stream_v) {
  using namespace tbe;
  if (const int rc = check_rows("tbe_expert_dispatch", N, k, D, dtype)) return rc;
  if (N == 0) return TBE_OK;
  TBE_REQUIRE(x && positions && offsets && y, "tbe_expert_dispatch: null pointer argument");
  TBE_REQUIRE(E > 0 && (N == 1 || row_stride >= 0), "tbe_expert_dispatch: E must be > 0, row_stride >= 0");
  const int64_t es = any_elem_size(dtype);
  TBE_REQUIRE(aligned_to(es, x, y) && aligned_to(4, positions, offsets),
              "tbe_expert_dispatch: a pointer is not aligned to its elements");
  RowArgs a{};
  a.x = static_cast<const char*>(x);
  a.x_stride = N == 1 ? 0 : row_stride * es;
  a.positions = positions;
  a.kept = offsets + E;
  a.out = static_cast<char*>(y);
  a.row_bytes = D * es;
  a.M = static_cast<int32_t>(N * k);
  a.k = static_cast<int>(k);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  switch (vector_bytes_of(addr_bits(x) | addr_bits(y) | static_cast<uint64_t>(a.x_stride) | static_cast<uint64_t>(a.row_bytes))) {
    case 16: return launch_dispatch<16>(a, N, stream);
    case 8: return launch_dispatch<8>(a, N, stream);
    case 4: return launch_dispatch<4>(a, N, stream);
    default: return launch_dispatch<2>(a, N, stream);
  }
}

extern "C" int tbe_expert_combine(const void* y, const int32_t* positions, const int32_t* offsets, const void* weights,
                                  void* out, int64_t N, int64_t k, int64_t D, int64_t E, int dtype, void* stream_v) {
  using namespace tbe;
  if (const int rc = check_rows("tbe_expert_combine", N, k, D, dtype)) return rc;
  if (N == 0) return TBE_OK;
  TBE_REQUIRE(y && positions && offsets && out, "tbe_expert_combine: null pointer argument");
  TBE_REQUIRE(E > 0, "tbe_expert_combine: E must be > 0");
  TBE_REQUIRE(aligned_to(any_elem_size(dtype), y, out) && aligned_to(acc_size(dtype), weights) &&
                  aligned_to(4, positions, offsets),
              "tbe_expert_combine: a pointer is not aligned to its elements");
  RowArgs a{};
  a.x = static_cast<const char*>(y);
  a.row_bytes = a.x_stride = D * any_elem_size(dtype);
  a.positions = positions;
  a.kept = offsets + E;
  a.weights = weights;
  a.out = static_cast<char*>(out);
  a.M = static_cast<int32_t>(N * k);
  a.k = static_cast<int>(k);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  const int vb = vector_bytes_of(addr_bits(y) | addr_bits(out) | static_cast<uint64_t>(a.row_bytes));
  switch (dtype) {
    case TBE_F16: return launch_combine_type<__half>(a, vb, N, stream);
    case TBE_BF16: return launch_combine_type<__nv_bfloat16>(a, vb, N, stream);
    case TBE_F32: return launch_combine_type<float>(a, vb, N, stream);
    default: return launch_combine_type<double>(a, vb, N, stream);
  }
}

extern "C" int tbe_expert_combine_backward(const void* grad_out, int64_t grad_stride, const void* y,
                                           const int32_t* positions, const int32_t* offsets, const void* weights,
                                           void* grad_y, void* grad_weights, int64_t N, int64_t k, int64_t D, int64_t E,
                                           int dtype, void* stream_v) {
  using namespace tbe;
  if (const int rc = check_rows("tbe_expert_combine_backward", N, k, D, dtype)) return rc;
  if (N == 0 || (!grad_y && !grad_weights)) return TBE_OK;
  TBE_REQUIRE(grad_out && positions && offsets && weights && (y || !grad_weights),
              "tbe_expert_combine_backward: null pointer argument");
  TBE_REQUIRE(E > 0 && (N == 1 || grad_stride >= 0), "tbe_expert_combine_backward: E must be > 0, grad_stride >= 0");
  const int64_t es = any_elem_size(dtype);
  TBE_REQUIRE(aligned_to(es, grad_out, y, grad_y) && aligned_to(acc_size(dtype), weights, grad_weights) &&
                  aligned_to(4, positions, offsets),
              "tbe_expert_combine_backward: a pointer is not aligned to its elements");
  GradArgs a{};
  a.grad_out = static_cast<const char*>(grad_out);
  a.go_stride = N == 1 ? 0 : grad_stride * es;
  a.y = static_cast<const char*>(y);
  a.positions = positions;
  a.kept = offsets + E;
  a.weights = weights;
  a.grad_y = static_cast<char*>(grad_y);
  a.grad_weights = grad_weights;
  a.row_bytes = D * es;
  a.N = N;
  a.M = static_cast<int32_t>(N * k);
  a.k = static_cast<int>(k);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  const int vb = vector_bytes_of(addr_bits(grad_out) | addr_bits(y) | addr_bits(grad_y) |
                                 static_cast<uint64_t>(a.go_stride) | static_cast<uint64_t>(a.row_bytes));
  switch (dtype) {
    case TBE_F16: return launch_backward_type<__half>(a, vb, stream);
    case TBE_BF16: return launch_backward_type<__nv_bfloat16>(a, vb, stream);
    case TBE_F32: return launch_backward_type<float>(a, vb, stream);
    default: return launch_backward_type<double>(a, vb, stream);
  }
}
