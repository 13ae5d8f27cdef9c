// Layer norm over the last dim, and its first and second derivatives: fhob_layer_norm, fhob_layer_norm_backward,
// fhob_layer_norm_bwdbwd.
//
//   mu = mean x, r = 1 / sqrt(mean (x - mu)^2 + eps), h = (x - mu) r                 y = h w + b
//   g = dy w:      dx = r (g - mean g - h mean(g h))          dw = sum dy h          db = sum dy
//   cotangents v of dx, vw of dw, vb of db; a = mean v, c = mean(v h), m = mean g, q = mean(g h):
//     p = v - a - h c:   ddy = r w p + vw h + vb              dw2 = sum dy r p
//     e = vw dy - r (g c + v q):
//       dx2 = r (e - mean e - h mean(e h)) - r^2 h mean(p (g - m))
//   (sums over rows for dw, db, dw2; means over a row).  The last mean stands for mean(v g) - a m - c q, which it equals for every eps:
//   mean(p (g - m)) = mean(v g) - m a - a mean(g - m) - c mean(h g) + c m mean h, where mean(g - m) = mean h = 0.  Both of its factors are
//   centred, so nothing cancels when v or g have a large common part.  (Not p (g - m - h q): that adds c q (mean(h^2) - 1), and
//   mean(h^2) = var / (var + eps) is one only for eps = 0.)
//
// What bounds it: each matrix is read once and written once, so the memory.
//  - A row belongs to a group: 2 to 32 lanes of a warp or up to 32 warps, 8 to 32 elements a lane.  It is in registers, in fp32,
//    from its only load to its results; sums over it are shuffles, then, if the group has several warps, one exchange
//    through shared memory per round.  Rounds: two in the forward (the variance is a sum of squares around the mean), one
//    in the backward, two in the double backward.
//  - What is left next to the memory is latency: a row's conversion, sums, exchange and stores follow one another, and the 16 to 24 warps
//    an SM that the registers allow (24 to 25 % of the most) issue in 50 to 57 % of the cycles.  So that these are short, elements are
//    converted once, the arithmetic is on packed pairs, and the vectors over the columns stay in registers or (double backward) in a thread's
//    own shared memory.  (Converted where they are used, with scalar arithmetic, and without the copies below: 16384 x 2048 bf16 forward
//    42 us, backward 75, double backward 175; now 26 (5.1 TB/s), 43 (4.7, of which the second launch takes 6) and 72 (4.6).  fp32 50 (5.4), 69 (5.9)
//    and 112 (6.0).)
//  - What keeps the memory busy is the number of bytes on their way.  Rows come through a ring in shared memory, up to
//    three rows ahead of the one in work, by asynchronous copies.  On the 16-byte grid a thread copies its own elements
//    alone: it is the only one to read them, so nothing waits but for its own copies.
//  - A thread owns the same columns of all its rows, so what the sums over rows add up stays in its registers; the groups of a
//    block are added up in shared memory and the blocks' sums in a second launch, always in the same order.
//  - Rows off the 16-byte grid (an odd number of columns) are copied by their group together, in the 16-byte pieces of memory
//    that hold them, and read element by element: neighbouring threads own neighbouring columns then.
#include "fhob_common.cuh"
#include "tc_common.cuh"

namespace fhob {
namespace {

constexpr int LN_MAX_WARPS = 32;

struct LnParams {
  const void *x, *dy, *v;                  // rows at their strides
  long long x_row, dy_row, v_row;
  const void *w, *b, *vw, *vb;             // any may be NULL
  const float *mean_in, *rstd_in;
  void *y, *dx;                            // y | dx, and of the double backward ddy | dx2; contiguous
  float *mean, *rstd;
  float* partial;                          // [block][0 = dw, 1 = db][cols], NULL when no such sum is wanted
  int rows, cols, warps, lanes;            // of a group: warps, and lanes of a warp (32 if there are several warps)
  int w_f32;                               // type of w, b, vw, vb: fp32, or that of the matrices
  int want_dw, want_db;
  float eps, inv_cols;
};

// How a thread's elements lie in a row: in pieces of 16 bytes (V elements each), or, V == 2, in pairs of neighbours (16 bits), or
// one here and one there (fp32).
template <class T, int V>
constexpr bool kWide = V * sizeof(T) == 16;
template <class T, int V>
constexpr bool kTogether = V * sizeof(T) == 16 || sizeof(T) == 2;

// `bytes` of 16 are read, the others zero
__device__ __forceinline__ void cp_async(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
template <class T>
__device__ __forceinline__ float2 unpack(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <class T>
__device__ __forceinline__ uint32_t pack(const float2& x) { return pack16<std::is_same<T, __half>::value>(x.x, x.y); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// What a thread needs to know of its place.  Element e of its piece i is at column(i, e).  SUB: several rows share a warp.
template <class T, int V, bool SUB>
struct Place {
  static constexpr bool kSub = SUB;
  int group, groups;         // of the block
  int warp, warps;           // of the group
  int lanes;                 // of a warp
  int first, width;          // this thread of the group's threads
  int above;                 // groups of this warp in front of this thread's
  __device__ __forceinline__ Place(int warps_per_group, int lanes_per_group) {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    warps = SUB ? 1 : warps_per_group;
    lanes = SUB ? lanes_per_group : 32;
    const int per_warp = SUB ? 32 / lanes : 1;
    above = SUB ? lane / lanes : 0;
    group = w / warps * per_warp + above;
    groups = (blockDim.x >> 5) / warps * per_warp;
    warp = w % warps;
    first = warp * 32 + (SUB ? lane % lanes : lane);
    width = warps * lanes;
  }
  __device__ __forceinline__ int column(int i, int e = 0) const {
    return kTogether<T, V> ? (first + i * width) * V + e : first + (i * V + e) * width;
  }
  // x at the columns of a pair of piece i, zero behind the last column.  (Pieces of 16 bytes are whole.)
  __device__ __forceinline__ float2 inside(float x, int i, int cols) const {
    const float here = column(i) < cols ? x : 0.f;
    return make_float2(here, kWide<T, V> ? here : (column(i, 1) < cols ? x : 0.f));
  }
  __device__ __forceinline__ void meet() const {   // the group
    if (SUB || warps == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(width) : "memory");
  }
  // Stores piece i of a row.
  __device__ __forceinline__ void store(T* row, int i, int cols, const float2 (&x)[V / 2]) const {
    const int c = column(i);
    if (c >= cols) return;
    if constexpr (!kWide<T, V>) {
      if constexpr (sizeof(T) == 2)
        if (c + 1 < cols && (reinterpret_cast<uintptr_t>(row) & 2) == 0) {
          *reinterpret_cast<uint32_t*>(row + c) = pack<T>(x[0]);
          return;
        }
      row[c] = static_cast<T>(x[0].x);
      if (column(i, 1) < cols) row[column(i, 1)] = static_cast<T>(x[0].y);
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(row + c) = make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
    } else {
      *reinterpret_cast<uint4*>(row + c) = make_uint4(pack<T>(x[0]), pack<T>(x[1]), pack<T>(x[2]), pack<T>(x[3]));
    }
  }
  // Piece i of a vector over the columns; `otherwise` where there is no vector or no such column.
  __device__ __forceinline__ void vector(float2 (&to)[V / 2], const void* from, int f32, int i, int cols, float otherwise) const {
    auto element = [&](int e) {
      const int c = column(i, e);
      if (!from || c >= cols) return otherwise;
      return f32 ? static_cast<const float*>(from)[c] : static_cast<float>(static_cast<const T*>(from)[c]);
    };
    if (kWide<T, V> && from && !f32 && sizeof(T) == 2 && column(i) < cols) {
      const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const T*>(from) + column(i));
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < V / 2; ++j) to[j] = unpack<T>(ws[j & 3]);
      return;
    }
#pragma unroll
    for (int j = 0; j < V / 2; ++j) to[j] = make_float2(element(2 * j), element(2 * j + 1));
  }
};

// Sums of four (or, the last ones unused, fewer) values over a group, in every thread of it.  `exchange`: four floats per warp
// of the block; two such areas take turns, so that one meeting a round is enough (a warp that is a round ahead writes to the
// other area, and cannot be two ahead).
//  In a whole warp, a lane passes on half of its values in each of the first steps and adds up the other half: two values
//  take 5 shuffles, four 6, where each by itself takes 5.  Lane 8 k then has value k (one value: every lane; two: lane 16 k).
template <int N, class P>
__device__ __forceinline__ void group_sum(float (&x)[N], const P& at, float* exchange) {
  constexpr unsigned kAll = 0xffffffffu;
  if constexpr (P::kSub) {
    for (int o = at.lanes >> 1; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] += __shfl_xor_sync(kAll, x[i], o);
    return;
  }
  const int lane = threadIdx.x & 31;
  float y = x[0];
  if constexpr (N > 2) {
    const bool upper = lane & 16;
    const float x3 = N > 3 ? x[N - 1] : 0.f;
    float a0 = (upper ? x[2] : x[0]) + __shfl_xor_sync(kAll, upper ? x[0] : x[2], 16);
    float a1 = (upper ? x3 : x[1]) + __shfl_xor_sync(kAll, upper ? x[1] : x3, 16);
    const bool odd = lane & 8;
    y = (odd ? a1 : a0) + __shfl_xor_sync(kAll, odd ? a0 : a1, 8);
  } else if constexpr (N == 2) {
    const bool upper = lane & 16;
    y = (upper ? x[1] : x[0]) + __shfl_xor_sync(kAll, upper ? x[0] : x[1], 16);
    y += __shfl_xor_sync(kAll, y, 8);
  } else {
    y += __shfl_xor_sync(kAll, y, 16);
    y += __shfl_xor_sync(kAll, y, 8);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) y += __shfl_xor_sync(kAll, y, o);
  constexpr int kStep = N > 2 ? 8 : 16;   // lanes between the values
  if (at.warps == 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __shfl_sync(kAll, y, i * kStep);
    return;
  }
  float* mine = exchange + at.group * at.warps * 4;
  if ((lane & (kStep - 1)) == 0) mine[at.warp * 4 + lane / kStep] = y;
  at.meet();
  // Every warp adds up the same numbers in the same order.  Few are read by every lane; of more, lane 4 w + i takes value i of
  // warp w (of every eighth warp), then the lanes of a value add up.
  if (at.warps <= 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.f;
    for (int w = 0; w < at.warps; ++w) {
      const float4 v = reinterpret_cast<const float4*>(mine)[w];
      x[0] += v.x;
      if constexpr (N > 1) x[1] += v.y;
      if constexpr (N > 2) x[2] += v.z;
      if constexpr (N > 3) x[3] += v.w;
    }
    return;
  }
  y = 0.f;
  if ((lane & 3) < N)
    for (int j = lane; j < at.warps * 4; j += 32) y += mine[j];
#pragma unroll
  for (int o = 16; o > 2; o >>= 1) y += __shfl_xor_sync(kAll, y, o);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = __shfl_sync(kAll, y, i);
}

// How the three kernels are laid out: blocks with room for 256 to 1024 threads, 512 threads an SM with 128 registers each (168 in
// blocks of 384, 80 in those of 768 and 64 in those of 1024, which only long rows take), 768 where less is kept of each.
enum { kLnForward, kLnBackward, kLnBwdbwd };
constexpr int ln_threads(int what, int each) { return what == kLnForward && each <= 16 ? 768 : 512; }   // of an SM
template <int WHAT, class T, int V, int NV, int THREADS, bool SUB>
struct LnCfg {
  static constexpr int kMatrices = WHAT == kLnForward ? 1 : (WHAT == kLnBackward ? 2 : 3);
  static constexpr int kBlocks = ln_threads(WHAT, NV * V) > THREADS ? ln_threads(WHAT, NV * V) / THREADS : 1;   // of an SM
  // Bytes of a row of the ring.  Off the grid a row may start anywhere in a piece of 16 bytes: one more for each group (and a word
  // that the last pair of the last group looks into).
  static constexpr int kRow = THREADS * NV * V * static_cast<int>(sizeof(T)) + (kWide<T, V> ? 0 : 16 * THREADS / (SUB ? 2 : 32));
  // Where the vectors over the columns are kept through the rows: in registers, or (kShare) in shared memory, a thread's own, or neither:
  // read again for every row.
  static constexpr bool kHold = WHAT != kLnBwdbwd || NV * V <= 8 || THREADS == 384;
  static constexpr bool kShare = !kHold && THREADS == 512;
  // Of the backward: the weight, for long rows (12288 columns, 4096 rows bf16 149 -> 117 us; off the grid 9001 84 -> 92).
  static constexpr bool kShareW = WHAT == kLnBackward && kWide<T, V> && THREADS >= 768;
  static constexpr int kVectors = (kShare ? 3 : kShareW ? 1 : 0) * THREADS * NV * V * 4;   // bytes behind the ring
  static constexpr int kFit = (200 * 1024 - kVectors) / kBlocks / (kMatrices * kRow);
  static constexpr int kStages = kFit > 4 ? 4 : kFit;                         // rows of the ring
  static constexpr int kExchange = 2 * LN_MAX_WARPS * 16;                     // bytes in front of it: two areas for the sums over a row
  static constexpr int kRing = kMatrices * kRow * kStages;
  static constexpr int kSmem = kExchange + kRing + kVectors;
  static_assert(kStages >= 1, "a row of the ring");
  static_assert(WHAT == kLnForward || THREADS * NV * V * 4 <= kRing, "room for the sums over rows, see block_columns");
};

// The ring.  On the grid it is a thread's own: piece i of (stage, matrix) is THREADS * 16 bytes on from piece i - 1.  Off the
// grid a row lies as in memory, from the piece of 16 bytes on that holds its first element.
template <class C, class T, int V, int NV, int THREADS, bool SUB>
struct Ring {
  uint32_t base;
  const Place<T, V, SUB>& at;
  int cols;
  __device__ __forceinline__ Ring(const void* smem, const Place<T, V, SUB>& place, int n) : at(place), cols(n) {
    base = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
    if (kWide<T, V>) base += threadIdx.x * 16;
    else base += at.group * (at.width * NV * V * static_cast<int>(sizeof(T)) + 16);
  }
  __device__ __forceinline__ uint32_t slot(int stage, int matrix) const { return base + (stage * C::kMatrices + matrix) * C::kRow; }
  __device__ __forceinline__ void copy(int stage, int matrix, const T* row, bool live) const {
    const uint32_t to = slot(stage, matrix);
    if constexpr (kWide<T, V>) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const bool there = live && at.column(i) < cols;
        cp_async(to + i * (THREADS * 16), there ? row + at.column(i) : row, there ? 16 : 0);
      }
    } else {
      // (what lies in front of the row in its first 16 bytes of memory belongs to the same allocation: that starts on 16 bytes)
      const uintptr_t start = reinterpret_cast<uintptr_t>(row) & ~static_cast<uintptr_t>(15);
      const int bytes = live ? static_cast<int>(reinterpret_cast<uintptr_t>(row) - start) + cols * static_cast<int>(sizeof(T)) : 0;
      constexpr int kPieces = NV * V * static_cast<int>(sizeof(T)) / 16;
#pragma unroll
      for (int i = 0; i <= kPieces; ++i) {
        // (behind the row zeros: nothing that is read later is older)
        const int from = (at.first + i * at.width) * 16, left = min(16, bytes - from);
        if (i < kPieces || at.first == 0) cp_async(to + from, reinterpret_cast<const void*>(left > 0 ? start + from : start), left > 0 ? left : 0);
      }
    }
  }
  // `row_address`: the low bits of the row's address.  Zeros behind the last column and for rows that do not exist.
  __device__ __forceinline__ void read(float2 (&to)[NV][V / 2], int stage, int matrix, uint32_t row_address) const {
    const uint32_t from = slot(stage, matrix);
    if constexpr (kWide<T, V>) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        uint32_t w[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(from + i * (THREADS * 16)));
        if constexpr (sizeof(T) == 4) {
          to[i][0] = f2(w[0], w[1]);
          to[i][1] = f2(w[2], w[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) to[i][j] = unpack<T>(w[j]);
        }
      }
    } else {
      const uint32_t first = from + (row_address & 15u);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const uint32_t here = first + at.column(i) * static_cast<uint32_t>(sizeof(T));
        uint32_t w, next = 0u;
        if constexpr (sizeof(T) == 4) {
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(here));
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(next) : "r"(here + at.width * 4));
          to[i][0] = f2(w, next);
        } else if (here & 2u) {   // the pair lies in two words
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(here - 2));
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(next) : "r"(here + 2));
          to[i][0] = unpack<T>(__funnelshift_r(w, next, 16));
        } else {
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(here));
          to[i][0] = unpack<T>(w);
        }
      }
    }
  }
};
// The rows of a matrix that a group goes through: one to copy next, one to work on next.
template <class T>
struct Walk {
  const T* start;
  const T* ahead;
  long long by;        // elements from a row to the group's next
  uint32_t address;    // of the row to work on, low bits
  __device__ __forceinline__ Walk(const void* matrix, long long stride, int row, int step) {
    start = static_cast<const T*>(matrix);
    ahead = start + row * stride;
    by = step * stride;
    address = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ahead));
  }
  __device__ __forceinline__ const T* next(bool live) {   // rows that do not exist are not read
    const T* at = live ? ahead : start;
    ahead += by;
    return at;
  }
  __device__ __forceinline__ uint32_t worked() {
    const uint32_t at = address;
    address += static_cast<uint32_t>(by) * static_cast<uint32_t>(sizeof(T));
    return at;
  }
};
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// Adds up the groups' sums over rows and leaves the block's in `partial` (cols floats).  `scratch`: a row of cols floats per
// warp or group of warps, in the ring, which is no longer in use.
template <class T, int V, int NV, bool SUB>
__device__ __forceinline__ void block_columns(float2 (&sum)[NV][V / 2], const Place<T, V, SUB>& at, int cols, float* scratch, float* partial) {
  // the groups of a warp hold the same columns in lanes `lanes` apart
  for (int o = at.lanes; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        sum[i][j].x += __shfl_xor_sync(0xffffffffu, sum[i][j].x, o);
        sum[i][j].y += __shfl_xor_sync(0xffffffffu, sum[i][j].y, o);
      }
  const int rows = (blockDim.x >> 5) / at.warps, mine = (threadIdx.x >> 5) / at.warps;
  __syncthreads();
  if (at.above == 0)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        const int c0 = at.column(i, 2 * j), c1 = at.column(i, 2 * j + 1);
        if (c0 < cols) scratch[mine * cols + c0] = sum[i][j].x;
        if (c1 < cols) scratch[mine * cols + c1] = sum[i][j].y;
      }
  __syncthreads();
  for (int c = threadIdx.x; c < cols; c += blockDim.x) {
    float total = scratch[c];
    for (int r = 1; r < rows; ++r) total += scratch[r * cols + c];
    partial[c] = total;
  }
}

template <class T, int V, int NV, int THREADS, bool SUB>
__global__ void __launch_bounds__(THREADS, LnCfg<kLnForward, T, V, NV, THREADS, SUB>::kBlocks) ln_forward_kernel(const __grid_constant__ LnParams p) {
  using C = LnCfg<kLnForward, T, V, NV, THREADS, SUB>;
  constexpr int H = V / 2;   // pairs of a piece
  extern __shared__ __align__(16) float exchange[];
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const Place<T, V, SUB> at(p.warps, p.lanes);
  const Ring<C, T, V, NV, THREADS, SUB> ring(reinterpret_cast<char*>(exchange) + C::kExchange, at, p.cols);
  const int step = gridDim.x * at.groups;
  int row = blockIdx.x * at.groups + at.group;
  Walk<T> xs(p.x, p.x_row, row, step);
  auto fetch = [&](int stage, int r) {
    ring.copy(stage, 0, xs.next(r < p.rows), r < p.rows);
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) fetch(i, row + i * step);
  float2 w[NV][H], b[NV][H];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    at.vector(w[i], p.w, p.w_f32, i, p.cols, 1.f);
    at.vector(b[i], p.b, p.w_f32, i, p.cols, 0.f);
  }
  for (int stage = 0; row - at.above < p.rows; row += step, stage = stage + 1 == C::kStages ? 0 : stage + 1) {
    fetch(stage == 0 ? C::kStages - 1 : stage - 1, row + (C::kStages - 1) * step);   // where the row before this one was
    copies_wait<C::kStages - 1>();
    if (!kWide<T, V>) at.meet();   // the group's copies
    float2 x[NV][H], s2 = both(0.f);
    ring.read(x, stage, 0, xs.worked());
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < H; ++j) s2 = __fadd2_rn(s2, x[i][j]);
    float s[1] = {s2.x + s2.y};
    group_sum<1>(s, at, exchange);
    const float mean = s[0] * p.inv_cols;
    s2 = both(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float2 minus = at.inside(-mean, i, p.cols);   // zeros stay zeros behind the last column
#pragma unroll
      for (int j = 0; j < H; ++j) {
        x[i][j] = __fadd2_rn(x[i][j], minus);
        s2 = __ffma2_rn(x[i][j], x[i][j], s2);
      }
    }
    s[0] = s2.x + s2.y;
    group_sum<1>(s, at, exchange + 4 * LN_MAX_WARPS);
    const float r = rsqrtf(fmaf(s[0], p.inv_cols, p.eps));
    if (row < p.rows) {
      T* y = static_cast<T*>(p.y) + static_cast<long long>(row) * p.cols;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < H; ++j) x[i][j] = __ffma2_rn(__fmul2_rn(x[i][j], both(r)), w[i][j], b[i][j]);
        at.store(y, i, p.cols, x[i]);
      }
      if (at.first == 0) {
        p.mean[row] = mean;
        p.rstd[row] = r;
      }
    }
  }
  copies_wait<0>();
}

template <class T, int V, int NV, int THREADS, bool SUB>
__global__ void __launch_bounds__(THREADS, LnCfg<kLnBackward, T, V, NV, THREADS, SUB>::kBlocks) ln_backward_kernel(const __grid_constant__ LnParams p) {
  using C = LnCfg<kLnBackward, T, V, NV, THREADS, SUB>;
  constexpr int H = V / 2;
  extern __shared__ __align__(16) float exchange[];
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const Place<T, V, SUB> at(p.warps, p.lanes);
  char* in_ring = reinterpret_cast<char*>(exchange) + C::kExchange;
  const Ring<C, T, V, NV, THREADS, SUB> ring(in_ring, at, p.cols);
  const int step = gridDim.x * at.groups;
  int row = blockIdx.x * at.groups + at.group;
  Walk<T> xs(p.x, p.x_row, row, step), dys(p.dy, p.dy_row, row, step);
  auto fetch = [&](int stage, int r) {
    ring.copy(stage, 0, xs.next(r < p.rows), r < p.rows);
    ring.copy(stage, 1, dys.next(r < p.rows), r < p.rows);
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) fetch(i, row + i * step);
  float2 w[NV][H], dw[NV][H], db[NV][H];
  float2* const shared = reinterpret_cast<float2*>(in_ring + C::kRing) + threadIdx.x;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    at.vector(w[i], p.w, p.w_f32, i, p.cols, 1.f);
    if (C::kShareW)
#pragma unroll
      for (int j = 0; j < H; ++j) shared[(i * H + j) * THREADS] = w[i][j];
#pragma unroll
    for (int j = 0; j < H; ++j) dw[i][j] = db[i][j] = both(0.f);
  }
  float next_mean = 0.f, next_r = 0.f;
  auto fetch_statistics = [&](int r) {
    next_mean = r < p.rows ? p.mean_in[r] : 0.f;
    next_r = r < p.rows ? p.rstd_in[r] : 0.f;
  };
  fetch_statistics(row);
  int turn = 0;
  for (int stage = 0; row - at.above < p.rows; row += step, turn ^= 1, stage = stage + 1 == C::kStages ? 0 : stage + 1) {
    fetch(stage == 0 ? C::kStages - 1 : stage - 1, row + (C::kStages - 1) * step);   // where the row before this one was
    const float mean = next_mean, r = next_r;
    fetch_statistics(row + step);
    copies_wait<C::kStages - 1>();
    if (!kWide<T, V>) at.meet();   // the group's copies
    float2 h[NV][H], g[NV][H], s0 = both(0.f), s1 = both(0.f);   // sums of g, g h
    ring.read(h, stage, 0, xs.worked());
    ring.read(g, stage, 1, dys.worked());
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float2 minus = at.inside(-mean, i, p.cols);   // behind the last column and row h and dy are zero
#pragma unroll
      for (int j = 0; j < H; ++j) {
        h[i][j] = __fmul2_rn(__fadd2_rn(h[i][j], minus), both(r));
        dw[i][j] = __ffma2_rn(g[i][j], h[i][j], dw[i][j]);
        db[i][j] = __fadd2_rn(db[i][j], g[i][j]);
        g[i][j] = __fmul2_rn(g[i][j], C::kShareW ? shared[(i * H + j) * THREADS] : w[i][j]);
        s0 = __fadd2_rn(s0, g[i][j]);
        s1 = __ffma2_rn(g[i][j], h[i][j], s1);
      }
    }
    float s[2] = {s0.x + s0.y, s1.x + s1.y};
    group_sum<2>(s, at, exchange + turn * 4 * LN_MAX_WARPS);
    if (row < p.rows) {
      const float2 m = both(-s[0] * p.inv_cols), q = both(-s[1] * p.inv_cols);
      T* dx = static_cast<T*>(p.dx) + static_cast<long long>(row) * p.cols;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < H; ++j) g[i][j] = __fmul2_rn(__ffma2_rn(h[i][j], q, __fadd2_rn(g[i][j], m)), both(r));
        at.store(dx, i, p.cols, g[i]);
      }
    }
  }
  copies_wait<0>();
  if (p.partial) {
    float* to = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols;
    if (p.want_dw) block_columns<T, V, NV, SUB>(dw, at, p.cols, reinterpret_cast<float*>(in_ring), to);
    if (p.want_db) block_columns<T, V, NV, SUB>(db, at, p.cols, reinterpret_cast<float*>(in_ring), to + p.cols);
  }
}

template <class T, int V, int NV, int THREADS, bool SUB>
__global__ void __launch_bounds__(THREADS, LnCfg<kLnBwdbwd, T, V, NV, THREADS, SUB>::kBlocks) ln_bwdbwd_kernel(const __grid_constant__ LnParams p) {
  using C = LnCfg<kLnBwdbwd, T, V, NV, THREADS, SUB>;
  constexpr int H = V / 2;
  extern __shared__ __align__(16) float exchange[];
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const Place<T, V, SUB> at(p.warps, p.lanes);
  char* in_ring = reinterpret_cast<char*>(exchange) + C::kExchange;
  const Ring<C, T, V, NV, THREADS, SUB> ring(in_ring, at, p.cols);
  const int step = gridDim.x * at.groups;
  int row = blockIdx.x * at.groups + at.group;
  Walk<T> xs(p.x, p.x_row, row, step), dys(p.dy, p.dy_row, row, step), vs(p.v ? p.v : p.x, p.v ? p.v_row : p.x_row, row, step);
  auto fetch = [&](int stage, int r) {
    ring.copy(stage, 0, xs.next(r < p.rows), r < p.rows);
    ring.copy(stage, 1, dys.next(r < p.rows), r < p.rows);
    ring.copy(stage, 2, vs.next(r < p.rows), p.v && r < p.rows);   // zeros if there is none
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) fetch(i, row + i * step);
  float2 w[NV][H], vw[NV][H], vb[NV][H], dw2[NV][H];
  // what of them is not kept in registers is read where it is needed
  float2* const shared = reinterpret_cast<float2*>(in_ring + C::kRing) + threadIdx.x;
  auto again = [&](float2 (&to)[H], int which, const void* from, int i, float otherwise) {
    if constexpr (C::kShare) {
#pragma unroll
      for (int j = 0; j < H; ++j) to[j] = shared[((which * NV + i) * H + j) * THREADS];
    } else if constexpr (!C::kHold) {
      at.vector(to, from, p.w_f32, i, p.cols, otherwise);
    }
  };
  auto w_again = [&](int i) { again(w[i], 0, p.w, i, 1.f); };
  auto vw_again = [&](int i) { again(vw[i], 1, p.vw, i, 0.f); };
  auto vb_again = [&](int i) { again(vb[i], 2, p.vb, i, 0.f); };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (C::kHold || C::kShare) {
      at.vector(w[i], p.w, p.w_f32, i, p.cols, 1.f);
      at.vector(vw[i], p.vw, p.w_f32, i, p.cols, 0.f);
      at.vector(vb[i], p.vb, p.w_f32, i, p.cols, 0.f);
    }
    if (C::kShare)
#pragma unroll
      for (int j = 0; j < H; ++j) {
        shared[((0 * NV + i) * H + j) * THREADS] = w[i][j];
        shared[((1 * NV + i) * H + j) * THREADS] = vw[i][j];
        shared[((2 * NV + i) * H + j) * THREADS] = vb[i][j];
      }
#pragma unroll
    for (int j = 0; j < H; ++j) dw2[i][j] = both(0.f);
  }
  float next_mean = 0.f, next_r = 0.f;
  auto fetch_statistics = [&](int r) {
    next_mean = r < p.rows ? p.mean_in[r] : 0.f;
    next_r = r < p.rows ? p.rstd_in[r] : 0.f;
  };
  fetch_statistics(row);
  for (int stage = 0; row - at.above < p.rows; row += step, stage = stage + 1 == C::kStages ? 0 : stage + 1) {
    fetch(stage == 0 ? C::kStages - 1 : stage - 1, row + (C::kStages - 1) * step);   // where the row before this one was
    const float mean = next_mean, r = next_r;
    fetch_statistics(row + step);
    copies_wait<C::kStages - 1>();
    if (!kWide<T, V>) at.meet();   // the group's copies
    // h, dy and v; all zero behind the last column and the last row
    float2 h[NV][H], d[NV][H], u[NV][H], s0 = both(0.f), s1 = both(0.f), s2 = both(0.f), s3 = both(0.f);
    ring.read(h, stage, 0, xs.worked());
    ring.read(d, stage, 1, dys.worked());
    ring.read(u, stage, 2, vs.worked());
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float2 minus = at.inside(-mean, i, p.cols);
      w_again(i);
#pragma unroll
      for (int j = 0; j < H; ++j) {
        h[i][j] = __fmul2_rn(__fadd2_rn(h[i][j], minus), both(r));
        const float2 g = __fmul2_rn(d[i][j], w[i][j]);
        s0 = __fadd2_rn(s0, u[i][j]);
        s1 = __ffma2_rn(u[i][j], h[i][j], s1);
        s2 = __fadd2_rn(s2, g);
        s3 = __ffma2_rn(g, h[i][j], s3);
      }
    }
    float s[4] = {s0.x + s0.y, s1.x + s1.y, s2.x + s2.y, s3.x + s3.y};
    group_sum<4>(s, at, exchange);
    const float a = s[0] * p.inv_cols, c = s[1] * p.inv_cols, m = s[2] * p.inv_cols, q = s[3] * p.inv_cols;
    s0 = s1 = s2 = both(0.f);   // sums of p (g - m), e, e h
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float2 minus = at.inside(-a, i, p.cols);
      w_again(i);
      vw_again(i);
#pragma unroll
      for (int j = 0; j < H; ++j) {
        const float2 g = __fmul2_rn(d[i][j], w[i][j]);
        const float2 e = __ffma2_rn(vw[i][j], d[i][j], __ffma2_rn(g, both(-r * c), __fmul2_rn(u[i][j], both(-r * q))));
        const float2 pp = __ffma2_rn(h[i][j], both(-c), __fadd2_rn(u[i][j], minus));
        dw2[i][j] = __ffma2_rn(__fmul2_rn(d[i][j], both(r)), pp, dw2[i][j]);
        s0 = __ffma2_rn(pp, __fadd2_rn(g, both(-m)), s0);
        s1 = __fadd2_rn(s1, e);
        s2 = __ffma2_rn(e, h[i][j], s2);
        u[i][j] = pp;
        d[i][j] = e;
      }
    }
    float t[3] = {s0.x + s0.y, s1.x + s1.y, s2.x + s2.y};
    group_sum<3>(t, at, exchange + 4 * LN_MAX_WARPS);
    if (row < p.rows) {
      const float k = t[0] * p.inv_cols * r, me = t[1] * p.inv_cols, meh = t[2] * p.inv_cols;
      T *ddy = static_cast<T*>(p.y) + static_cast<long long>(row) * p.cols, *dx2 = static_cast<T*>(p.dx) + static_cast<long long>(row) * p.cols;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        w_again(i);
        vw_again(i);
        vb_again(i);
#pragma unroll
        for (int j = 0; j < H; ++j) {
          u[i][j] = __ffma2_rn(__fmul2_rn(w[i][j], both(r)), u[i][j], __ffma2_rn(vw[i][j], h[i][j], vb[i][j]));
          d[i][j] = __fmul2_rn(__ffma2_rn(h[i][j], both(-(meh + k)), __fadd2_rn(d[i][j], both(-me))), both(r));
        }
        at.store(ddy, i, p.cols, u[i]);
        at.store(dx2, i, p.cols, d[i]);
      }
    }
  }
  copies_wait<0>();
  if (p.partial) block_columns<T, V, NV, SUB>(dw2, at, p.cols, reinterpret_cast<float*>(in_ring), p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols);
}

// Sums over the blocks: a block takes 32 columns, its 32 warps a share of the rows of `partial` each, in order.
template <class W>
__global__ void __launch_bounds__(1024) ln_columns_kernel(const float* partial, int blocks, int cols, W* dw, W* db) {
  __shared__ float part[32][33];
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool second = blockIdx.y == 1 || !dw;
  const int c = blockIdx.x * 32 + lane;
  const float* from = partial + (second ? cols : 0) + c;
  float sum = 0.f;
  if (c < cols)
#pragma unroll 10
    for (int i = warp; i < blocks; i += 32) sum += from[static_cast<long long>(i) * 2 * cols];
  part[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 32; ++i) sum += part[i][lane];
    (second ? db : dw)[c] = static_cast<W>(sum);
  }
}

// How a call is cut up.
struct LnGrid {
  bool wide;
  int each, lanes, warps;      // elements of a thread; of a group: lanes and warps
  int room, threads, blocks;   // threads that a block has room for, and that it has (whole groups of several warps); blocks
};
constexpr int kSms = 148;
constexpr int kLnMostBlocks = 2 * kSms;   // that leave sums over rows, see ln_threads and ln_grid

LnGrid ln_grid(int what, long long rows, int cols, bool wide, bool bits16) {
  LnGrid g;
  g.wide = wide;
  // 16 elements a thread: what is done once a row and thread (exchanges, addresses) is shared by as many.  Where there are
  // too few rows to fill the GPU a row's own time counts: 8.
  g.each = rows <= kSms && cols <= 4096 ? 8 : 16;
  // The forward keeps little of each: 32 (bf16, 2048 columns 27.8 -> 26.3 us, 8192 40 -> 29; fp32 8192 51 -> 50, but 2048 21.6 -> 22.5).
  if (what == kLnForward && wide && cols >= (bits16 ? 1024 : 4097) && g.each == 16) g.each = 32;
  // The double backward keeps much: 8.  16, with the vectors over the columns in shared memory, for 16-bit elements unless rows are short
  // (512 columns 77 -> 60 us, 2048 90 -> 74, 4096 107 -> 86, 2001 154 -> 122; fp32 2048 62 -> 65, 2001 84 -> 94), and for long rows (8001 fp32
  // 378 -> 225).
  if (what == kLnBwdbwd && cols <= 4096 && !(bits16 && cols > 256 && rows > kSms)) g.each = 8;
  g.lanes = 32;
  while (g.lanes > 2 && g.lanes / 2 * g.each >= cols) g.lanes >>= 1;
  // As many warps as a row needs; what follows takes the next power of two of them.
  g.warps = (cols + 32 * g.each - 1) / (32 * g.each);
  int room = 1;
  while (room < g.warps) room <<= 1;
  // Larger blocks leave fewer sums over rows to add up (16384 x 2048 bf16, backward 44.2 -> 43.0 us), which in the double backward pays
  // for rows of few warps only (8 elements a thread, 512 columns 80 -> 77 us, 2048 90 -> 102).
  const bool several = what == kLnBwdbwd && g.each == 8 && room > 4;
  const int least = what == kLnForward || g.lanes < 32 || several ? 256 : 512;
  auto blocks_of_sm = [&](int threads) {
    const int n = ln_threads(what, g.each) / threads;
    return n > 0 ? n : 1;
  };
  g.room = room * 32 > least ? room * 32 : least;
  // Larger blocks also where these have more rows at once in work (forward, 2501 columns bf16 101 -> 75 us, 5001 108 -> 81).
  auto rows_at_once = [&](int threads) { return blocks_of_sm(threads) * (threads / (32 * g.warps)); };
  if (g.lanes == 32 && g.room < 512 && rows_at_once(512) > rows_at_once(g.room)) g.room = 512;
  if (what == kLnForward && !wide && g.each == 16 && g.room == 512 && rows_at_once(768) > rows_at_once(g.room)) g.room = 768;
  // What fits closer has more registers a thread: long rows of up to 24 warps (double backward, 12288 columns bf16 480 -> 280 us), and in the
  // double backward those of fp32 with up to 12, which then keep the vectors (6144 columns 127 -> 107).
  if (g.room == 1024 && g.warps <= 24 && g.each == 16) g.room = 768;
  if (what == kLnBwdbwd && wide && !bits16 && g.each == 16 && g.warps <= 12) g.room = 384;
  g.threads = g.lanes < 32 ? g.room : g.room / (32 * g.warps) * 32 * g.warps;
  const int groups = g.threads / (g.warps * g.lanes);
  const long long wanted = (rows + groups - 1) / groups;
  const long long resident = static_cast<long long>(kSms) * blocks_of_sm(g.room);
  g.blocks = static_cast<int>(wanted < resident ? wanted : resident);
  return g;
}

template <int WHAT, class T, int V, int NV>
int ln_run(const LnParams& p, const LnGrid& g, cudaStream_t s) {
  auto go = [&](auto threads, auto sub) -> int {
    constexpr int kThreads = decltype(threads)::value;
    constexpr bool kSub = decltype(sub)::value;
    using C = LnCfg<WHAT, T, V, NV, kThreads, kSub>;
    constexpr auto kernel = [] {
      if constexpr (WHAT == kLnForward) return ln_forward_kernel<T, V, NV, kThreads, kSub>;
      else if constexpr (WHAT == kLnBackward) return ln_backward_kernel<T, V, NV, kThreads, kSub>;
      else return ln_bwdbwd_kernel<T, V, NV, kThreads, kSub>;
    }();
    const int st = allow_smem(kernel, C::kSmem);
    if (st != FHOB_OK) return st;
    FHOB_CUDA_OK(launch_pdl(kernel, static_cast<unsigned>(g.blocks), static_cast<unsigned>(g.threads), C::kSmem, 1, s, p));
    return FHOB_OK;
  };
  // (what ln_grid does not ask for is not built)
  constexpr int kEach = NV * V;
  constexpr bool kGrid = kWide<T, V>, kSecond = WHAT == kLnBwdbwd, kHeld = kSecond && kGrid && sizeof(T) == 4 && kEach == 16;
  if constexpr (kEach == 8 || (kEach == 16 && !kSecond))
    if (g.lanes < 32) return go(std::integral_constant<int, 256>{}, std::true_type{});
  if constexpr (kHeld)
    if (g.room == 384) return go(std::integral_constant<int, 384>{}, std::false_type{});
  if constexpr (WHAT == kLnForward || (kSecond && kEach == 8))
    if (g.room == 256) return go(std::integral_constant<int, 256>{}, std::false_type{});
  if constexpr (!(kEach == 16 && WHAT == kLnForward && kGrid))
    if (g.room == 512) return go(std::integral_constant<int, 512>{}, std::false_type{});
  if constexpr (kEach == 16 && !(WHAT == kLnForward && kGrid)) {
    if (g.room == 768) return go(std::integral_constant<int, 768>{}, std::false_type{});
    if (g.room == 1024) return go(std::integral_constant<int, 1024>{}, std::false_type{});
  }
  return FHOB_ERR_SHAPE;
}

template <int WHAT, class T>
int ln_pick(const LnParams& p, const LnGrid& g, cudaStream_t s) {
  constexpr int kPiece = 16 / sizeof(T);
  if constexpr (WHAT == kLnForward)
    if (g.wide && g.each == 32) return ln_run<WHAT, T, kPiece, 32 / kPiece>(p, g, s);
  if (g.wide) return g.each == 8 ? ln_run<WHAT, T, kPiece, 8 / kPiece>(p, g, s) : ln_run<WHAT, T, kPiece, 16 / kPiece>(p, g, s);
  return g.each == 8 ? ln_run<WHAT, T, 2, 4>(p, g, s) : ln_run<WHAT, T, 2, 8>(p, g, s);
}

bool bad_type(int t) { return t != FHOB_BF16 && t != FHOB_F32 && t != FHOB_F16; }

// Checks what the three calls share, fills the parameters and launches; `dw`, `db`: where the sums over rows go.
template <int WHAT>
int ln_call(const FhobLayerNorm* n, LnParams& p, void* dw, void* db, cudaStream_t s) {
  const int es = n->dtype == FHOB_F32 ? 4 : 2;
  const void* matrices[] = {p.x, p.dy, p.v, p.y, p.dx};
  const long long strides[] = {p.x_row, p.dy_row, p.v_row, n->cols, n->cols};
  uintptr_t together = 0;
  for (int i = 0; i < 5; ++i)
    if (matrices[i]) {
      if (strides[i] < 0) return FHOB_ERR_ARG;
      together |= reinterpret_cast<uintptr_t>(matrices[i]) | static_cast<uintptr_t>(strides[i] * es);
    }
  together |= static_cast<uintptr_t>(n->cols) * es;
  if (together % es) return FHOB_ERR_ALIGN;
  uintptr_t vectors = reinterpret_cast<uintptr_t>(dw) | reinterpret_cast<uintptr_t>(db);
  for (const void* vector : {n->w, p.b, p.vw, p.vb}) {
    vectors |= reinterpret_cast<uintptr_t>(vector);
    together |= reinterpret_cast<uintptr_t>(vector);
  }
  if (vectors % (n->w_dtype == FHOB_F32 ? 4 : 2) || (reinterpret_cast<uintptr_t>(n->mean) | reinterpret_cast<uintptr_t>(n->rstd)) % 4) return FHOB_ERR_ALIGN;
  p.w = n->w;
  p.w_f32 = n->w_dtype == FHOB_F32;
  p.rows = static_cast<int>(n->rows);
  p.cols = n->cols;
  p.eps = n->eps;
  p.inv_cols = 1.f / static_cast<float>(n->cols);
  const LnGrid g = ln_grid(WHAT, n->rows, n->cols, together % 16 == 0, es == 2);
  p.warps = g.warps;
  p.lanes = g.lanes;
  if (dw || db) {
    const size_t need = static_cast<size_t>(g.blocks) * 2 * n->cols * sizeof(float);
    if (!n->workspace || (reinterpret_cast<uintptr_t>(n->workspace) & 255u) || n->workspace_bytes < need) return FHOB_ERR_WORKSPACE;
    p.partial = static_cast<float*>(n->workspace);
    p.want_dw = dw != nullptr;
    p.want_db = db != nullptr;
  }
  int st;
  if (n->dtype == FHOB_F32) st = ln_pick<WHAT, float>(p, g, s);
  else st = n->dtype == FHOB_F16 ? ln_pick<WHAT, __half>(p, g, s) : ln_pick<WHAT, __nv_bfloat16>(p, g, s);
  if (st != FHOB_OK || !p.partial) return st;
  const dim3 grid((n->cols + 31) / 32, dw && db ? 2 : 1);
  auto columns = [&](auto type) -> int {
    using W = decltype(type);
    FHOB_CUDA_OK(launch_pdl(ln_columns_kernel<W>, grid, 1024, 0, 1, s, static_cast<const float*>(p.partial), g.blocks, p.cols, static_cast<W*>(dw),
                            static_cast<W*>(db)));
    return FHOB_OK;
  };
  if (n->w_dtype == FHOB_F32) return columns(float{});
  return n->w_dtype == FHOB_F16 ? columns(__half{}) : columns(__nv_bfloat16{});
}

int ln_check(const FhobLayerNorm* n) {
  if (!n || n->rows <= 0 || n->cols <= 0 || !n->x) return FHOB_ERR_ARG;
  if (bad_type(n->dtype) || bad_type(n->w_dtype) || (n->w_dtype != FHOB_F32 && n->w_dtype != n->dtype)) return FHOB_ERR_ARG;
  if (!n->mean || !n->rstd) return FHOB_ERR_ARG;
  return n->cols > FHOB_LAYER_NORM_MAX_COLS || n->rows > FHOB_LAYER_NORM_MAX_ROWS ? FHOB_ERR_SHAPE : FHOB_OK;
}

}  // namespace
}  // namespace fhob

using namespace fhob;

extern "C" {

size_t fhob_layer_norm_workspace_bytes(int32_t cols) {
  return cols > 0 ? static_cast<size_t>(kLnMostBlocks) * 2 * sizeof(float) * static_cast<size_t>(cols) : 0;
}

int fhob_layer_norm(const FhobLayerNorm* n, void* y, void* stream) {
  const int st = ln_check(n);
  if (st != FHOB_OK) return st;
  if (!y || !(n->eps >= 0.f)) return FHOB_ERR_ARG;
  LnParams p = {};
  p.x = n->x; p.x_row = n->x_row;
  p.b = n->b;
  p.y = y;
  p.mean = n->mean; p.rstd = n->rstd;
  return ln_call<kLnForward>(n, p, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

int fhob_layer_norm_backward(const FhobLayerNorm* n, const void* dy, int64_t dy_row, void* dx, void* dw, void* db, void* stream) {
  const int st = ln_check(n);
  if (st != FHOB_OK) return st;
  if (!dy || !dx) return FHOB_ERR_ARG;
  LnParams p = {};
  p.x = n->x; p.x_row = n->x_row;
  p.dy = dy; p.dy_row = dy_row;
  p.mean_in = n->mean; p.rstd_in = n->rstd;
  p.dx = dx;
  return ln_call<kLnBackward>(n, p, dw, db, static_cast<cudaStream_t>(stream));
}

int fhob_layer_norm_bwdbwd(const FhobLayerNorm* n, const void* dy, int64_t dy_row, const void* ddx, int64_t ddx_row, const void* ddw,
                           const void* ddb, void* ddy, void* dx2, void* dw2, void* stream) {
  const int st = ln_check(n);
  if (st != FHOB_OK) return st;
  if (!dy || !ddy || !dx2) return FHOB_ERR_ARG;
  LnParams p = {};
  p.x = n->x; p.x_row = n->x_row;
  p.dy = dy; p.dy_row = dy_row;
  p.v = ddx; p.v_row = ddx_row;
  p.vw = ddw; p.vb = ddb;
  p.mean_in = n->mean; p.rstd_in = n->rstd;
  p.y = ddy; p.dx = dx2;
  return ln_call<kLnBwdbwd>(n, p, dw2, nullptr, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
