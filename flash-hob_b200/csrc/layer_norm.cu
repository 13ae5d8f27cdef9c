// Layer norm over the last dim, and its first and second derivatives: fhob_layer_norm, fhob_layer_norm_backward,
// fhob_layer_norm_bwdbwd.
//
//   mu = mean x, r = 1 / sqrt(mean (x - mu)^2 + eps), h = (x - mu) r                 y = h w + b
//   g = dy w:      dx = r (g - mean g - h mean(g h))          dw = sum dy h          db = sum dy
//   cotangents v of dx, vw of dw, vb of db; a = mean v, c = mean(v h), m = mean g, q = mean(g h):
//     p = v - a - h c:   ddy = r w p + vw h + vb              dw2 = sum dy r p
//     e = vw dy - r (g c + v q):
//       dx2 = r (e - mean e - h mean(e h)) - r^2 h mean(p (g - m - h q))
//   (sums over rows for dw, db, dw2; means over a row).  mean(p (g - m - h q)) equals mean(v g) - a m - c q, but its
//   terms do not cancel when v or g have a large common part.
//
// What bounds it: each matrix is read once and written once, so the memory.  A row belongs to a group of one to 32 warps, which
// keep it in registers (as it came, 16 bits an element) from its only load to its results; sums over a row are
// shuffles, then, if the group has several warps, one exchange through shared memory per round.  Rounds: two in the forward
// (the variance is a sum of squares around the mean), one in the backward, two in the double backward.
// A thread owns the same columns of all its rows, so what the sums over rows add up stays in its registers; the groups
// of a block are added up in shared memory and the blocks' sums in a second launch, always in the same order.
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
  long long rows;
  int cols, warps;                         // warps of a group
  int w_f32;                               // type of w, b, vw, vb: fp32, or that of the matrices
  int want_dw, want_db;
  float eps, inv_cols;
};

// V elements of a row at column c, as they are in memory
template <class T, int V>
struct Piece {
  alignas(V * sizeof(T) > 16 ? 16 : V * sizeof(T)) T e[V];
};
template <class T, int V>
__device__ __forceinline__ void load_piece(Piece<T, V>& to, const T* from) {
  if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(to.e) = *reinterpret_cast<const uint4*>(from);
  else if constexpr (V * sizeof(T) == 4) *reinterpret_cast<uint32_t*>(to.e) = *reinterpret_cast<const uint32_t*>(from);
  else to.e[0] = from[0];
}
template <class T, int V>
__device__ __forceinline__ void store_piece(T* to, const Piece<T, V>& from) {
  if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from.e);
  else if constexpr (V * sizeof(T) == 4) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from.e);
  else to[0] = from.e[0];
}

// What a thread needs to know of its place: its columns are (warp_in_group * 32 + lane + i * width) * V, i < NV.
template <int V>
struct Place {
  int group, groups, lane, warp, warps, width, first;   // groups of a block; width = threads of a group
  __device__ __forceinline__ explicit Place(int warps_per_group) {
    warps = warps_per_group;
    const int w = threadIdx.x >> 5;
    group = w / warps;
    groups = (blockDim.x >> 5) / warps;
    warp = w - group * warps;
    lane = threadIdx.x & 31;
    width = warps * 32;
    first = warp * 32 + lane;
  }
  __device__ __forceinline__ int column(int i) const { return (first + i * width) * V; }
};

// Sums of N values over a group, in every thread of it.  `exchange`: N floats per warp of the block; two areas take turns,
// so that one meeting a round is enough (a warp that is a round ahead writes to the other area, and cannot be two ahead).
template <int N, int V>
__device__ __forceinline__ void group_sum(float (&x)[N], const Place<V>& at, float* exchange) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += __shfl_xor_sync(0xffffffffu, x[i], o);
  if (at.warps == 1) return;
  float* mine = exchange + at.group * at.warps * N;
  if (at.lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) mine[at.warp * N + i] = x[i];
  asm volatile("bar.sync %0, %1;" ::"r"(at.group + 1), "r"(at.width) : "memory");
  // every warp adds up the same numbers in the same order
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = at.lane < at.warps ? mine[at.lane * N + i] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += __shfl_xor_sync(0xffffffffu, x[i], o);
}

// fp32 copies of a vector's elements at this thread's columns; `otherwise` where there is no vector
template <class T, int V, int NV>
__device__ __forceinline__ void load_vector(float (&to)[NV][V], const void* from, int f32, const Place<V>& at, int cols, float otherwise) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = at.column(i) + j;
      to[i][j] = otherwise;
      if (from && c < cols) to[i][j] = f32 ? static_cast<const float*>(from)[c] : static_cast<float>(static_cast<const T*>(from)[c]);
    }
}

template <class T, int V, int NV>
__device__ __forceinline__ void load_row(Piece<T, V> (&to)[NV], const void* from, long long row, long long stride, const Place<V>& at, int cols) {
  const T* base = static_cast<const T*>(from) + row * stride;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (at.column(i) < cols) {
      load_piece<T, V>(to[i], base + at.column(i));
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) to[i].e[j] = static_cast<T>(0.f);
    }
  }
}

// Adds up the groups' sums over rows and leaves the block's in `partial` (cols floats).
template <int V, int NV>
__device__ __forceinline__ void block_columns(const float (&sum)[NV][V], const Place<V>& at, int cols, float* scratch, float* partial) {
  if (at.groups == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (at.column(i) + j < cols) partial[at.column(i) + j] = sum[i][j];
    return;
  }
  // group by group, in their order, through one row of shared memory
  for (int g = 0; g < at.groups; ++g) {
    __syncthreads();
    if (at.group == g) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = at.column(i) + j;
          if (c < cols) scratch[c] = g == 0 ? sum[i][j] : scratch[c] + sum[i][j];
        }
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < cols; c += blockDim.x) partial[c] = scratch[c];
  __syncthreads();
}

template <class T, int V, int NV, int MOST>
__global__ void __launch_bounds__(MOST, 1) ln_forward_kernel(const __grid_constant__ LnParams p) {
  extern __shared__ float exchange[];   // two areas of one float per warp
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const Place<V> at(p.warps);
  float w[NV][V], b[NV][V];
  load_vector<T, V, NV>(w, p.w, p.w_f32, at, p.cols, 1.f);
  load_vector<T, V, NV>(b, p.b, p.w_f32, at, p.cols, 0.f);
  const long long step = static_cast<long long>(gridDim.x) * at.groups;
  for (long long row = static_cast<long long>(blockIdx.x) * at.groups + at.group; row < p.rows; row += step) {
    Piece<T, V> x[NV];
    load_row<T, V, NV>(x, p.x, row, p.x_row, at, p.cols);
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += static_cast<float>(x[i].e[j]);
    group_sum<1, V>(s, at, exchange);
    const float mean = s[0] * p.inv_cols;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = static_cast<float>(x[i].e[j]) - mean;
        if (at.column(i) + j < p.cols) s[0] = fmaf(d, d, s[0]);
      }
    group_sum<1, V>(s, at, exchange + LN_MAX_WARPS);
    const float r = 1.f / sqrtf(fmaf(s[0], p.inv_cols, p.eps));
    T* y = static_cast<T*>(p.y) + row * p.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Piece<T, V> out;
#pragma unroll
      for (int j = 0; j < V; ++j) out.e[j] = static_cast<T>(fmaf((static_cast<float>(x[i].e[j]) - mean) * r, w[i][j], b[i][j]));
      if (at.column(i) < p.cols) store_piece<T, V>(y + at.column(i), out);
    }
    if (at.first == 0) {
      p.mean[row] = mean;
      p.rstd[row] = r;
    }
  }
}

template <class T, int V, int NV, int MOST>
__global__ void __launch_bounds__(MOST, 1) ln_backward_kernel(const __grid_constant__ LnParams p) {
  extern __shared__ float exchange[];   // two areas of two floats per warp, then a row for the sums over rows
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const Place<V> at(p.warps);
  float w[NV][V], dw[NV][V], db[NV][V];
  load_vector<T, V, NV>(w, p.w, p.w_f32, at, p.cols, 1.f);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.f;
  const long long step = static_cast<long long>(gridDim.x) * at.groups;
  int turn = 0;
  for (long long row = static_cast<long long>(blockIdx.x) * at.groups + at.group; row < p.rows; row += step, turn ^= 1) {
    Piece<T, V> x[NV], dy[NV];
    load_row<T, V, NV>(x, p.x, row, p.x_row, at, p.cols);
    load_row<T, V, NV>(dy, p.dy, row, p.dy_row, at, p.cols);
    const float mean = p.mean_in[row], r = p.rstd_in[row];
    float s[2] = {0.f, 0.f};   // sums of g, g h  (dy is zero behind the last column)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float h = (static_cast<float>(x[i].e[j]) - mean) * r, d = static_cast<float>(dy[i].e[j]), g = d * w[i][j];
        dw[i][j] = fmaf(d, h, dw[i][j]);
        db[i][j] += d;
        s[0] += g;
        s[1] = fmaf(g, h, s[1]);
      }
    group_sum<2, V>(s, at, exchange + turn * 2 * LN_MAX_WARPS);
    const float m = s[0] * p.inv_cols, q = s[1] * p.inv_cols;
    T* dx = static_cast<T*>(p.dx) + row * p.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Piece<T, V> out;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float h = (static_cast<float>(x[i].e[j]) - mean) * r, g = static_cast<float>(dy[i].e[j]) * w[i][j];
        out.e[j] = static_cast<T>(r * (g - m - h * q));
      }
      if (at.column(i) < p.cols) store_piece<T, V>(dx + at.column(i), out);
    }
  }
  if (p.partial) {
    float* scratch = exchange + 4 * LN_MAX_WARPS;
    float* to = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols;
    if (p.want_dw) block_columns<V, NV>(dw, at, p.cols, scratch, to);
    if (p.want_db) block_columns<V, NV>(db, at, p.cols, scratch, to + p.cols);
  }
}

template <class T, int V, int NV, int MOST>
__global__ void __launch_bounds__(MOST, 1) ln_bwdbwd_kernel(const __grid_constant__ LnParams p) {
  extern __shared__ float exchange[];   // areas of four and of three floats per warp, then a row for the sums over rows
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const Place<V> at(p.warps);
  float w[NV][V], vw[NV][V], vb[NV][V], dw2[NV][V];
  load_vector<T, V, NV>(w, p.w, p.w_f32, at, p.cols, 1.f);
  load_vector<T, V, NV>(vw, p.vw, p.w_f32, at, p.cols, 0.f);
  load_vector<T, V, NV>(vb, p.vb, p.w_f32, at, p.cols, 0.f);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) dw2[i][j] = 0.f;
  const long long step = static_cast<long long>(gridDim.x) * at.groups;
  for (long long row = static_cast<long long>(blockIdx.x) * at.groups + at.group; row < p.rows; row += step) {
    Piece<T, V> x[NV], dy[NV], v[NV];
    load_row<T, V, NV>(x, p.x, row, p.x_row, at, p.cols);
    load_row<T, V, NV>(dy, p.dy, row, p.dy_row, at, p.cols);
    if (p.v) {
      load_row<T, V, NV>(v, p.v, row, p.v_row, at, p.cols);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) v[i].e[j] = static_cast<T>(0.f);
    }
    const float mean = p.mean_in[row], r = p.rstd_in[row];
    float s[4] = {0.f, 0.f, 0.f, 0.f};   // v, v h, g, g h
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float h = (static_cast<float>(x[i].e[j]) - mean) * r, u = static_cast<float>(v[i].e[j]);
        const float g = static_cast<float>(dy[i].e[j]) * w[i][j];
        s[0] += u;
        s[1] = fmaf(u, h, s[1]);
        s[2] += g;
        s[3] = fmaf(g, h, s[3]);
      }
    group_sum<4, V>(s, at, exchange);
    const float a = s[0] * p.inv_cols, c = s[1] * p.inv_cols, m = s[2] * p.inv_cols, q = s[3] * p.inv_cols;
    float t[3] = {0.f, 0.f, 0.f};        // p (g - m - h q), e, e h
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float h = (static_cast<float>(x[i].e[j]) - mean) * r, u = static_cast<float>(v[i].e[j]), d = static_cast<float>(dy[i].e[j]);
        const float g = d * w[i][j], pp = u - a - h * c;
        const float e = fmaf(vw[i][j], d, -r * (g * c + u * q));   // zero behind the last column, as d and u are
        dw2[i][j] = fmaf(d * r, pp, dw2[i][j]);
        if (at.column(i) + j < p.cols) t[0] = fmaf(pp, g - m - h * q, t[0]);
        t[1] += e;
        t[2] = fmaf(e, h, t[2]);
      }
    group_sum<3, V>(t, at, exchange + 4 * LN_MAX_WARPS);
    const float k = t[0] * p.inv_cols * r, me = t[1] * p.inv_cols, meh = t[2] * p.inv_cols;
    T *ddy = static_cast<T*>(p.y) + row * p.cols, *dx2 = static_cast<T*>(p.dx) + row * p.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Piece<T, V> o1, o2;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float h = (static_cast<float>(x[i].e[j]) - mean) * r, u = static_cast<float>(v[i].e[j]), d = static_cast<float>(dy[i].e[j]);
        const float e = fmaf(vw[i][j], d, -r * (d * w[i][j] * c + u * q));
        o1.e[j] = static_cast<T>(fmaf(r * w[i][j], u - a - h * c, fmaf(vw[i][j], h, vb[i][j])));
        o2.e[j] = static_cast<T>(r * (e - me - h * (meh + k)));
      }
      if (at.column(i) < p.cols) {
        store_piece<T, V>(ddy + at.column(i), o1);
        store_piece<T, V>(dx2 + at.column(i), o2);
      }
    }
  }
  if (p.partial) block_columns<V, NV>(dw2, at, p.cols, exchange + 7 * LN_MAX_WARPS, p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols);
}

// Sums over the blocks: a warp takes 32 columns, eight warps of a block a share of the rows of `partial` each, in order.
template <class W>
__global__ void __launch_bounds__(256) ln_columns_kernel(const float* partial, int blocks, int cols, W* dw, W* db) {
  __shared__ float part[8][33];
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool second = blockIdx.y == 1 || !dw;
  const int c = blockIdx.x * 32 + lane;
  const float* from = partial + (second ? cols : 0) + c;
  float sum = 0.f;
  if (c < cols)
#pragma unroll 8
    for (int i = warp; i < blocks; i += 8) sum += from[static_cast<long long>(i) * 2 * cols];
  part[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) sum += part[i][lane];
    (second ? db : dw)[c] = static_cast<W>(sum);
  }
}

enum { kLnForward, kLnBackward, kLnBwdbwd };

// How a call is cut up.  A thread has at most 16 elements of a row: what it keeps of each column besides (weights, sums:
// two to four fp32 numbers) then stays in registers at two blocks of 256 threads an SM.
struct LnGrid {
  int v, nv, warps, threads, blocks;
};
constexpr int kSms = 148;
constexpr int kLnMostBlocks = 4 * kSms;

LnGrid ln_grid(int what, long long rows, int cols, int element, int v) {
  LnGrid g;
  g.v = v;
  // 8 elements a thread where that is one warp's row anyway, or where there are too few rows to fill the GPU and
  // a row's own time counts; else 16
  const int each = cols <= 256 || rows <= kSms ? 8 : 16;
  g.nv = each / v;
  g.warps = 1;
  while (g.warps < LN_MAX_WARPS && g.warps * 32 * each < cols) g.warps <<= 1;
  if (g.warps * 32 * each < cols) g.nv = 16 / v;
  g.threads = g.warps * 32 > 256 ? g.warps * 32 : 256;
  const int groups = g.threads / (g.warps * 32);
  const long long wanted = (rows + groups - 1) / groups;
  const long long resident = static_cast<long long>(kSms) * (what == kLnForward ? 4 : 2) * 256 / g.threads;
  g.blocks = static_cast<int>(wanted < resident ? wanted : (resident > kSms ? resident : kSms));
  return g;
}

template <int WHAT, class T, int V, int NV>
int ln_run(const LnParams& p, const LnGrid& g, cudaStream_t s) {
  auto go = [&](auto most) -> int {
    constexpr int kMost = decltype(most)::value;
    constexpr auto kernel = WHAT == kLnForward ? ln_forward_kernel<T, V, NV, kMost>
                                               : (WHAT == kLnBackward ? ln_backward_kernel<T, V, NV, kMost> : ln_bwdbwd_kernel<T, V, NV, kMost>);
    // areas for the sums of a row, and of several groups (rows of up to 4 warps * 32 * 16 elements) a row for the sums over rows
    const int groups = g.threads / (g.warps * 32);
    const int smem = 4 * (7 * LN_MAX_WARPS + (groups > 1 ? p.cols : 0));
    FHOB_CUDA_OK(launch_pdl(kernel, static_cast<unsigned>(g.blocks), static_cast<unsigned>(g.threads), smem, 1, s, p));
    return FHOB_OK;
  };
  return g.threads > 512 ? go(std::integral_constant<int, 1024>{}) : go(std::integral_constant<int, 512>{});
}

template <int WHAT, class T>
int ln_pick(const LnParams& p, const LnGrid& g, cudaStream_t s) {
  constexpr int kWide = 16 / sizeof(T);
  if (g.v == kWide) return g.nv * g.v == 8 ? ln_run<WHAT, T, kWide, 8 / kWide>(p, g, s) : ln_run<WHAT, T, kWide, 16 / kWide>(p, g, s);
  if constexpr (sizeof(T) == 2)
    if (g.v == 2) return g.nv == 4 ? ln_run<WHAT, T, 2, 4>(p, g, s) : ln_run<WHAT, T, 2, 8>(p, g, s);
  return g.nv == 8 ? ln_run<WHAT, T, 1, 8>(p, g, s) : ln_run<WHAT, T, 1, 16>(p, g, s);
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
  const int v = together % 16 == 0 ? 16 / es : (es == 2 && together % 4 == 0 ? 2 : 1);
  p.w = n->w;
  p.w_f32 = n->w_dtype == FHOB_F32;
  p.rows = n->rows;
  p.cols = n->cols;
  p.eps = n->eps;
  p.inv_cols = 1.f / static_cast<float>(n->cols);
  const LnGrid g = ln_grid(WHAT, n->rows, n->cols, es, v);
  p.warps = g.warps;
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
    FHOB_CUDA_OK(launch_pdl(ln_columns_kernel<W>, grid, 256, 0, 1, s, static_cast<const float*>(p.partial), g.blocks, p.cols, static_cast<W*>(dw),
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
  return n->cols > FHOB_LAYER_NORM_MAX_COLS ? FHOB_ERR_SHAPE : FHOB_OK;
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
