// Rotary positions with several axes: fhob_rotary.
//
// The first 2 * pairs elements of a row are pairs (x, y), either (j, pairs + j) or neighbours (2 j, 2 j + 1);
// pair j turns by the angle a = position[axis of j] * frequency[j]:
//
//     (x, y) -> (x cos a - y sin a, x sin a + y cos a)          inverse: the angle negated
//
// Angles.  Positions go to 2^31 and beyond, where the fp32 product of position and frequency is off by whole
// radians.  A frequency is taken as a 64-bit fraction of a turn, frequency / 2 pi mod 1, times 2^64; its integer product
// with the position, which drops whole turns by itself, is the angle as such a fraction: exact up to
// position * frequency * 2^-52 radians, from the double that the frequency is divided in.  The upper 32 bits make
// the fp32 argument of sincospif (rounded to at most 2^-25 of a turn half: 1e-7 radians).
//
// What bounds it: the row is read once and written once, so the memory.  A thread owns the same pairs of one token
// in `group` heads: it works out their sines once, then passes over the heads of all tensors, 16 bytes of either
// half of a row a load (a warp covers whole rows), four heads in flight.
#include "fhob_common.cuh"
#include "tc_common.cuh"

namespace fhob {
namespace {

constexpr int RO_THREADS = 256;

struct RoParams {
  const void* in[2];
  void* out[2];
  int heads[2];
  long long in_row[2], in_head[2], in_batch[2];   // element strides; results are contiguous (batch, heads, n, d)
  const void* positions;
  long long pos_axis, pos_batch, pos_n;           // element strides
  const void* frequencies;
  int positions64, frequencies64;
  long long n;
  long long tokens;                               // batch * n
  int d, pairs, tail, per_row, tokens_per_block, group, groups;
  float sign;
  uint8_t axis[FHOB_ROTARY_MAX_PAIRS];
};

// N elements, aligned to the largest power of two (up to 16 bytes) that divides their bytes.
template <int N, class T>
__device__ __forceinline__ void copy_elements(T* to, const T* from) {
  constexpr int kBytes = N * static_cast<int>(sizeof(T));
  if constexpr (kBytes >= 16) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(from)[i];
  } else if constexpr (kBytes == 8) {
    *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(from);
  } else if constexpr (kBytes == 4) {
    *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = from[i];
  }
}

// frequency / 2 pi mod 1 as a 64-bit fraction
__device__ __forceinline__ unsigned long long turn_fraction(double frequency) {
  const double turns = frequency * 0.15915494309189533577;   // 1 / (2 pi)
  return __double2ull_rn((turns - floor(turns)) * 18446744073709551616.0);   // (2^64 saturates)
}

// P pairs a thread.  P == 1 reads and writes single elements, at any alignment.
template <class T, int P, bool NEIGHBOURS>
__global__ void __launch_bounds__(RO_THREADS) rotary_kernel(const __grid_constant__ RoParams p) {
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const long long token_block = blockIdx.x / static_cast<unsigned>(p.groups);
  const int group = static_cast<int>(blockIdx.x - token_block * p.groups);
  const int local = threadIdx.x / p.per_row;
  const long long token = token_block * p.tokens_per_block + local;
  if (local >= p.tokens_per_block || token >= p.tokens) return;
  const long long batch = token / p.n, at = token - batch * p.n;
  const int all = p.heads[0] + p.heads[1], h_begin = group * p.group, h_end = min(all, h_begin + p.group);
  const int rotated = p.pairs / P;   // pieces of a row that turn; the others are copied
  const long long pos_at = batch * p.pos_batch + at * p.pos_n;

  for (int piece = threadIdx.x - local * p.per_row; piece < rotated + p.tail / P; piece += p.per_row) {
    const bool turns = piece < rotated;
    float co[P], si[P];
    if (turns) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int j = piece * P + i;
        const double f = p.frequencies64 ? static_cast<const double*>(p.frequencies)[j] : static_cast<double>(static_cast<const float*>(p.frequencies)[j]);
        const long long where = p.axis[j] * p.pos_axis + pos_at;
        const long long pos = p.positions64 ? static_cast<const long long*>(p.positions)[where] : static_cast<long long>(static_cast<const int*>(p.positions)[where]);
        const unsigned long long angle = turn_fraction(f) * static_cast<unsigned long long>(pos);
        sincospif(static_cast<float>(static_cast<int>(angle >> 32)) * 4.656612873077393e-10f, &si[i], &co[i]);   // 2^-31: half turns
        si[i] *= p.sign;
      }
    }
    // columns of the two elements of the piece's first pair, or of the piece itself
    const int c0 = turns ? (NEIGHBOURS ? 2 * P * piece : P * piece) : 2 * p.pairs + P * (piece - rotated);
    const int c1 = NEIGHBOURS ? c0 + P : c0 + p.pairs;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int first = t == 0 ? 0 : p.heads[0], lo = max(h_begin - first, 0), hi = min(h_end - first, p.heads[t]);
      const T* in = static_cast<const T*>(p.in[t]) + batch * p.in_batch[t] + at * p.in_row[t];
      T* out = static_cast<T*>(p.out[t]) + (batch * p.heads[t] * p.n + at) * p.d;
      const long long in_head = p.in_head[t], out_head = p.n * p.d;
      constexpr int kAhead = 4;
      for (int h = lo; h < hi; h += kAhead) {
        alignas(16) T a[kAhead][P], b[kAhead][P];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (h + u < hi) {
            const T* row = in + (h + u) * in_head;
            copy_elements<P>(a[u], row + c0);
            if (turns) copy_elements<P>(b[u], row + c1);
          }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (h + u < hi) {
            T* row = out + (h + u) * out_head;
            if (turns) {
#pragma unroll
              for (int i = 0; i < P; ++i) {
                // neighbours: the piece's 2 P elements are x0 y0 x1 y1 ..., the first half of them in a
                T& ex = NEIGHBOURS ? (2 * i < P ? a[u][2 * i < P ? 2 * i : 0] : b[u][2 * i < P ? 0 : 2 * i - P]) : a[u][i];
                T& ey = NEIGHBOURS ? (2 * i + 1 < P ? a[u][2 * i + 1 < P ? 2 * i + 1 : 0] : b[u][2 * i + 1 < P ? 0 : 2 * i + 1 - P]) : b[u][i];
                const float x = static_cast<float>(ex), y = static_cast<float>(ey);
                ex = static_cast<T>(fmaf(x, co[i], -(y * si[i])));
                ey = static_cast<T>(fmaf(x, si[i], y * co[i]));
              }
              copy_elements<P>(row + c1, b[u]);
            }
            copy_elements<P>(row + c0, a[u]);
          }
      }
    }
  }
}

template <class T>
int rotary_launch(const FhobRotary& r, RoParams& p, cudaStream_t s) {
  // most pairs a thread can take: 16 bytes of either element kind, and whole pieces on every address and stride
  constexpr int kMost = 16 / sizeof(T);
  int most = kMost;
  auto fits = [&](int n) {
    const long long bytes = n * static_cast<long long>(sizeof(T));
    if (r.pairs % n || p.tail % n || r.d % n) return false;
    for (int t = 0; t < r.tensors; ++t) {
      if ((reinterpret_cast<uintptr_t>(p.in[t]) | reinterpret_cast<uintptr_t>(p.out[t])) & static_cast<uintptr_t>(bytes - 1)) return false;
      if (p.in_row[t] * static_cast<long long>(sizeof(T)) % bytes || p.in_head[t] * static_cast<long long>(sizeof(T)) % bytes ||
          p.in_batch[t] * static_cast<long long>(sizeof(T)) % bytes)
        return false;
    }
    return r.d * static_cast<long long>(sizeof(T)) % bytes == 0 && 2 * r.pairs * static_cast<long long>(sizeof(T)) % bytes == 0;
  };
  while (most > 1 && !fits(most)) most >>= 1;
  auto go = [&](auto per_thread, auto neighbours) -> int {
    constexpr int P = decltype(per_thread)::value;
    constexpr auto kernel = rotary_kernel<T, P, decltype(neighbours)::value>;
    const int pieces = (r.pairs + p.tail) / P;
    p.per_row = pieces < RO_THREADS ? pieces : RO_THREADS;
    p.tokens_per_block = RO_THREADS / p.per_row;
    const long long token_blocks = (p.tokens + p.tokens_per_block - 1) / p.tokens_per_block;
    const int all = p.heads[0] + p.heads[1];
    // Heads a thread passes over: sixteen share the work for the sines, fewer while the blocks do not fill the GPU.
    p.group = 16;
    while (p.group > 1 && token_blocks * ((all + p.group - 1) / p.group) < 4LL * sm_count()) p.group >>= 1;
    p.groups = (all + p.group - 1) / p.group;
    if (token_blocks > 0x7fffffffLL / p.groups) return FHOB_ERR_SHAPE;
    FHOB_CUDA_OK(launch_pdl(kernel, static_cast<unsigned>(token_blocks * p.groups), RO_THREADS, 0, 1, s, p));
    return FHOB_OK;
  };
  auto pick = [&](auto neighbours) -> int {
    if constexpr (kMost == 8)
      if (most == 8) return go(std::integral_constant<int, 8>{}, neighbours);
    if (most >= 4) return go(std::integral_constant<int, 4>{}, neighbours);
    if (most == 2) return go(std::integral_constant<int, 2>{}, neighbours);
    return go(std::integral_constant<int, 1>{}, neighbours);
  };
  return r.interleaved ? pick(std::true_type{}) : pick(std::false_type{});
}

}  // namespace
}  // namespace fhob

using namespace fhob;

extern "C" int fhob_rotary(const FhobRotary* r, void* stream) {
  if (!r || r->tensors < 1 || r->tensors > 2 || r->batch <= 0 || r->n <= 0 || r->d <= 0) return FHOB_ERR_ARG;
  if (r->pairs < 1 || r->axes < 1 || !r->positions || !r->frequencies || !r->axis_of_pair) return FHOB_ERR_ARG;
  if (r->dtype != FHOB_BF16 && r->dtype != FHOB_F32 && r->dtype != FHOB_F16) return FHOB_ERR_ARG;
  if (r->pairs > FHOB_ROTARY_MAX_PAIRS || 2 * r->pairs > r->d || r->d > FHOB_ROTARY_MAX_DIM) return FHOB_ERR_SHAPE;
  RoParams p = {};
  for (int t = 0; t < r->tensors; ++t) {
    const FhobRotaryTensor& x = r->tensor[t];
    if (!x.in || !x.out || x.heads <= 0) return FHOB_ERR_ARG;
    if (x.heads > (1 << 20)) return FHOB_ERR_SHAPE;
    const uintptr_t es = r->dtype == FHOB_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(x.in) | reinterpret_cast<uintptr_t>(x.out)) % es) return FHOB_ERR_ALIGN;
    p.in[t] = x.in;
    p.out[t] = x.out;
    p.heads[t] = x.heads;
    p.in_row[t] = x.row; p.in_head[t] = x.head; p.in_batch[t] = x.batch;
  }
  for (int i = 0; i < r->pairs; ++i) {
    if (r->axis_of_pair[i] >= r->axes) return FHOB_ERR_ARG;
    p.axis[i] = r->axis_of_pair[i];
  }
  p.positions = r->positions;
  p.pos_axis = r->pos_axis; p.pos_batch = r->pos_batch; p.pos_n = r->pos_n;
  p.frequencies = r->frequencies;
  p.positions64 = r->positions_are_64_bit; p.frequencies64 = r->frequencies_are_64_bit;
  p.n = r->n;
  if (r->batch > 0x7fffffffffffLL / r->n) return FHOB_ERR_SHAPE;
  p.tokens = r->batch * r->n;
  p.d = r->d; p.pairs = r->pairs; p.tail = r->d - 2 * r->pairs;
  p.sign = r->inverse ? -1.f : 1.f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (r->dtype == FHOB_F32) return rotary_launch<float>(*r, p, s);
  return r->dtype == FHOB_F16 ? rotary_launch<__half>(*r, p, s) : rotary_launch<__nv_bfloat16>(*r, p, s);
}
