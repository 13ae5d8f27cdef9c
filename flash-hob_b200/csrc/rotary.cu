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
// What bounds it: a row is read once and written once, so the memory; then the instructions for the sines, which cost
// as many as a dozen heads' rows if every thread works out its own.  A block takes a few tokens in all heads of all tensors.
// Its threads work out the angles of these tokens together, into shared memory; then a thread owns four pairs
// of one token's rows (a warp covers whole rows) and passes over heads, four in flight, the first of them while
// the angles are worked out.  32 heads N = 8192 D = 128 bf16: 46 us, 5.8 TB/s (55 when every thread worked out its own angles);
// a token of 8 x 32 heads 3.2 us.  fp32, 32 + 32 heads N = 8192 D = 128: 89 us, 6.0 TB/s.
#include "fhob_common.cuh"
#include "tc_common.cuh"

namespace fhob {
namespace {

constexpr int RO_THREADS = 256;
constexpr int RO_ANGLES = 2048;   // most angles of a block

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
  int d, pairs, tail;
  int per_row, block_tokens, copies;              // threads of a row, tokens of a block, heads it works on at once
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

// P elements in memory order <-> fp32 pairs (P == 1: the first of a pair)
template <class T, int P>
struct Elements {
  static constexpr int kHalf = P > 1 ? P / 2 : 1;
  alignas(P * sizeof(T) > 16 ? 16 : P * sizeof(T)) T e[P];
  __device__ __forceinline__ void unpack(float2 (&x)[kHalf]) const {
    if constexpr (P == 1) {
      x[0] = make_float2(static_cast<float>(e[0]), 0.f);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < kHalf; ++i) x[i] = make_float2(e[2 * i], e[2 * i + 1]);
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(e);
#pragma unroll
      for (int i = 0; i < kHalf; ++i) {
        if constexpr (std::is_same<T, __half>::value) x[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        else x[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      }
    }
  }
  __device__ __forceinline__ void pack(const float2 (&x)[kHalf]) {
    if constexpr (P == 1) {
      e[0] = static_cast<T>(x[0].x);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < kHalf; ++i) {
        e[2 * i] = x[i].x;
        e[2 * i + 1] = x[i].y;
      }
    } else {
      uint32_t* w = reinterpret_cast<uint32_t*>(e);
#pragma unroll
      for (int i = 0; i < kHalf; ++i) w[i] = pack16<std::is_same<T, __half>::value>(x[i].x, x[i].y);
    }
  }
};

// P pairs a thread.  P == 1 reads and writes single elements, at any alignment.
template <class T, int P, bool NEIGHBOURS>
__global__ void __launch_bounds__(RO_THREADS, 4) rotary_kernel(const __grid_constant__ RoParams p) {
  __shared__ float2 angles[RO_ANGLES];   // [token][pair]: cosine, sine
  pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  const long long first_token = static_cast<long long>(blockIdx.x) * p.block_tokens;
  const int slots = p.block_tokens * p.per_row, copy = threadIdx.x / slots, slot = threadIdx.x - copy * slots;
  const int local = slot / p.per_row, rotated = p.pairs / P;   // pieces of a row that turn; the others are copied
  const int here = static_cast<int>(min(static_cast<long long>(p.block_tokens), p.tokens - first_token));
  const bool works = copy < p.copies && local < here;
  // batch entry and place in it of the block's token t
  const long long first_batch = p.tokens <= 0x7fffffff ? static_cast<int>(first_token) / static_cast<int>(p.n) : first_token / p.n;
  const long long first_at = first_token - first_batch * p.n;
  auto place_of = [&](int t, long long& batch, long long& at) {
    batch = first_batch;
    at = first_at + t;
    if (at < p.n) return;
    const long long more = at <= 0x7fffffff ? static_cast<int>(at) / static_cast<int>(p.n) : at / p.n;
    batch += more;
    at -= more * p.n;
  };
  long long batch, at;
  place_of(works ? local : 0, batch, at);

  constexpr int kAhead = 4, H = Elements<T, P>::kHalf;
  Elements<T, P> a[kAhead], b[kAhead];
  int piece = slot - local * p.per_row, c0 = 0, c1 = 0;
  bool turns = false;
  // heads copy, copy + copies, ... of one tensor, then of the other, four at a time
  const T* in;
  T* out;
  long long in_step, out_step;
  int tensor, left;
  auto start = [&](int t) {
    tensor = t;
    left = p.heads[t] - copy;
    in_step = p.copies * p.in_head[t];
    out_step = p.copies * p.n * p.d;
    in = static_cast<const T*>(p.in[t]) + batch * p.in_batch[t] + at * p.in_row[t] + copy * p.in_head[t];
    out = static_cast<T*>(p.out[t]) + ((batch * p.heads[t] + copy) * p.n + at) * p.d;
  };
  auto begin = [&] {   // columns of the two elements of the piece's first pair, or of the piece itself
    turns = piece < rotated;
    c0 = turns ? (NEIGHBOURS ? 2 * P * piece : P * piece) : 2 * p.pairs + P * (piece - rotated);
    c1 = NEIGHBOURS ? c0 + P : c0 + p.pairs;
    start(0);
    if (left <= 0) start(1);
  };
  auto load = [&] {
    const T* row = in;
#pragma unroll
    for (int u = 0; u < kAhead; ++u, row += in_step)
      if (u * p.copies < left) {
        copy_elements<P>(a[u].e, row + c0);
        if (turns) copy_elements<P>(b[u].e, row + c1);
      }
  };
  if (works) {
    begin();
    load();
  }

  {
    int t = threadIdx.x / p.pairs, j = threadIdx.x - t * p.pairs, known = -1;
    const int t_step = RO_THREADS / p.pairs, j_step = RO_THREADS - t_step * p.pairs;
    unsigned long long fraction = 0;
    auto position = [&](int t, int j) {
      if (t >= here) return 0LL;
      long long tb, ta;
      place_of(t, tb, ta);
      const long long where = p.axis[j] * p.pos_axis + tb * p.pos_batch + ta * p.pos_n;
      return p.positions64 ? static_cast<const long long*>(p.positions)[where] : static_cast<long long>(static_cast<const int*>(p.positions)[where]);
    };
    long long pos = position(t, j);
    while (t < here) {
      int next_t = t + t_step, next_j = j + j_step;
      if (next_j >= p.pairs) {
        next_j -= p.pairs;
        ++next_t;
      }
      const long long next_pos = position(next_t, next_j);   // on its way meanwhile
      if (j != known) {
        const double f = p.frequencies64 ? static_cast<const double*>(p.frequencies)[j] : static_cast<double>(static_cast<const float*>(p.frequencies)[j]);
        fraction = turn_fraction(f);
        known = j;
      }
      const unsigned long long angle = fraction * static_cast<unsigned long long>(pos);
      float2 x;
      sincospif(static_cast<float>(static_cast<int>(angle >> 32)) * 4.656612873077393e-10f, &x.y, &x.x);   // 2^-31: half turns
      x.y *= p.sign;
      angles[t * p.pairs + j] = x;
      t = next_t;
      j = next_j;
      pos = next_pos;
    }
  }
  __syncthreads();
  if (!works) return;

  for (;;) {
    float2 co[H], si[H];   // of pairs 2 i and 2 i + 1 of the piece
    if (turns) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 x = angles[local * p.pairs + piece * P + i];
        (i % 2 ? co[i / 2].y : co[i / 2].x) = x.x;
        (i % 2 ? si[i / 2].y : si[i / 2].x) = x.y;
      }
    }
    while (left > 0) {
      T* row = out;
#pragma unroll
      for (int u = 0; u < kAhead; ++u, row += out_step)
        if (u * p.copies < left) {
          if (turns) {
            float2 x[H], y[H];
            a[u].unpack(x);
            b[u].unpack(y);
            if constexpr (NEIGHBOURS && P > 1) {   // x0 y0 x1 y1 ...: the first half of them in a
              float2 both[2 * H];
#pragma unroll
              for (int i = 0; i < H; ++i) {
                both[i] = x[i];
                both[H + i] = y[i];
              }
#pragma unroll
              for (int i = 0; i < P; ++i) {
                const float c = i % 2 ? co[i / 2].y : co[i / 2].x, d = i % 2 ? si[i / 2].y : si[i / 2].x;
                both[i] = __ffma2_rn(both[i], make_float2(c, c), __fmul2_rn(make_float2(both[i].y, both[i].x), make_float2(-d, d)));
              }
#pragma unroll
              for (int i = 0; i < H; ++i) {
                x[i] = both[i];
                y[i] = both[H + i];
              }
            } else {
#pragma unroll
              for (int i = 0; i < H; ++i) {
                const float2 px = x[i], minus = make_float2(-si[i].x, -si[i].y);
                x[i] = __ffma2_rn(px, co[i], __fmul2_rn(y[i], minus));
                y[i] = __ffma2_rn(px, si[i], __fmul2_rn(y[i], co[i]));
              }
            }
            a[u].pack(x);
            b[u].pack(y);
            copy_elements<P>(row + c1, b[u].e);
          }
          copy_elements<P>(row + c0, a[u].e);
        }
      in += kAhead * in_step;
      out += kAhead * out_step;
      left -= kAhead * p.copies;
      if (left <= 0 && tensor == 0) start(1);
      if (left > 0) load();
    }
    piece += p.per_row;   // (rows of more pieces than a block has threads)
    if (piece >= rotated + p.tail / P) break;
    begin();
    load();
  }
}

template <class T>
int rotary_launch(const FhobRotary& r, RoParams& p, cudaStream_t s) {
  // most pairs a thread can take: whole pieces on every address and stride
  constexpr int kMost = 4;   // (8 bytes of a 16-bit row a load: with 16 the registers leave half the threads, 32 heads N = 8192 D = 128 56 -> 46 us)
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
    const int pieces = (r.pairs + p.tail) / P, all = p.heads[0] + p.heads[1];
    p.per_row = pieces < RO_THREADS ? pieces : RO_THREADS;
    // A block works on `copies` heads of its tokens at once, four heads in flight each: up to 16 heads a copy (32 + 1 heads
    // N = 8192 D = 128 with 8 32.1 us, with 16 26.8), 8 by itself (8 + 8 heads with 16 52.5 us, with 8 48.6), and fewer where the tokens are too
    // few to fill the GPU.  (The angle of a pair from positions brought into shared memory first: 1 + 1 heads 192 -> 147 us, but 16 + 16 46 -> 48.)
    const int most = RO_THREADS / p.per_row;
    p.block_tokens = most;
    auto blocks = [&] { return (p.tokens + p.block_tokens - 1) / p.block_tokens; };
    while (p.block_tokens > 1 && (p.block_tokens * r.pairs > RO_ANGLES || (all + most / p.block_tokens - 1) / (most / p.block_tokens) > (p.block_tokens == most ? 8 : 16) || blocks() < 4LL * sm_count()) &&
           (p.block_tokens * r.pairs > RO_ANGLES || most / (p.block_tokens / 2) <= all))
      p.block_tokens >>= 1;
    p.copies = most / p.block_tokens;
    if (blocks() > 0x7fffffffLL) return FHOB_ERR_SHAPE;
    FHOB_CUDA_OK(launch_pdl(kernel, static_cast<unsigned>(blocks()), RO_THREADS, 0, 1, s, p));
    return FHOB_OK;
  };
  auto pick = [&](auto neighbours) -> int {
    if (most == 4) return go(std::integral_constant<int, 4>{}, neighbours);
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
  if (reinterpret_cast<uintptr_t>(r->positions) % (r->positions_are_64_bit ? 8 : 4) || reinterpret_cast<uintptr_t>(r->frequencies) % (r->frequencies_are_64_bit ? 8 : 4))
    return FHOB_ERR_ALIGN;
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
