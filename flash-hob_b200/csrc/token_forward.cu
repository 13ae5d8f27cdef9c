// Forward of one or two queries (a token that is answered with) against a window and first keys: O and the logsumexp.
//
//   s_j = scale q . k_j,  O = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  L = m + log sum_j exp(s_j - m)
//
// What bounds it: every visible key and value is read once for the one or two queries, so the memory: 128 heads of one query,
// W = 1024 and 4 first keys, D = 128 read 67 MB.  The tensor-core forward has 128-row query tiles and goes through a head
// in one CTA, tile after tile: 26 us there.  Here 15.5 us (4.3 TB/s; 4000 keys 5.3, 8000 6.1, fp32 5.0, 6.2 and 6.6):
//  - eight lanes read one key's row, one, two or four times 16 bytes a lane: a product takes three shuffles.  Each such group goes
//    through keys of its own with a running maximum and sum of its own: groups, warps and CTAs meet at the end;
//  - a group takes four keys at a time: their rows of K and V are all on their way before the first is used.  What counts besides is
//    the number of instructions, since a call of few heads has one warp a scheduler: with 16 lanes a key 16 heads take 9.5 us
//    instead of 5.8 (and a ring of asynchronous copies gained nothing);
//  - a head's keys are shared by the CTAs of a cluster, five batches a CTA and up to 8 CTAs: a number that depends on the
//    lengths alone, as the order in which their results are added up.
#include "tc_common.cuh"

namespace fhob {
namespace {

struct TkParams {
  const void *q, *k, *v;
  void* o;             // NULL: L alone
  float* lse;
  int* status;
  View vq, vk, vv;
  int n_q, n_k, d, d_v, window, sinks;
  int first, count;    // keys that any query sees: 0 .. sinks - 1, then first .. first + count - sinks - 1
  float sl2;           // scale * log2(e)
};

constexpr int TK_LANES = 8, TK_GROUPS = 32 / TK_LANES, TK_BATCH = 4;

template <class T>
struct Lane {   // 16 bytes of a row
  static constexpr int V = 16 / sizeof(T);
  static __device__ __forceinline__ void unpack(const uint4& w, float2* x) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    if constexpr (sizeof(T) == 4) {
      x[0] = f2(u[0], u[1]);
      x[1] = f2(u[2], u[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) x[i] = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        else x[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
      }
    }
  }
};

// A load that stays where it is written: the compiler would move those of a batch to their uses, one behind the other.
__device__ __forceinline__ uint4 load16(const void* from) {
  uint4 w;
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "l"(from) : "memory");
  return w;
}

// Puts the results of two sets of keys on a common maximum: (m, l, a) += (m2, l2, a2).
template <int H>
__device__ __forceinline__ void merge(float& m, float& l, float2 (&a)[H], float m2, float l2, const float2 (&a2)[H]) {
  const float top = fmaxf(m, m2);
  // (no maximum but a sum: NaN is kept)
  const float w1 = m == -INFINITY ? 1.f : ex2(m - top), w2 = m2 == -INFINITY ? 1.f : ex2(m2 - top);
  // a side without a sum has nothing to add: its weight may be anything
  const bool none1 = l == 0.f, none2 = l2 == 0.f;
  l = (none1 ? 0.f : l * w1) + (none2 ? 0.f : l2 * w2);
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const float2 x = none1 ? make_float2(0.f, 0.f) : make_float2(a[h].x * w1, a[h].y * w1);
    const float2 y = none2 ? make_float2(0.f, 0.f) : make_float2(a2[h].x * w2, a2[h].y * w2);
    a[h] = __fadd2_rn(x, y);
  }
  m = top;
}

// P pieces of 16 bytes a lane (piece i of lane j is the row's piece 8 i + j), R queries
template <class T, int P, int R, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, WARPS > 4 ? 1 : (R > 1 ? 3 : 4)) token_kernel(const __grid_constant__ TkParams p, int parts) {
  constexpr int V = Lane<T>::V, H = P * V / 2, kCols = TK_LANES * P * V;
  constexpr int kPitch = kCols + 4;   // floats of a staged row: O, maximum, sum
  __shared__ __align__(16) float staged[WARPS][R][kPitch];
  pdl_wait();
  if (threadIdx.x == 0) {
    pdl_launch_dependents();
    if (blockIdx.x == 0 && p.status) *p.status = 0;   // every call starts clean
  }
  const int head = blockIdx.x / parts, part = blockIdx.x - head * parts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / TK_LANES, at = (lane % TK_LANES) * V;
  const int hb = head / p.vk.heads, hh = head - hb * p.vk.heads;
  auto base = [&](const void* x, const View& v) { return static_cast<const T*>(x) + hb * v.batch + hh * v.head + at; };
  const T *q = base(p.q, p.vq), *k = base(p.k, p.vk), *v = base(p.v, p.vv);
  auto column = [&](int i) { return at + i * TK_LANES * V; };   // of piece i
  const int off = p.n_k - p.n_q;

  float2 qs[R][H], acc[R][H];
  float m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      if (column(i) < p.d && r < p.n_q) w = *reinterpret_cast<const uint4*>(q + r * p.vq.row + i * TK_LANES * V);
      Lane<T>::unpack(w, &qs[r][i * V / 2]);
    }
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int h = 0; h < H; ++h) acc[r][h] = make_float2(0.f, 0.f);
  }

  // this group's keys: every streams-th one of the part's, counted over first keys and window
  constexpr int kStreams = WARPS * TK_GROUPS, kRound = kStreams * TK_BATCH;
  const int rounds = (p.count + kRound - 1) / kRound;   // shared out whole
  const int begin = static_cast<int>(static_cast<long long>(rounds) * part / parts) * kRound;
  const int end = min(p.count, static_cast<int>(static_cast<long long>(rounds) * (part + 1) / parts) * kRound);
  // (the same number of rounds for all groups: the shuffles are the warp's)
  for (int x0 = begin; x0 < end; x0 += kRound) {
    uint4 kw[TK_BATCH][P], vw[TK_BATCH][P];
    int key[TK_BATCH];
#pragma unroll
    for (int u = 0; u < TK_BATCH; ++u) {
      const int x = x0 + (u * WARPS + warp) * TK_GROUPS + group;
      key[u] = x >= end ? -1 : (x < p.sinks ? x : p.first + x - p.sinks);
      const T* from = k + (key[u] < 0 ? 0 : key[u]) * p.vk.row;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        kw[u][i] = make_uint4(0u, 0u, 0u, 0u);
        if (key[u] >= 0 && column(i) < p.d) kw[u][i] = load16(from + i * TK_LANES * V);
      }
    }
#pragma unroll
    for (int u = 0; u < TK_BATCH; ++u) {
      const T* from = v + (key[u] < 0 ? 0 : key[u]) * p.vv.row;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        vw[u][i] = make_uint4(0u, 0u, 0u, 0u);
        if (key[u] >= 0 && column(i) < p.d_v && p.o) vw[u][i] = load16(from + i * TK_LANES * V);
      }
    }
    float s[R][TK_BATCH];
#pragma unroll
    for (int u = 0; u < TK_BATCH; ++u) {
      float2 ks[H];
#pragma unroll
      for (int i = 0; i < P; ++i) Lane<T>::unpack(kw[u][i], &ks[i * V / 2]);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float2 dot = __fmul2_rn(qs[r][0], ks[0]);
#pragma unroll
        for (int h = 1; h < H; ++h) dot = __ffma2_rn(qs[r][h], ks[h], dot);
        s[r][u] = dot.x + dot.y;
      }
    }
#pragma unroll
    for (int o = TK_LANES / 2; o > 0; o >>= 1)
#pragma unroll
      for (int u = 0; u < TK_BATCH; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][u] += __shfl_xor_sync(0xffffffffu, s[r][u], o);
    uint32_t hidden[R];   // bit u: key u of the batch, for a query that another shares it with
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = m[r];
      hidden[r] = 0u;
#pragma unroll
      for (int u = 0; u < TK_BATCH; ++u) {
        bool seen = key[u] >= 0;   // by a single query: every key of the list
        if (R > 1) seen = seen && r < p.n_q && pair_visible(r, key[u], off, 1, p.window, p.sinks);
        s[r][u] = seen ? s[r][u] * p.sl2 : -INFINITY;
        if (R > 1 && !seen) hidden[r] |= 1u << u;
        top = fmaxf(top, s[r][u]);
      }
      const float from = top == -INFINITY ? 0.f : top;   // no maximum yet: 0 for hidden keys, NaN for NaN scores
      const float alpha = m[r] == -INFINITY ? 1.f : ex2(m[r] - from);
      m[r] = top;
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < TK_BATCH; ++u) {
        s[r][u] = ex2(s[r][u] - from);
        sum += s[r][u];
      }
      l[r] = fmaf(l[r], alpha, sum);
#pragma unroll
      for (int h = 0; h < H; ++h) acc[r][h] = __fmul2_rn(acc[r][h], make_float2(alpha, alpha));
    }
#pragma unroll
    for (int u = 0; u < TK_BATCH; ++u) {
      float2 vs[H];
#pragma unroll
      for (int i = 0; i < P; ++i) Lane<T>::unpack(vw[u][i], &vs[i * V / 2]);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          // a hidden key's value may be anything
          const float2 x = R > 1 && (hidden[r] >> u & 1u) ? make_float2(0.f, 0.f) : vs[h];
          acc[r][h] = __ffma2_rn(make_float2(s[r][u], s[r][u]), x, acc[r][h]);
        }
    }
  }

  // groups of the warp, then warps, then the CTAs of the cluster
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int o = TK_LANES; o < 32; o <<= 1) {
      float2 a2[H];
      const float m2 = __shfl_xor_sync(0xffffffffu, m[r], o), l2 = __shfl_xor_sync(0xffffffffu, l[r], o);
#pragma unroll
      for (int h = 0; h < H; ++h) a2[h] = make_float2(__shfl_xor_sync(0xffffffffu, acc[r][h].x, o), __shfl_xor_sync(0xffffffffu, acc[r][h].y, o));
      // both sides of a pair add up in the same order
      if (lane & o) {
        float mm = m2, ll = l2;
        merge<H>(mm, ll, a2, m[r], l[r], acc[r]);
        m[r] = mm;
        l[r] = ll;
#pragma unroll
        for (int h = 0; h < H; ++h) acc[r][h] = a2[h];
      } else {
        merge<H>(m[r], l[r], acc[r], m2, l2, a2);
      }
    }
    if (group == 0) {
#pragma unroll
      for (int i = 0; i < P; ++i)
#pragma unroll
        for (int h = 0; h < V / 2; ++h) *reinterpret_cast<float2*>(&staged[warp][r][column(i) + 2 * h]) = acc[r][i * V / 2 + h];
      if (at == 0) {
        staged[warp][r][kCols] = m[r];
        staged[warp][r][kCols + 1] = l[r];
      }
    }
  }
  __syncthreads();
  // A warp a query, a lane the columns 2 lane, 2 lane + 64, ...  What is added up is read before the first sum.
  constexpr int kMine = (kCols + 63) / 64;   // pairs of columns of a lane
  float2 a[kMine];
  float mt, lt;
  auto add_up = [&](auto most, int count, auto&& load) {   // load(i, at): element `at` of the i-th result
    constexpr int kMost = decltype(most)::value;
    float2 all[kMost][kMine];
    float ms[kMost], ls[kMost];
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      ms[i] = -INFINITY;
      ls[i] = 0.f;
#pragma unroll
      for (int c = 0; c < kMine; ++c) {
        const int col = 2 * lane + 64 * c;
        all[i][c] = i < count && col < kCols ? make_float2(load(i, col), load(i, col + 1)) : make_float2(0.f, 0.f);
      }
      if (i < count) {
        ms[i] = load(i, kCols);
        ls[i] = load(i, kCols + 1);
      }
    }
    mt = ms[0];
    lt = ls[0];
#pragma unroll
    for (int c = 0; c < kMine; ++c) a[c] = all[0][c];
#pragma unroll
    for (int i = 1; i < kMost; ++i)
      if (i < count) merge<kMine>(mt, lt, a, ms[i], ls[i], all[i]);
  };
  if (warp < R) {
    add_up(std::integral_constant<int, WARPS>{}, WARPS, [&](int i, int c) { return staged[i][warp][c]; });
    __syncwarp();
    if (parts > 1) {   // this CTA's result, where its first warp's was
#pragma unroll
      for (int c = 0; c < kMine; ++c)
        if (2 * lane + 64 * c < kCols) *reinterpret_cast<float2*>(&staged[0][warp][2 * lane + 64 * c]) = a[c];
      if (lane == 0) {
        staged[0][warp][kCols] = mt;
        staged[0][warp][kCols + 1] = lt;
      }
    }
  }
  if (parts > 1) cluster_sync();
  if (warp < p.n_q && warp < R && warp % parts == part) {
    if (parts > 1) {
      uint32_t there[kMaxParts];
#pragma unroll
      for (int c = 0; c < kMaxParts; ++c) there[c] = cluster_map(smem_u32(&staged[0][warp][0]), c < parts ? c : 0);
      add_up(std::integral_constant<int, kMaxParts>{}, parts, [&](int i, int c) { return cluster_ld(there[i] + 4 * c); });
    }
    const size_t row = static_cast<size_t>(head) * p.n_q + warp;
    if (lane == 0) p.lse[row] = lt == 0.f ? -INFINITY : (mt + log2f(lt)) * 0.6931471805599453f;
    if (p.o) {
      const float inv = lt == 0.f ? 0.f : 1.f / lt;
      T* o = static_cast<T*>(p.o) + row * p.d_v;
#pragma unroll
      for (int c = 0; c < kMine; ++c) {
        const int col = 2 * lane + 64 * c;
        if (col < p.d_v) {   // an even number of columns
          o[col] = static_cast<T>(a[c].x * inv);
          o[col + 1] = static_cast<T>(a[c].y * inv);
        }
      }
    }
  }
  if (parts > 1) cluster_sync();   // the others are done with this CTA's shared memory
}

template <class T>
int token_launch(const TkParams& p, int heads, cudaStream_t s) {
  const int pieces = ((p.d > p.d_v ? p.d : p.d_v) * static_cast<int>(sizeof(T)) + 15) / 16;
  // Up to five rounds of 64 keys a CTA of 4 warps (128 heads W = 1024: 15.6 us; with four 21.8, with six 16.3; 16 heads 6.4, 5.7 and 6.8: at other
  // lengths the three have not been compared).  What 8 such CTAs would take long for, CTAs of 16 warps share.  64 heads of 500, 1000, 2000, 4000,
  // 8000 and 16000 keys, bf16: 10, 11, 16, 27, 45 and 106 us (1.7, 2.9, 4.1, 4.9, 5.8 and 5.0 TB/s).
  constexpr int kRound = 4 * TK_GROUPS * TK_BATCH;
  int parts = (p.count + 5 * kRound - 1) / (5 * kRound);
  parts = parts > kMaxParts ? kMaxParts : parts;
  auto go = [&](auto each, auto rows) -> int {
    constexpr int P = decltype(each)::value, R = decltype(rows)::value;
    const unsigned grid = static_cast<unsigned>(heads * parts);
    if (p.count <= 8192) FHOB_CUDA_OK(launch_pdl(token_kernel<T, P, R, 4>, grid, 128, 0, parts, s, p, parts));
    else FHOB_CUDA_OK(launch_pdl(token_kernel<T, P, R, 16>, grid, 512, 0, parts, s, p, parts));
    return FHOB_OK;
  };
  auto rows = [&](auto each) -> int {
    return p.n_q == 1 ? go(each, std::integral_constant<int, 1>{}) : go(each, std::integral_constant<int, 2>{});
  };
  if (pieces <= TK_LANES) return rows(std::integral_constant<int, 1>{});
  if constexpr (sizeof(T) == 4)
    if (pieces > 2 * TK_LANES) return rows(std::integral_constant<int, 4>{});
  return rows(std::integral_constant<int, 2>{});
}

}  // namespace

// Rows of whole 16-byte pieces at 16-byte addresses and strides.  (Calls without first keys keep the kernels they had.)
bool token_supported(const Problem& p, const void* o_out) {
  const int es = p.dtype == FHOB_F32 ? 4 : 2, d_v = head_dim_v(p);
  const uintptr_t all = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
                        static_cast<uintptr_t>(p.d * es) | static_cast<uintptr_t>(d_v * es);
  return p.sinks > 0 && p.n_q <= 2 && (all & 15u) == 0 && (reinterpret_cast<uintptr_t>(o_out) & 3u) == 0 && p.d <= 128 && d_v <= 128 &&
         static_cast<long long>(p.bh) * kMaxParts <= 0x7fffffffLL;
}

int token_forward(const Problem& p, void* o_out, float* lse_out, int* status, cudaStream_t s) {
  TkParams t;
  const int d_v = head_dim_v(p);
  t.q = p.q; t.k = p.k; t.v = p.v;
  t.o = o_out;
  t.lse = lse_out;
  t.status = status;
  t.vq = tensor_view(p, kTenQ, p.n_q, p.d);
  t.vk = tensor_view(p, kTenK, p.n_k, p.d);
  t.vv = tensor_view(p, kTenV, p.n_k, d_v);
  t.n_q = p.n_q; t.n_k = p.n_k; t.d = p.d; t.d_v = d_v; t.window = p.window; t.sinks = p.sinks;
  // the first query's window starts earliest; query i sees up to key i + n_k - n_q
  const int first = p.n_k - p.n_q - p.window + 1;
  t.first = first > p.sinks ? first : p.sinks;
  t.count = p.sinks + p.n_k - t.first;
  t.sl2 = p.scale * kLog2e;
  if (p.dtype == FHOB_F32) return token_launch<float>(t, p.bh, s);
  return p.dtype == FHOB_F16 ? token_launch<__half>(t, p.bh, s) : token_launch<__nv_bfloat16>(t, p.bh, s);
}

}  // namespace fhob
