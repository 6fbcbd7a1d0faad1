// Log probabilities of given tokens, entropies and the most likely tokens of
// rows of logits, for gfx950. Appended to the prelude (hip/prelude.h) and
// compiled at run time by hipRTC, once per type of the logits, LP_KIND:
//   0  fp32       1  fp16       2  bf16
//
// Of a row x: m = max x, S = sum e^(x - m), T = sum e^(x - m) (x - m). Then token
// i's log probability is (x_i - m) - log S and the entropy log S - T / S. Each
// thread keeps these of what it has seen, against its own maximum, so that a row
// is read once; they are brought to a common maximum and added at the end. Sums
// are fp32, of a thread's elements in order, then over lanes and waves in order.
//
// The k most likely: of 64 disjoint groups of threads (a lane of each wave), the
// kth largest of their maxima is a bound that k elements reach. The few threads whose maximum does
// look at their elements again and list those that reach it; an element's rank
// is the number of listed ones before it. Elements are compared as a key of their
// value's order and, in the same word, their id's from the lowest.
//
// What bounds it: many rows, memory (8192 rows of 50257 in fp32 267 us, 6.2 TB/s; with
// five alternatives 279); few, a CU's share of the bandwidth (200 rows of 128001 in
// bf16, a row a CU: 13.4 us, then 7 for 20 alternatives), the chain from launch to
// loads to reductions (8 rows of 50257 7.0 us, with five 9.0), half of it fetching
// instructions that run once.
//
// A NaN or +inf in a row makes its results NaN (its order: NaN is the largest); a
// row of -inf alone allows nothing: all its log probabilities are -inf, its
// entropy 0.

#define LP_F32 0
#define LP_F16 1
#define LP_BF16 2
#if LP_KIND == LP_F32
typedef float lp_t;
#else
typedef unsigned short lp_t;
#endif
#define LP_VEC (16 / (int)sizeof(lp_t))    // elements of a 16-byte load
#define LP_LIST 1024                       // elements listed at most; more are found one by one
#define LP_TOP 64                          // k at most, and the groups
#define LP_LOG2E 1.44269504088896340736f

typedef unsigned long lp_key;

__device__ __forceinline__ float lp_f(lp_t v) {
#if LP_KIND == LP_F32
  return v;
#elif LP_KIND == LP_F16
  return h2f(v);
#else
  return __builtin_bit_cast(float, (unsigned)v << 16);
#endif
}
__device__ __forceinline__ void lp_unpack(vh_u32x4 w, float* v) {
#if LP_KIND == LP_F32
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned u = w[j];               // (a bit_cast of a vector's element takes its first)
    v[j] = __builtin_bit_cast(float, u);
  }
#else
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = lp_f((unsigned short)(w[j] & 0xffffu));
    v[2 * j + 1] = lp_f((unsigned short)(w[j] >> 16));
  }
#endif
}

// An element's key, above 0 and below ~0 (a NaN of id 0 has a bit to spare); a value back from it.
__device__ __forceinline__ unsigned lp_word(float v) {
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.0f);       // (-0 is 0)
  return v != v ? 0xfffffffeu : b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ lp_key lp_key_of(float v, int id) { return (lp_key)lp_word(v) << 32 | (unsigned)~id; }
__device__ __forceinline__ float lp_value(lp_key k) {
  const unsigned o = (unsigned)(k >> 32);
  return __builtin_bit_cast(float, o ^ (o >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int lp_id(lp_key k) { return (int)~(unsigned)k; }

// What is known of some elements.
struct LpSums {
  float m, s, t;
};
__device__ __forceinline__ float lp_ref(float m) { return m == -INFINITY ? 0.0f : m; }
// ... against a maximum of m or more. x - m is cut off where e^(x - m) has long
// been 0, so that their product is (-inf, or the type's lowest value, in a row).
__device__ __forceinline__ void lp_move(LpSums& a, float m) {
  const float ref = lp_ref(m), d = a.m - ref, c = __builtin_amdgcn_exp2f(d * LP_LOG2E);
  a.t = c * fmaf(fmaxf(d, -1e4f), a.s, a.t);
  a.s *= c;
  a.m = m;
}
template <int N>
__device__ __forceinline__ float lp_add(LpSums& a, const float* v) {      // (the elements' largest)
  float m = v[0];
#pragma unroll
  for (int j = 1; j < N; ++j) m = fmaxf(m, v[j]);
  if (__any(m > a.m)) lp_move(a, fmaxf(a.m, m));
  const float ref = lp_ref(a.m);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float d = v[j] - ref, e = __builtin_amdgcn_exp2f(d * LP_LOG2E);
    a.s += e;
    a.t = fmaf(e, fmaxf(d, -1e4f), a.t);
  }
  return m;
}
// The waves' together.
template <int NW>
__device__ __forceinline__ LpSums lp_all(const LpSums* sums) {
  const int lane = threadIdx.x & 63;
  LpSums a = {-INFINITY, 0.0f, 0.0f};
  if (lane < NW) a = sums[lane];
  lp_move(a, wave_red_max(a.m));
  a.s = wave_red_sum(a.s);
  a.t = wave_red_sum(a.t);
  return a;
}

// A thread's elements of x[0 .. n), in chunks of U loads of 16 bytes, NT loads
// apart; one more chunk is an element before the first 16-byte boundary or behind
// the last whole load.
template <int NT, int U>
struct LpSpan {
  static constexpr int N = U * LP_VEC;
  const lp_t* x;
  int n, head, loads;
  __device__ __forceinline__ LpSpan(const lp_t* from, int count) : x(from), n(count) {
    head = min(n, (int)((16 - ((size_t)x & 15)) & 15) / (int)sizeof(lp_t));
    loads = (n - head) / LP_VEC;
  }
  __device__ __forceinline__ void get(int i, vh_u32x4* w) const {  // the chunk that begins with load i
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = ((const vh_u32x4*)(x + head))[min(i + u * NT, loads - 1)];
  }
  // How many elements a chunk has; the others, behind them, are made -inf.
  __device__ __forceinline__ int open(int i, const vh_u32x4* w, float* v) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      lp_unpack(w[u], v + u * LP_VEC);
      if (i + u * NT >= loads) {
#pragma unroll
        for (int j = 0; j < LP_VEC; ++j) v[u * LP_VEC + j] = -INFINITY;
      }
    }
    return min(U, (loads - i + NT - 1) / NT) * LP_VEC;
  }
  __device__ __forceinline__ int id(int i, int j) const { return head + (i + j / LP_VEC * NT) * LP_VEC + j % LP_VEC; }
  // The element beside the loads: its id, or -1 for none.
  __device__ __forceinline__ int beside() const {
    const int t = threadIdx.x, behind = head + loads * LP_VEC + t - head;
    return t < head ? t : behind < n ? behind : -1;
  }
  __device__ __forceinline__ void one(int id, float* v) const {
    v[0] = lp_f(x[id]);
#pragma unroll
    for (int j = 1; j < N; ++j) v[j] = -INFINITY;
  }
  // All chunks: see(first load (-1: the element beside), elements, how many, the id of one). The next chunk's loads are
  // in flight while one is seen.
  template <typename F>
  __device__ __forceinline__ void visit(F see) const {
    vh_u32x4 w[U];
    float v[N];
    const int extra = beside();
    if ((int)threadIdx.x < loads) get(threadIdx.x, w);
    for (int i = threadIdx.x; i < loads; i += U * NT) {
      const int have = open(i, w, v);
      if (i + U * NT < loads) get(i + U * NT, w);
      see(i, v, have);
    }
    if (extra >= 0) {
      one(extra, v);
      see(-1, v, 1);
    }
  }
  __device__ __forceinline__ int id_of(int i, int j) const { return i < 0 ? beside() : id(i, j); }
};

// A row's results. `x` is the row.
struct LpRow {
  const lp_t* x;
  float ref, log_s;
};
__device__ __forceinline__ LpRow lp_row(const lp_t* x, const LpSums& a) {
  return LpRow{x, lp_ref(a.m), a.s == 0.0f ? 0.0f : logf(a.s)};    // (0: -inf - 0, where nothing is allowed)
}
__device__ __forceinline__ float lp_prob(const LpRow& r, float v) { return (v - r.ref) - r.log_s; }
__device__ __forceinline__ void lp_given(const LpRow& r, int V, const int* __restrict__ given, int wide, int C, long row,
                                         int c, float* __restrict__ out) {
  const long at = row * C + c;
  const long id = wide ? ((const long*)given)[at] : given[at];
  out[at] = id >= 0 && id < V ? lp_prob(r, lp_f(r.x[id])) : __builtin_nanf("");
}

// The code from here on runs once a block, and most of what it would take as
// straight lines is fetching them (64 comparisons as such 2500 cycles, 1400 the
// second time): short loops, few instructions.
//
// The kth largest of a wave's values, each lane with one, or a bound below it that
// few more reach: of 16 lanes' maxima each fourth for k up to 8, 32 up to 20.
__device__ __forceinline__ float lp_kth(float g, int k) {
  int lanes = 64;
  if (k <= 20) {
    lanes = 32;
    g = vh_pair32(g, op_max);
  }
  if (k <= 8) {
    lanes = 16;
    g = vh_pair16(g, op_max);
  }
  int above = 0;
#pragma nounroll
  for (int i = 0; i < lanes; i += 16)
#pragma unroll
    for (int j = 0; j < 16; ++j)
      above += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, g), i + j)) > g ? 1 : 0;
  return wave_red_min(above < k ? g : INFINITY);                   // the least of those that fewer than k are above
}
// A group's largest, of its waves'.
template <int NW>
__device__ __forceinline__ float lp_group(const float (*owns)[64], int lane) {
  float g = owns[0][lane];
#pragma unroll
  for (int w = 1; w < NW; ++w) g = fmaxf(g, owns[w][lane]);
  return g;
}
// -inf as a bound: fewer groups than k have anything else, and what else there is is listed.
__device__ __forceinline__ float lp_least(float bound) { return fmaxf(bound, -3.402823466e38f); }
// Those of each lane's N elements that reach a bound into the list, one of each lane
// at a time; the lanes in this branch take places together. (Values are read
// again: choosing a register takes more.) A full list's length goes on past
// LP_LIST, by little.
template <int N, typename R, typename F>
__device__ __forceinline__ void lp_list(const lp_t* __restrict__ x, R reaches, lp_key* list, int* listed, F id_of) {
  lp_key in = 0;                                                   // bit N - 1 - j: element j
#pragma unroll
  for (int j = 0; j < N; ++j) in = in + in + (reaches(j) ? 1 : 0);
#pragma nounroll
  while (in) {
    const int bit = 63 - __builtin_clzl(in), id = id_of(N - 1 - bit);
    in &= ~((lp_key)1 << bit);
    const lp_t value = x[id];
    const lp_key lanes = __ballot(1);
    const int before = __builtin_popcountl(lanes & (((lp_key)1 << (threadIdx.x & 63)) - 1));
    int at = 0;
    if (before == 0)
      at = __hip_atomic_fetch_add(listed, __builtin_popcountl(lanes), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    at = __builtin_amdgcn_readfirstlane(at) + before;
    if (at < LP_LIST) list[at] = lp_key_of(lp_f(value), id);
    else in = 0;
  }
}
// The listed ones' ranks, of which `found` gets those below k, 64 at a time. Of
// few the first wave counts the larger ones; of more each wave a share of them,
// in `ranks`, which is zeroed (2000 rows of 50257 in bf16, 64 of some 300 listed:
// 143 -> 130 us; of a few it would be a barrier more).
template <int NT, typename F>
__device__ __forceinline__ void lp_order(const lp_key* list, int* ranks, int count, int k, F found) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool alone = NT == 64 || count <= 16;
  const int waves = alone ? 1 : NT / 64;
  if (wave >= waves) return;
  for (int c = 0; c < count; c += 64) {
    const int i = min(c + lane, count - 1);
    const lp_key key = list[i];
    int rank = 0;
#pragma nounroll
    for (int j = wave; j < count; j += 4 * waves) {                // (reads past the last are its own again)
      lp_key o[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] = list[min(j + u * waves, count - 1)];
#pragma unroll
      for (int u = 0; u < 4; ++u) rank += j + u * waves < count && o[u] > key ? 1 : 0;
    }
    if (alone) {
      if (c + lane < count && rank < k) found(rank, key);
    } else if (c + lane < count && rank) {
      __hip_atomic_fetch_add(ranks + i, rank, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  }
  if (alone) return;
  vh_lds_sync();
  for (int i = threadIdx.x; i < count; i += NT)
    if (ranks[i] < k) found(ranks[i], list[i]);
}
// The places behind `count` listed elements, by one wave: the rest of x[0 .. n),
// whose ids begin at `first`, is -inf, and follows by its ids (of the lowest
// count + k ids k are at least, if there are as many); 0 where nothing does.
template <typename F>
__device__ __forceinline__ void lp_none(const lp_t* __restrict__ x, int n, int first, int count, int k, F found) {
  const int lane = threadIdx.x & 63;
  int at = count;
  for (int i = 0; at < k && i < n; i += 64) {
    const bool none = i + lane < n && lp_f(x[i + lane]) == -INFINITY;
    const lp_key all = __ballot(none);
    const int rank = at + __builtin_popcountl(all & (((lp_key)1 << lane) - 1));
    if (none && rank < k) found(rank, lp_key_of(-INFINITY, first + i + lane));
    at += __builtin_popcountl(all);
  }
  for (int i = at + lane; i < k; i += 64) found(i, 0);
}
// Where more reach the bound than are listed (a mask's finite value, a flat row), or
// there are NaNs: the same with keys in the place of values. No two are equal,
// and of equal values each group has its lowest id, so that the bound lies among the
// lowest ids. `chunks` hands out N of a thread's keys (0 for none) and their ids; the row
// is read twice more, where the largest key below the last, k times, reads it k times
// (2000 rows of 50257 in bf16, three allowed, 64 asked for 2890 -> 240 us, with a NaN 2750
// -> 187; 200 of 128001, 20: 354 -> 60, 314 -> 50). The largest alone is found in one
// reading (8192 flat rows of 50257 in fp32, by keys / one by one: 879 / 662; two of
// them 884 / 1186, of rows with a NaN 672 / 673).
// False where these are more than are listed too: single groups have most of the large ones.
template <int NT, int N, typename C, typename F>
__device__ __forceinline__ bool lp_by_keys(const lp_t* __restrict__ x, C chunks, lp_key* list, int* listed, int* ranks,
                                           int k, F found) {
  static_assert(NT <= LP_LIST, "a key a thread");
  const int tid = threadIdx.x, lane = tid & 63;
  lp_key top = 0;
  chunks([&](auto key, auto) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const lp_key o = key(j);
      top = o > top ? o : top;
    }
  });
  vh_lds_sync();                                                   // the list's length is read
  list[tid] = top;
  if (tid == 0) *listed = 0;
  vh_lds_sync();
  lp_key g = list[lane];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) g = list[64 * w + lane] > g ? list[64 * w + lane] : g;
  int above = 0;
#pragma nounroll
  for (int i = 0; i < 64; ++i) {
    const unsigned hi = __builtin_amdgcn_readlane((int)(g >> 32), i), lo = __builtin_amdgcn_readlane((int)g, i);
    above += ((lp_key)hi << 32 | lo) > g ? 1 : 0;
  }
  lp_key least = above < k ? g : ~(lp_key)0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const lp_key other = (lp_key)__shfl_xor((long)least, o, 64);
    least = other < least ? other : least;
  }
  least = least ? least : 1;                                       // (fewer groups than k have any)
  vh_lds_sync();                                                   // the groups are read
  chunks([&](auto key, auto id) { lp_list<N>(x, [&](int j) { return key(j) >= least; }, list, listed, id); });
  vh_lds_sync();
  const int count = *listed;
  if (count > LP_LIST) return false;
  lp_order<NT>(list, ranks, count, k, found);
  if (tid < 64)
    for (int i = count + lane; i < k; i += 64) found(i, 0);
  return true;
}
// The block's largest key.
template <int NW>
__device__ __forceinline__ lp_key lp_block_best(lp_key top, lp_key* best) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const lp_key other = (lp_key)__shfl_xor((long)top, o, 64);
    top = other > top ? other : top;
  }
  vh_lds_sync();
  if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = top;
  vh_lds_sync();
  top = best[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) top = best[w] > top ? best[w] : top;
  return top;
}

// A block makes one of `parts` parts of a row, of `each` elements: its results,
// or with several parts its sums and most likely, in `ws`, for lp_join.
template <int NT>
__device__ __forceinline__ void lp_rows_body(const lp_t* __restrict__ X, long pitch, int V, const int* __restrict__ given,
                                             int wide, int C, int k, int parts, int each, float* __restrict__ out_given,
                                             float* __restrict__ out_entropy, float* __restrict__ out_top,
                                             int* __restrict__ out_ids, lp_key* __restrict__ ws) {
  constexpr int NW = NT / 64, U = 4;
  typedef LpSpan<NT, U> Span;
  __shared__ LpSums sums[NW];
  __shared__ float owns[NW][64];
  __shared__ int listed, ranks[NW > 1 ? LP_LIST : 1];
  __shared__ float bound;
  __shared__ lp_key list[LP_LIST];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x % parts), first = part * each, n = min(each, V - first);
  const lp_t* x = X + row * pitch;
  const Span span(x + first, n);
  LpSums a = {-INFINITY, 0.0f, 0.0f};
  // Of the thread's chunks: which has its largest element, and the largest of the others.
  int chunk = -1;
  float other = -INFINITY;
  span.visit([&](int i, const float* v, int) {
    const float old = a.m, m = lp_add<Span::N>(a, v);
    other = fmaxf(other, fminf(m, old));
    chunk = m > old ? i : chunk;
  });
  const float own = a.m;
  lp_move(a, wave_red_max(a.m));
  a.s = wave_red_sum(a.s);
  a.t = wave_red_sum(a.t);
  if (lane == 0) sums[wave] = a;
  owns[wave][lane] = own;
  if (tid == 0) listed = 0;
  if (NW > 1 && k)
    for (int i = tid; i < LP_LIST; i += NT) ranks[i] = 0;
  vh_lds_sync();
  a = lp_all<NW>(sums);
  const LpRow r = lp_row(x, a);
  lp_key* mine = ws + (row * parts + part) * (2 + k);
  if (parts == 1) {
    for (int c = tid; c < C; c += NT) lp_given(r, V, given, wide, C, row, c, out_given);
    if (tid == 0) out_entropy[row] = a.s == 0.0f ? 0.0f : r.log_s - a.t / a.s;
  } else if (tid == 0) {
    mine[0] = (lp_key)__builtin_bit_cast(unsigned, a.m) << 32 | __builtin_bit_cast(unsigned, a.s);
    mine[1] = __builtin_bit_cast(unsigned, a.t);
  }
  if (k == 0) return;
  auto found = [&](int rank, lp_key key) {
    if (parts > 1) {
      mine[2 + rank] = key;
    } else {
      out_top[row * k + rank] = lp_prob(r, lp_value(key));
      out_ids[row * k + rank] = lp_id(key);
    }
  };
  float least;
  if (NW <= 4 || k <= 8) {                                         // little for a SIMD's waves: each by itself
    least = lp_least(lp_kth(lp_group<NW>(owns, lane), k));
  } else {
    if (wave == 0) {
      const float b = lp_kth(lp_group<NW>(owns, lane), k);
      if (lane == 0) bound = b;
    }
    vh_lds_sync();
    least = lp_least(bound);
  }
  const bool odd = a.s != a.s;                                     // a NaN or +inf: found one by one
  if (!odd && own >= least) {
    auto look = [&](int i, const float* v, int) {
      lp_list<Span::N>(x, [&](int j) { return v[j] >= least; }, list, &listed,
                       [&](int j) { return first + span.id_of(i, j); });
    };
    if (other >= least) {
      span.visit(look);
    } else {
      float v[Span::N];
      if (chunk < 0) {
        span.one(span.beside(), v);
      } else {
        vh_u32x4 w[U];
        span.get(chunk, w);
        span.open(chunk, w, v);
      }
      look(chunk, v, 0);
    }
  }
  vh_lds_sync();
  const int count = listed;
  if (!odd && count <= LP_LIST) {
    lp_order<NT>(list, ranks, count, k, found);
    if (wave == 0) lp_none(x + first, n, first, count, k, found);
    return;
  }
  auto chunks = [&](auto see) {
    span.visit([&](int i, const float* v, int have) {
      auto id = [&](int j) { return first + span.id_of(i, j); };
      see([&](int j) { return j < have ? lp_key_of(v[j], id(j)) : (lp_key)0; }, id);
    });
  };
  if (k > 1 && lp_by_keys<NT, Span::N>(x, chunks, list, &listed, ranks, k, found)) return;
  // the largest key below the last, k times
  __shared__ lp_key best[NW];
  lp_key last = ~(lp_key)0;
  for (int rank = 0; rank < k; ++rank) {
    lp_key top = 0;
    chunks([&](auto key, auto) {
#pragma unroll
      for (int j = 0; j < Span::N; ++j) {
        const lp_key o = key(j);
        if (o < last && o > top) top = o;
      }
    });
    last = lp_block_best<NW>(top, best);
    if (tid == 0) found(rank, last);
    if (last == 0) last = 1;                                       // none left: none after it either
  }
}
#define LP_ROWS(name, threads)                                                                                     \
  extern "C" __global__ __launch_bounds__(threads) void name(                                                      \
      const lp_t* __restrict__ X, long pitch, int V, const int* __restrict__ given, int wide, int C, int k, int parts, \
      int each, float* __restrict__ out_given, float* __restrict__ out_entropy, float* __restrict__ out_top,       \
      int* __restrict__ out_ids, lp_key* __restrict__ ws) {                                                        \
    lp_rows_body<threads>(X, pitch, V, given, wide, C, k, parts, each, out_given, out_entropy, out_top, out_ids, ws); \
  }
LP_ROWS(lp_rows64, 64)
LP_ROWS(lp_rows256, 256)
LP_ROWS(lp_rows512, 512)
LP_ROWS(lp_rows1024, 1024)

// A part of NT L loads of 16 bytes of a row, which stay in registers: nothing is
// looked at again. Loads are where they fall, at any alignment; the row's last
// one begins early enough to end with it, and the elements that it has in common
// with the one before count as -inf.
typedef unsigned lp_u4 __attribute__((ext_vector_type(4), aligned(sizeof(lp_t))));
template <int L>
__device__ __forceinline__ void lp_part_body(const lp_t* __restrict__ X, long pitch, int V, int k, int parts, int each,
                                             lp_key* __restrict__ ws) {
  constexpr int NT = 256, NW = NT / 64;
  __shared__ LpSums sums[NW];
  __shared__ float owns[NW][64];
  __shared__ int listed, ranks[LP_LIST];
  __shared__ lp_key list[LP_LIST];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x % parts), first = part * each, end = min(first + each, V);
  const lp_t* x = X + row * pitch;
  vh_u32x4 w[L];
#pragma unroll
  for (int l = 0; l < L; ++l) w[l] = *(const lp_u4*)(x + min(first + (l * NT + tid) * LP_VEC, V - LP_VEC));
  float v[L * LP_VEC];
#pragma unroll
  for (int l = 0; l < L; ++l) {
    lp_unpack(w[l], v + l * LP_VEC);
    const int e = first + (l * NT + tid) * LP_VEC, early = e < end ? e - (V - LP_VEC) : LP_VEC;     // elements not its own
    if (early > 0) {
#pragma unroll
      for (int j = 0; j < LP_VEC; ++j) v[l * LP_VEC + j] = j >= early ? v[l * LP_VEC + j] : -INFINITY;
    }
  }
  auto id_of = [&](int j) { return min(first + (j / LP_VEC * NT + tid) * LP_VEC, V - LP_VEC) + j % LP_VEC; };
  float own = v[0];
#pragma unroll
  for (int j = 1; j < L * LP_VEC; ++j) own = fmaxf(own, v[j]);
  own = fmaxf(own, -INFINITY);                                     // (a NaN where all are)
  owns[wave][lane] = own;
  if (tid == 0) listed = 0;
  if (k)
    for (int i = tid; i < LP_LIST; i += NT) ranks[i] = 0;
  vh_lds_sync();
  const float g = lp_group<NW>(owns, lane);
  LpSums a = {wave_red_max(g), 0.0f, 0.0f};
  if (k) {
    const float least = lp_least(lp_kth(g, k));                    // (each wave by itself)
    if (own >= least) lp_list<L * LP_VEC>(x, [&](int j) { return v[j] >= least; }, list, &listed, id_of);
  }
  const float ref = lp_ref(a.m);
#pragma unroll
  for (int j = 0; j < L * LP_VEC; ++j) {
    const float d = v[j] - ref, e = __builtin_amdgcn_exp2f(d * LP_LOG2E);
    a.s += e;
    a.t = fmaf(e, fmaxf(d, -1e4f), a.t);
  }
  a.s = wave_red_sum(a.s);
  a.t = wave_red_sum(a.t);
  if (lane == 0) sums[wave] = a;
  vh_lds_sync();
  a = lp_all<NW>(sums);
  lp_key* mine = ws + (row * parts + part) * (2 + k);
  if (tid == 0) {
    mine[0] = (lp_key)__builtin_bit_cast(unsigned, a.m) << 32 | __builtin_bit_cast(unsigned, a.s);
    mine[1] = __builtin_bit_cast(unsigned, a.t);
  }
  if (k == 0) return;
  const int count = listed;
  auto found = [&](int rank, lp_key key) { mine[2 + rank] = key; };
  if (a.s == a.s && count <= LP_LIST) {
    lp_order<NT>(list, ranks, count, k, found);
    if (wave == 0) lp_none(x + first, end - first, first, count, k, found);
    return;
  }
  auto chunks = [&](auto see) {
    see([&](int j) {
      const int e = first + (j / LP_VEC * NT + tid) * LP_VEC, early = e - (V - LP_VEC);
      return e < end && j % LP_VEC >= early ? lp_key_of(v[j], id_of(j)) : (lp_key)0;
    }, id_of);
  };
  if (k > 1 && lp_by_keys<NT, L * LP_VEC>(x, chunks, list, &listed, ranks, k, found)) return;
  __shared__ lp_key best[NW];
  lp_key last = ~(lp_key)0;
  for (int rank = 0; rank < k; ++rank) {
    lp_key top = 0;
    chunks([&](auto key, auto) {
#pragma unroll
      for (int j = 0; j < L * LP_VEC; ++j) {
        const lp_key o = key(j);
        if (o < last && o > top) top = o;
      }
    });
    last = lp_block_best<NW>(top, best);
    if (tid == 0) found(rank, last);
    if (last == 0) last = 1;                                       // none left: none after it either
  }
}
#define LP_PART(name, loads)                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void name(const lp_t* __restrict__ X, long pitch, int V, int k, int parts, \
                                                         int each, lp_key* __restrict__ ws) {                      \
    lp_part_body<loads>(X, pitch, V, k, parts, each, ws);                                                          \
  }
LP_PART(lp_part2, 2)
LP_PART(lp_part4, 4)
LP_PART(lp_part8, 8)

// The parts of a row (64 at most, of k listed elements each, MOST in all) put
// together by a wave, as a part is by its block.
template <int MOST>
__device__ __forceinline__ void lp_join_body(const lp_t* __restrict__ X, long pitch, int V, const int* __restrict__ given,
                                             int wide, int C, int k, int parts, float* __restrict__ out_given,
                                             float* __restrict__ out_entropy, float* __restrict__ out_top,
                                             int* __restrict__ out_ids, const lp_key* __restrict__ ws) {
  __shared__ lp_key list[MOST];
  const int lane = threadIdx.x, n = parts * k;
  const long row = blockIdx.x;
  const lp_key* from = ws + row * parts * (2 + k);
  auto entry = [&](int i) {
    const int p = i / k;
    return from[p * (2 + k) + 2 + i - p * k];
  };
  constexpr int E = 4;                                             // a lane's first entries
  lp_key own[E];
#pragma unroll
  for (int e = 0; e < E; ++e) own[e] = lane + 64 * e < n ? entry(lane + 64 * e) : 0;
  LpSums a = {-INFINITY, 0.0f, 0.0f};
  if (lane < parts) {
    const lp_key w = from[lane * (2 + k)];
    a.m = __builtin_bit_cast(float, (unsigned)(w >> 32));
    a.s = __builtin_bit_cast(float, (unsigned)w);
    a.t = __builtin_bit_cast(float, (unsigned)from[lane * (2 + k) + 1]);
  }
  lp_move(a, wave_red_max(a.m));
  a.s = wave_red_sum(a.s);
  a.t = wave_red_sum(a.t);
  const LpRow r = lp_row(X + row * pitch, a);
  for (int c = lane; c < C; c += 64) lp_given(r, V, given, wide, C, row, c, out_given);
  if (lane == 0) out_entropy[row] = a.s == 0.0f ? 0.0f : r.log_s - a.t / a.s;
  if (k == 0) return;
  // entries that reach the kth largest of the lanes' largest ones
  lp_key top = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) top = own[e] > top ? own[e] : top;
  for (int i = lane + 64 * E; i < n; i += 64) {
    const lp_key o = entry(i);
    top = o > top ? o : top;
  }
  const float g = top == 0 ? -INFINITY : lp_value(top);             // (a NaN counts as the largest)
  const unsigned least = lp_word(lp_kth(g != g ? INFINITY : g, k));
  int count = 0;
  auto pick = [&](lp_key key) {
    const bool in = key != 0 && (unsigned)(key >> 32) >= least;
    const lp_key all = __ballot(in);
    if (in) list[count + __builtin_popcountl(all & (((lp_key)1 << lane) - 1))] = key;
    count += __builtin_popcountl(all);
  };
#pragma unroll
  for (int e = 0; e < E; ++e) pick(own[e]);
  for (int i = 64 * E; i < n; i += 64) pick(i + lane < n ? entry(i + lane) : 0);
  vh_lds_sync();
  lp_order<64>(list, nullptr, count, k, [&](int rank, lp_key key) {
    out_top[row * k + rank] = lp_prob(r, lp_value(key));
    out_ids[row * k + rank] = lp_id(key);
  });
}
#define LP_JOIN(name, most)                                                                                        \
  extern "C" __global__ __launch_bounds__(64) void name(                                                           \
      const lp_t* __restrict__ X, long pitch, int V, const int* __restrict__ given, int wide, int C, int k, int parts, \
      float* __restrict__ out_given, float* __restrict__ out_entropy, float* __restrict__ out_top,                 \
      int* __restrict__ out_ids, const lp_key* __restrict__ ws) {                                                  \
    lp_join_body<most>(X, pitch, V, given, wide, C, k, parts, out_given, out_entropy, out_top, out_ids, ws);       \
  }
LP_JOIN(lp_join, 256)
LP_JOIN(lp_join_many, 64 * LP_TOP)
