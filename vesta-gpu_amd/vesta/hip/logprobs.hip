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
// The k most likely: of 64 disjoint groups of threads, the kth largest of their
// maxima is a bound that k elements reach. The few threads whose maximum does
// look at their elements again and list those that reach it; an element's rank
// is the number of listed ones before it. Elements are compared as a key of their
// value's order and, in the same word, their id's from the lowest.
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

// An element's key, above 0; a value back from it.
__device__ __forceinline__ lp_key lp_key_of(float v, int id) {
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.0f);       // (-0 is 0)
  const unsigned o = v != v ? 0xffffffffu : b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
  return (lp_key)o << 32 | (unsigned)~id;
}
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
__device__ __forceinline__ void lp_add(LpSums& a, const float* v) {
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
}

// A thread's elements of x[0 .. n): up to the first 16-byte boundary and behind
// the last whole load one each, between them every NT-th load of 16 bytes. `see`
// gets U loads' elements, the first's id (a load's first is NT loads after the
// one's before) and how many of them there are: the others are -inf.
template <int NT, int U, typename F>
__device__ __forceinline__ void lp_visit(const lp_t* __restrict__ x, int n, F see) {
  const int tid = threadIdx.x;
  const int head = min(n, (int)((16 - ((size_t)x & 15)) & 15) / (int)sizeof(lp_t));
  const int loads = (n - head) / LP_VEC, tail = head + loads * LP_VEC;
  const vh_u32x4* body = (const vh_u32x4*)(x + head);
  vh_u32x4 w[U];
  auto get = [&](int i) {
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = body[min(i + u * NT, loads - 1)];
  };
  if (tid < loads) get(tid);
  for (int i = tid; i < loads; i += U * NT) {
    float v[U * LP_VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      lp_unpack(w[u], v + u * LP_VEC);
      if (i + u * NT >= loads) {
#pragma unroll
        for (int j = 0; j < LP_VEC; ++j) v[u * LP_VEC + j] = -INFINITY;
      }
    }
    if (i + U * NT < loads) get(i + U * NT);
    see(v, head + i * LP_VEC, min(U, (loads - i + NT - 1) / NT) * LP_VEC);
  }
  const int rest = head + n - tail;                                // fewer than 16
  if (tid < rest) {
    const int id = tid < head ? tid : tail + tid - head;
    float v[U * LP_VEC];
    v[0] = lp_f(x[id]);
#pragma unroll
    for (int j = 1; j < U * LP_VEC; ++j) v[j] = -INFINITY;
    see(v, id, 1);
  }
}

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

// A block makes one of `parts` parts of a row, of `each` elements: its results,
// or with several parts its sums and most likely, in `ws`, for lp_join.
template <int NT>
__device__ __forceinline__ void lp_rows_body(const lp_t* __restrict__ X, long pitch, int V, const int* __restrict__ given,
                                             int wide, int C, int k, int parts, int each, float* __restrict__ out_given,
                                             float* __restrict__ out_entropy, float* __restrict__ out_top,
                                             int* __restrict__ out_ids, lp_key* __restrict__ ws) {
  constexpr int NW = NT / 64, U = 4;
  __shared__ LpSums sums[NW];
  __shared__ float groups[LP_TOP];
  __shared__ float bound;
  __shared__ int listed;
  __shared__ __attribute__((aligned(16))) lp_key list[LP_LIST];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x % parts), first = part * each, n = min(each, V - first);
  const lp_t* x = X + row * pitch;
  LpSums a = {-INFINITY, 0.0f, 0.0f};
  lp_visit<NT, U>(x + first, n, [&](const float* v, int, int) { lp_add<U * LP_VEC>(a, v); });
  const float own = a.m;                                           // the thread's largest
  lp_move(a, wave_red_max(a.m));
  a.s = wave_red_sum(a.s);
  a.t = wave_red_sum(a.t);
  if (lane == 0) sums[wave] = a;
  if (k) {
    const float g = group_red_max(own, NT / LP_TOP);
    if (tid % (NT / LP_TOP) == 0) groups[tid / (NT / LP_TOP)] = g;
    if (tid == 0) listed = 0;
  }
  vh_lds_sync();
  a = sums[0];
  float m = a.m;
#pragma unroll
  for (int w = 1; w < NW; ++w) m = fmaxf(m, sums[w].m);
  lp_move(a, m);
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    LpSums b = sums[w];
    lp_move(b, m);
    a.s += b.s;
    a.t += b.t;
  }
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
  if (wave == 0) {
    const float g = groups[lane];
    int rank = 0;
#pragma unroll
    for (int j = 0; j < LP_TOP; j += 4) {
      const vh_f32x4 o = *(const vh_f32x4*)(groups + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) rank += o[e] > g || (o[e] == g && j + e < lane) ? 1 : 0;
    }
    if (rank == k - 1) bound = g;
  }
  vh_lds_sync();
  // -inf as a bound: fewer groups than k have anything else, and what else there is is listed
  const float least = bound == -INFINITY ? -3.402823466e38f : bound;
  const bool odd = a.s != a.s;                                     // a NaN or +inf: found one by one
  if (!odd && own >= least) {
    lp_visit<NT, U>(x + first, n, [&](const float* v, int id, int) {
#pragma unroll
      for (int j = 0; j < U * LP_VEC; ++j)
        if (v[j] >= least) {
          const int at = atomicAdd(&listed, 1);
          if (at < LP_LIST) list[at] = lp_key_of(v[j], first + id + j / LP_VEC * (NT * LP_VEC) + j % LP_VEC);
        }
    });
  }
  vh_lds_sync();
  const int count = listed;
  if (!odd && count <= LP_LIST) {
    for (int i = tid; i < count; i += NT) {
      const lp_key key = list[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += list[j] > key ? 1 : 0;
      if (rank < k) found(rank, key);
    }
    // The rest are -inf, by their ids: of the lowest count + k ids k are at least, if the part has as many.
    if (wave == 0) {
      int at = count;
      for (int i = 0; at < k && i < n; i += 64) {
        const bool none = i + lane < n && lp_f(x[first + i + lane]) == -INFINITY;
        const lp_key all = __ballot(none);
        const int rank = at + __builtin_popcountl(all & (((lp_key)1 << lane) - 1));
        if (none && rank < k) found(rank, lp_key_of(-INFINITY, first + i + lane));
        at += __builtin_popcountl(all);
      }
      for (int i = at + lane; i < k; i += 64) found(i, 0);         // fewer than k elements in the part
    }
    return;
  }
  // More reach the bound than are listed (many ties), or there are NaNs: the
  // largest key below the last, k times.
  __shared__ lp_key best[NW];
  lp_key last = ~(lp_key)0;
  for (int rank = 0; rank < k; ++rank) {
    lp_key top = 0;
    lp_visit<NT, U>(x + first, n, [&](const float* v, int id, int have) {
#pragma unroll
      for (int j = 0; j < U * LP_VEC; ++j) {
        const lp_key key = j < have ? lp_key_of(v[j], first + id + j / LP_VEC * (NT * LP_VEC) + j % LP_VEC) : 0;
        if (key < last && key > top) top = key;
      }
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const lp_key other = (lp_key)__shfl_xor((long)top, o, 64);
      top = other > top ? other : top;
    }
    vh_lds_sync();
    if (lane == 0) best[wave] = top;
    vh_lds_sync();
    last = best[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) last = best[w] > last ? best[w] : last;
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
LP_ROWS(lp_rows256, 256)
LP_ROWS(lp_rows512, 512)
LP_ROWS(lp_rows1024, 1024)

// The parts of a row (64 at most) put together, a block a row.
extern "C" __global__ __launch_bounds__(256) void lp_join(const lp_t* __restrict__ X, long pitch, int V,
                                                          const int* __restrict__ given, int wide, int C, int k, int parts,
                                                          float* __restrict__ out_given, float* __restrict__ out_entropy,
                                                          float* __restrict__ out_top, int* __restrict__ out_ids,
                                                          const lp_key* __restrict__ ws) {
  __shared__ lp_key list[64 * LP_TOP];
  const int tid = threadIdx.x, lane = tid & 63;
  const long row = blockIdx.x;
  const lp_key* from = ws + row * parts * (2 + k);
  for (int i = tid; i < parts * k; i += 256) list[i] = from[i / k * (2 + k) + 2 + i % k];
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
  for (int c = tid; c < C; c += 256) lp_given(r, V, given, wide, C, row, c, out_given);
  if (tid == 0) out_entropy[row] = a.s == 0.0f ? 0.0f : r.log_s - a.t / a.s;
  vh_lds_sync();
  for (int i = tid; i < parts * k; i += 256) {
    const lp_key key = list[i];
    if (key == 0) continue;
    int rank = i % k;                                              // its own part's are in order, and so are the others'
    for (int p = 0; p < parts && rank < k; ++p) {
      if (p == i / k) continue;
      int lo = 0, hi = k;                                          // larger ones: lo at least, fewer than hi + 1
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list[p * k + mid] > key) lo = mid + 1; else hi = mid;
      }
      rank += lo;
    }
    if (rank < k) {
      out_top[row * k + rank] = lp_prob(r, lp_value(key));
      out_ids[row * k + rank] = lp_id(key);
    }
  }
}
