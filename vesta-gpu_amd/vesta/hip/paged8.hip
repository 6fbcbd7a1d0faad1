// Rows into and out of a paged cache in 8 bits (hip/form8.h), after hip/paged.hip.
//
// A wave takes rows of one head, so that what it reads or stores of the pool lies
// together (a head's rows of a page do), the powers too: with rows of all heads,
// whose powers reach memory two or four bytes at a time, 12,900 rows of 8 heads of
// 128 took 22.8 us to append. Bound by memory: these rows 14.4 us (80 MB, 5.5 TB/s),
// 28,800 rows of 25 heads of 64 appended in 67 and read back in 73.6 us (332 MB, 4.5
// TB/s; in 54.5 where the memory-side cache holds the pool), of 8 heads of 128 in 46.5
// (33 from the cache); eight rows 3.6 us, a launch and the loads that wait for one another.

// A lane's neighbour in its two.
__device__ __forceinline__ float pg8_other(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
}

// 16 values as elements, and their block's byte: two lanes have a block.
__device__ __forceinline__ vh_u32x4 pg8_hold(const float* x, unsigned& s) {
  float mx = 0.0f;
  bool odd = false;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float a = __builtin_fabsf(x[j]);
    const bool fin = a < INFINITY;                                 // (false for a NaN)
    mx = fmaxf(mx, fin ? a : 0.0f);
    odd |= !fin;
  }
#if PG_FORM == 1
  mx = odd ? INFINITY : mx;                                        // the whole block's
#endif
  mx = fmaxf(mx, pg8_other(mx));
  s = (unsigned)min(max((int)((__builtin_bit_cast(unsigned, mx) + PG8_ROUND) >> 23) - PG8_BELOW, PG8_LOW), PG8_HIGH);
  vh_u32x4 w = {0u, 0u, 0u, 0u};
#if PG_FORM == 1
  const float f = __builtin_bit_cast(float, (260u - s) << 23);     // 2^(133 - s)
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int q = (int)fminf(fmaxf(__builtin_rintf(x[j] * f), -127.0f), 127.0f);
    w[j >> 2] |= ((unsigned)q & 255u) << 8 * (j & 3);
  }
  if (mx == INFINITY) s = PG8_NAN;
#else
  const float f = __builtin_bit_cast(float, (254u - s) << 23);     // 2^(127 - s)
  float y[16];
#pragma unroll
  for (int j = 0; j < 16; ++j)
    y[j] = __builtin_fabsf(x[j]) < INFINITY ? fminf(fmaxf(x[j] * f, -448.0f), 448.0f) : __builtin_nanf("");
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j], y[4 * j + 1], 0, false);
    w[j] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j + 2], y[4 * j + 3], v, true);
  }
#endif
  return w;
}

// 16 values of a tensor's row as they are, and as fp32.
template <typename T>
struct Pg8Row {
  vh_u32x4 w[sizeof(T)];
  __device__ __forceinline__ void get(const T* p) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T); ++j) w[j] = ld16((const char*)p + 16 * j);
  }
  __device__ __forceinline__ void open(float* x) const {
#pragma unroll
    for (int j = 0; j < 4 * (int)sizeof(T); ++j) {
      const unsigned u = w[j / 4][j % 4];
      if constexpr (sizeof(T) == 4) {
        x[j] = __builtin_bit_cast(float, u);
      } else {
        x[2 * j] = pg_to_f((unsigned short)(u & 0xffffu));
        x[2 * j + 1] = pg_to_f((unsigned short)(u >> 16));
      }
    }
  }
};

// A lane's row i of the call's, its head's piece of PER values, and where the pool
// has them. A wave takes HEADS heads of ROWS rows.
template <int PER, int HEADS>
struct Pg8At {
  static constexpr int LANES = PG_E / PER, ROWS = 64 / LANES / HEADS;
  int i, h, e;                             // e: the piece's first dim
  size_t row;                              // of the pool
  bool ours, there;                        // a sequence's row, or what may be one; one that the pool has a place for
  unsigned bad;
  __device__ __forceinline__ bool task(int M, int H) {
    const int lane = threadIdx.x & 63;
    const unsigned groups = (unsigned)H / HEADS;                   // (HEADS 1, or H a multiple)
    const unsigned w = __builtin_amdgcn_readfirstlane(blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6)), g = w / groups;
    h = (int)(w - g * groups) * HEADS + lane / LANES % HEADS;
    e = lane % LANES * PER;
    i = (int)g * ROWS + lane / LANES / HEADS;
    return (size_t)g * ROWS < (size_t)M;
  }
  __device__ __forceinline__ void place(int pages, int shift, const int* __restrict__ table, int N,
                                        const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M,
                                        int H) {
    // the wave's first row's sequence; most often that of its last row too
    const int first = __builtin_amdgcn_readfirstlane(i);
    int b = pg_owner(starts, B, first);
    if (ROWS > 1 && b + 1 < B && starts[b + 1] < first + ROWS) b = pg_owner(starts, B, i);
    const PgSeq s = pg_seq(starts, lengths, b, M, N << shift);
    const int j = i - s.first, pos = s.len - s.count + j;
    // (starts that leave a sequence no row do not say which are behind it)
    ours = i < M && ((j >= 0 && j < s.count) || (s.count == 0 && (s.bad & PG_ERR_STARTS)));
    bad = i < M ? s.bad : 0u;
    there = ours && s.bad == 0 && pos >= 0;
    row = 0;
    if (!there) return;
    const int page = table[(size_t)b * N + (pos >> shift)];
    there = (unsigned)page < (unsigned)pages;
    if (!there) bad |= PG_ERR_PAGE;
    row = (((size_t)(there ? page : 0) * H + h) << shift) + (pos & ((1 << shift) - 1));
  }
};

// ---------------------------------------------------------------- append
// As the 16-bit cache's: nothing is stored for a sequence that cannot be. 16 values
// a lane, 1024 a wave, of 16 rows of 64 or 8 of 128 (8 values a lane, whose loads
// leave nothing out: 75 us for the 67 above), or of HEADS heads of one row of 128.
// Stores go past the caches (19.2 -> 17.3 us before the heads of a row were together).
template <typename T, int HEADS>
__device__ __forceinline__ void pg8_append_body(const T* __restrict__ k, const T* __restrict__ v, long krow, long khead,
                                                long vrow, long vhead, unsigned char* __restrict__ kp,
                                                unsigned char* __restrict__ vp, unsigned char* __restrict__ ks,
                                                unsigned char* __restrict__ vs, int pages, int shift,
                                                const int* __restrict__ table, int N, const int* __restrict__ starts,
                                                const int* __restrict__ lengths, int B, int M, int H,
                                                unsigned* __restrict__ err) {
  Pg8At<16, HEADS> at;
  if (!at.task(M, H)) return;
  const long i = min(at.i, M - 1);
  Pg8Row<T> kw, vw;
  kw.get(k + i * krow + at.h * khead + at.e);
  vw.get(v + i * vrow + at.h * vhead + at.e);
  __builtin_amdgcn_sched_barrier(0);                               // in flight while the place is looked up
  at.place(pages, shift, table, N, starts, lengths, B, M, H);
  float x[16];
  unsigned sk, sv;
  kw.open(x);
  const vh_u32x4 kx = pg8_hold(x, sk);
  vw.open(x);
  const vh_u32x4 vx = pg8_hold(x, sv);
  if (at.there) {
    __builtin_nontemporal_store(kx, (vh_u32x4*)(kp + at.row * PG_E + at.e));
    __builtin_nontemporal_store(vx, (vh_u32x4*)(vp + at.row * PG_E + at.e));
    if (at.e % 32 == 0) {
      ks[at.row * (PG_E / 32) + at.e / 32] = (unsigned char)sk;
      vs[at.row * (PG_E / 32) + at.e / 32] = (unsigned char)sv;
    }
  }
  if (at.bad) pg_raise(err, at.bad);
}
#define PG8_APPEND(name, type, heads)                                                                              \
  extern "C" __global__ __launch_bounds__(256) void name(                                                          \
      const type* __restrict__ k, const type* __restrict__ v, long krow, long khead, long vrow, long vhead,        \
      unsigned char* __restrict__ kp, unsigned char* __restrict__ vp, unsigned char* __restrict__ ks,              \
      unsigned char* __restrict__ vs, int pages, int shift, const int* __restrict__ table, int N,                  \
      const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M, int H,                        \
      unsigned* __restrict__ err) {                                                                                \
    pg8_append_body<type, heads>(k, v, krow, khead, vrow, vhead, kp, vp, ks, vs, pages, shift, table, N, starts,  \
                                 lengths, B, M, H, err);                                                           \
  }
PG8_APPEND(pg_append16, unsigned short, 1)
PG8_APPEND(pg_append32, float, 1)
#if PG_E == 128
PG8_APPEND(pg_append16x8, unsigned short, 8)
#endif

// ---------------------------------------------------------------- read
// The rows of the new tokens' positions back as values. A row of a token at a
// negative position, or of a sequence that cannot be, becomes 0; rows that are
// no sequence's stay.
//
// A lane stores 16 bytes beside its neighbours', whole lines, past the caches, so
// that the pool may stay in them; as 16 values a lane, two or four stores that leave
// bytes out, they need the caches to put lines together, and push it out (28,800
// rows, three pools in turn: 25 heads of 64 73 -> 72 us, 12 heads 39.3 -> 28.2, in fp32 62.5
// -> 42.2; 8 heads of 128 50 -> 33.4; past the caches with what is left out 106).

// A lane's elements, which are 16 bytes of values.
template <typename T>
struct Pg8Piece {
  typedef vh_u32x2 held;
  static __device__ __forceinline__ vh_u32x4 open(held w, pg_factor f) { return pg_open(w[0], w[1], f); }
};
template <>
struct Pg8Piece<float> {
  typedef unsigned held;
  static __device__ __forceinline__ vh_u32x4 open(held w, pg_factor f) {
    const vh_u32x2 v = pg_open4(w, f);
    vh_u32x4 o;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      o[2 * j] = __builtin_bit_cast(unsigned, pg_to_f((unsigned short)(v[j] & 0xffffu)));
      o[2 * j + 1] = __builtin_bit_cast(unsigned, pg_to_f((unsigned short)(v[j] >> 16)));
    }
    return o;
  }
};
template <typename T>
__device__ __forceinline__ void pg8_read_body(T* __restrict__ k, T* __restrict__ v, long krow, long khead, long vrow,
                                              long vhead, PG_POOL, int pages, int shift, const int* __restrict__ table,
                                              int N, const int* __restrict__ starts, const int* __restrict__ lengths,
                                              int B, int M, int H, unsigned* __restrict__ err) {
  typedef Pg8Piece<T> P;
  Pg8At<16 / (int)sizeof(T), 1> at;
  if (!at.task(M, H)) return;
  at.place(pages, shift, table, N, starts, lengths, B, M, H);
  typename P::held kw = {}, vw = {};
  unsigned sk = PG8_LOW, sv = PG8_LOW;
  if (at.there) {
    kw = *(const typename P::held*)(kp + at.row * PG_E + at.e);
    vw = *(const typename P::held*)(vp + at.row * PG_E + at.e);
    sk = ks[at.row * (PG_E / 32) + at.e / 32];
    sv = vs[at.row * (PG_E / 32) + at.e / 32];
  }
  if (at.ours) {
    const vh_u32x4 kx = P::open(kw, pg_power(sk)), vx = P::open(vw, pg_power(sv));
    vh_u32x4 *ko = (vh_u32x4*)(k + at.i * krow + at.h * khead + at.e), *vo = (vh_u32x4*)(v + at.i * vrow + at.h * vhead + at.e);
    __builtin_nontemporal_store(kx, ko);
    __builtin_nontemporal_store(vx, vo);
  }
  if (at.bad) pg_raise(err, at.bad);
}
#define PG8_READ(name, type)                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void name(                                                          \
      type* __restrict__ k, type* __restrict__ v, long krow, long khead, long vrow, long vhead, PG_POOL, int pages, \
      int shift, const int* __restrict__ table, int N, const int* __restrict__ starts,                             \
      const int* __restrict__ lengths, int B, int M, int H, unsigned* __restrict__ err) {                          \
    pg8_read_body<type>(k, v, krow, khead, vrow, vhead, PG_POOL_ARGS, pages, shift, table, N, starts, lengths, B,  \
                        M, H, err);                                                                                \
  }
PG8_READ(pg_read16, unsigned short)
PG8_READ(pg_read32, float)
