// Rows into and out of a paged cache in 8 bits (hip/form8.h), after hip/paged.hip.
//
// A wave takes 1024 values of one head: 16 values a lane, of 16 rows of 64 or 8 of
// 128, so that what it stores lies together (a head's rows of a page do), the
// powers too: as eight values of all heads a lane, whose powers reach memory two
// or four bytes at a time, 12,900 rows of 8 heads of 128 took 22.8 us to append.
// Bound by memory: these rows 16.3 us (80 MB, 4.9 TB/s), 28,800 rows of 25 heads of
// 64 read back in 65.5 us (332 MB, 5.05 TB/s); eight rows 3.6 us, a launch and the
// loads that wait for one another.

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

// A lane's row i of the call's, its head's piece of 16 values, and where the pool
// has them.
#define PG8_ROWS (1024 / PG_E)             // of a wave
struct Pg8At {
  int i, h, e;                             // e: the piece's first dim
  size_t row;                              // of the pool
  bool ours, there;                        // a sequence's row, or what may be one; one that the pool has a place for
  unsigned bad;
};
__device__ __forceinline__ bool pg8_task(Pg8At& o, int M, int H) {
  const int lane = threadIdx.x & 63;
  const unsigned w = __builtin_amdgcn_readfirstlane(blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6)), g = w / (unsigned)H;
  o.h = (int)(w - g * (unsigned)H);
  o.e = lane % (PG_E / 16) * 16;
  if ((size_t)g * PG8_ROWS >= (size_t)M) return false;
  o.i = (int)g * PG8_ROWS + lane / (PG_E / 16);
  return true;
}
__device__ __forceinline__ void pg8_place(Pg8At& o, int pages, int shift, const int* __restrict__ table, int N,
                                          const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M,
                                          int H) {
  // the wave's first row's sequence; most often that of its last row too
  const int first = __builtin_amdgcn_readfirstlane(o.i);
  int b = pg_owner(starts, B, first);
  if (b + 1 < B && starts[b + 1] < first + PG8_ROWS) b = pg_owner(starts, B, o.i);
  const PgSeq s = pg_seq(starts, lengths, b, M, N << shift);
  const int j = o.i - s.first, pos = s.len - s.count + j;
  o.ours = o.i < M && (s.bad != 0 || (j >= 0 && j < s.count));
  o.bad = o.i < M ? s.bad : 0u;
  o.there = o.ours && s.bad == 0 && pos >= 0;
  o.row = 0;
  if (!o.there) return;
  const int page = table[(size_t)b * N + (pos >> shift)];
  o.there = (unsigned)page < (unsigned)pages;
  if (!o.there) o.bad |= PG_ERR_PAGE;
  o.row = (((size_t)(o.there ? page : 0) * H + o.h) << shift) + (pos & ((1 << shift) - 1));
}

// ---------------------------------------------------------------- append
// As the 16-bit cache's: nothing is stored for a sequence that cannot be.
template <typename T>
__device__ __forceinline__ void pg8_append_body(const T* __restrict__ k, const T* __restrict__ v, long krow, long khead,
                                                long vrow, long vhead, unsigned char* __restrict__ kp,
                                                unsigned char* __restrict__ vp, unsigned char* __restrict__ ks,
                                                unsigned char* __restrict__ vs, int pages, int shift,
                                                const int* __restrict__ table, int N, const int* __restrict__ starts,
                                                const int* __restrict__ lengths, int B, int M, int H,
                                                unsigned* __restrict__ err) {
  Pg8At at;
  if (!pg8_task(at, M, H)) return;
  const long i = min(at.i, M - 1);
  Pg8Row<T> kw, vw;
  kw.get(k + i * krow + at.h * khead + at.e);
  vw.get(v + i * vrow + at.h * vhead + at.e);
  __builtin_amdgcn_sched_barrier(0);                               // in flight while the place is looked up
  pg8_place(at, pages, shift, table, N, starts, lengths, B, M, H);
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
#define PG8_APPEND(name, type)                                                                                     \
  extern "C" __global__ __launch_bounds__(256) void name(                                                          \
      const type* __restrict__ k, const type* __restrict__ v, long krow, long khead, long vrow, long vhead,        \
      unsigned char* __restrict__ kp, unsigned char* __restrict__ vp, unsigned char* __restrict__ ks,              \
      unsigned char* __restrict__ vs, int pages, int shift, const int* __restrict__ table, int N,                  \
      const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M, int H,                        \
      unsigned* __restrict__ err) {                                                                                \
    pg8_append_body<type>(k, v, krow, khead, vrow, vhead, kp, vp, ks, vs, pages, shift, table, N, starts, lengths, \
                          B, M, H, err);                                                                           \
  }
PG8_APPEND(pg_append16, unsigned short)
PG8_APPEND(pg_append32, float)

// ---------------------------------------------------------------- read
// The rows of the new tokens' positions back as values. A row of a token at a
// negative position, or of a sequence that cannot be, becomes 0; rows that are
// no sequence's stay.
// A lane's 16 values. In 16 bits its stores of 16 bytes leave as many out: the
// caches put the lines together (28,800 rows of 25 heads of 64 76.4 us; past the
// caches 95.6, and 100 in pieces that two lanes have exchanged such that a store
// leaves nothing out).
__device__ __forceinline__ void pg8_put(unsigned short* p, vh_u32x4 w, pg_factor f) {
#pragma unroll
  for (int j = 0; j < 2; ++j) *(vh_u32x4*)(p + 8 * j) = pg_open(w[2 * j], w[2 * j + 1], f);
}
// In 32 bits a store would leave out 48 bytes of 64: four lanes, whose 64 values
// are one row's, store the first's together, then the second's.
template <int FROM>
__device__ __forceinline__ void pg8_put4(float* p, vh_u32x4 w, pg_factor f) {
  constexpr int CTRL = FROM * 0x55;                                // of each four lanes the FROM-th
  const int q = threadIdx.x & 3;
  unsigned t[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) t[j] = (unsigned)__builtin_amdgcn_mov_dpp((int)w[j], CTRL, 0xF, 0xF, true);
  const pg_factor g =
      __builtin_bit_cast(pg_factor, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, f), CTRL, 0xF, 0xF, true));
  const vh_u32x2 v = pg_open4(q & 2 ? (q & 1 ? t[3] : t[2]) : (q & 1 ? t[1] : t[0]), g);
  *(vh_f32x4*)(p + 16 * (FROM - q) + 4 * q) =
      vh_f32x4{pg_to_f((unsigned short)(v[0] & 0xffffu)), pg_to_f((unsigned short)(v[0] >> 16)),
               pg_to_f((unsigned short)(v[1] & 0xffffu)), pg_to_f((unsigned short)(v[1] >> 16))};
}
__device__ __forceinline__ void pg8_put(float* p, vh_u32x4 w, pg_factor f) {
  pg8_put4<0>(p, w, f);
  pg8_put4<1>(p, w, f);
  pg8_put4<2>(p, w, f);
  pg8_put4<3>(p, w, f);
}
template <typename T>
__device__ __forceinline__ void pg8_read_body(T* __restrict__ k, T* __restrict__ v, long krow, long khead, long vrow,
                                              long vhead, PG_POOL, int pages, int shift, const int* __restrict__ table,
                                              int N, const int* __restrict__ starts, const int* __restrict__ lengths,
                                              int B, int M, int H, int past, unsigned* __restrict__ err) {
  Pg8At at;
  if (!pg8_task(at, M, H)) return;
  pg8_place(at, pages, shift, table, N, starts, lengths, B, M, H);
  vh_u32x4 kw = {0u, 0u, 0u, 0u}, vw = kw;
  unsigned sk = PG8_LOW, sv = PG8_LOW;
  if (at.there) {
    const vh_u32x4 *ka = (const vh_u32x4*)(kp + at.row * PG_E + at.e), *va = (const vh_u32x4*)(vp + at.row * PG_E + at.e);
    if (past) {                                                    // (the asm keeps this a branch of its own)
      asm volatile("" ::: "memory");
      kw = __builtin_nontemporal_load(ka);
      vw = __builtin_nontemporal_load(va);
      asm volatile("" ::: "memory");
    } else {
      kw = *ka;
      vw = *va;
    }
    sk = ks[at.row * (PG_E / 32) + at.e / 32];
    sv = vs[at.row * (PG_E / 32) + at.e / 32];
  }
  if (at.ours) {
    pg8_put(k + at.i * krow + at.h * khead + at.e, kw, pg_power(sk));
    pg8_put(v + at.i * vrow + at.h * vhead + at.e, vw, pg_power(sv));
  }
  if (at.bad) pg_raise(err, at.bad);
}
#define PG8_READ(name, type)                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void name(                                                          \
      type* __restrict__ k, type* __restrict__ v, long krow, long khead, long vrow, long vhead, PG_POOL, int pages, \
      int shift, const int* __restrict__ table, int N, const int* __restrict__ starts,                             \
      const int* __restrict__ lengths, int B, int M, int H, int past, unsigned* __restrict__ err) {                \
    pg8_read_body<type>(k, v, krow, khead, vrow, vhead, PG_POOL_ARGS, pages, shift, table, N, starts, lengths, B,  \
                        M, H, past, err);                                                                          \
  }
PG8_READ(pg_read16, unsigned short)
PG8_READ(pg_read32, float)
