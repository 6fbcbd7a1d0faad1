// Rows into and out of a paged cache in 8 bits (hip/form8.h), after hip/paged.hip.
// Eight values a thread, of a key and of a value row; the four threads of a
// block of 32 agree on its largest.

// A lane's neighbours in its four.
template <int CTRL>
__device__ __forceinline__ float pg8_quad(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}

// Eight values as elements, and their block's byte.
__device__ __forceinline__ vh_u32x2 pg8_hold(const float* x, unsigned& s) {
  float mx = 0.0f;
  bool odd = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = __builtin_fabsf(x[j]);
    const bool fin = a < INFINITY;                                 // (false for a NaN)
    mx = fmaxf(mx, fin ? a : 0.0f);
    odd |= !fin;
  }
#if PG_FORM == 1
  mx = odd ? INFINITY : mx;                                        // the whole block's
#endif
  mx = fmaxf(mx, pg8_quad<0xB1>(mx));                              // lanes 1 0 3 2
  mx = fmaxf(mx, pg8_quad<0x4E>(mx));                              // lanes 2 3 0 1
  s = (unsigned)min(max((int)((__builtin_bit_cast(unsigned, mx) + PG8_ROUND) >> 23) - PG8_BELOW, PG8_LOW), PG8_HIGH);
  vh_u32x2 w = {0u, 0u};
#if PG_FORM == 1
  const float f = __builtin_bit_cast(float, (260u - s) << 23);     // 2^(133 - s)
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int q = (int)fminf(fmaxf(__builtin_rintf(x[j] * f), -127.0f), 127.0f);
    w[j >> 2] |= ((unsigned)q & 255u) << 8 * (j & 3);
  }
  if (mx == INFINITY) s = PG8_NAN;
#else
  const float f = __builtin_bit_cast(float, (254u - s) << 23);     // 2^(127 - s)
  float y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    y[j] = __builtin_fabsf(x[j]) < INFINITY ? fminf(fmaxf(x[j] * f, -448.0f), 448.0f) : __builtin_nanf("");
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j], y[4 * j + 1], 0, false);
    w[j] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j + 2], y[4 * j + 3], v, true);
  }
#endif
  return w;
}

template <typename T>
__device__ __forceinline__ void pg8_get(const T* p, float* x);
template <>
__device__ __forceinline__ void pg8_get<unsigned short>(const unsigned short* p, float* x) {
  const vh_u32x4 v = ld16(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = pg_to_f((unsigned short)(v[j] & 0xffffu));
    x[2 * j + 1] = pg_to_f((unsigned short)(v[j] >> 16));
  }
}
template <>
__device__ __forceinline__ void pg8_get<float>(const float* p, float* x) {
  const vh_f32x4 a = *(const vh_f32x4*)p, b = *(const vh_f32x4*)(p + 4);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[j] = a[j];
    x[4 + j] = b[j];
  }
}

// Thread `at`'s row, head and dims, and where the pool has them; its place is
// none (false) where nothing may be stored, or read.
__device__ __forceinline__ bool pg8_place(size_t& row, int i, int h, int pages, int shift, const int* __restrict__ table,
                                          int N, const int* __restrict__ starts, const int* __restrict__ lengths, int B,
                                          int M, int H, bool& inside, unsigned& bad) {
  const int lo = pg_owner(starts, B, i);
  const PgSeq s = pg_seq(starts, lengths, lo, M, N << shift);
  const int j = i - s.first, pos = s.len - s.count + j;
  inside = s.bad != 0 || (j >= 0 && j < s.count);                  // a row that is a sequence's, or may be
  bad = s.bad;
  if (s.bad || !inside || pos < 0) return false;
  const int page = table[(size_t)lo * N + (pos >> shift)];
  if ((unsigned)page >= (unsigned)pages) {
    bad |= PG_ERR_PAGE;
    return false;
  }
  row = (((size_t)page * H + h) << shift) + (pos & ((1 << shift) - 1));
  return true;
}

// ---------------------------------------------------------------- append
// As pg_append: nothing is stored for a sequence that cannot be.
template <typename T>
__device__ __forceinline__ void pg8_append_body(const T* __restrict__ k, const T* __restrict__ v, long krow, long khead,
                                                long vrow, long vhead, unsigned char* __restrict__ kp,
                                                unsigned char* __restrict__ vp, unsigned char* __restrict__ ks,
                                                unsigned char* __restrict__ vs, int pages, int shift,
                                                const int* __restrict__ table, int N, const int* __restrict__ starts,
                                                const int* __restrict__ lengths, int B, int M, int H,
                                                unsigned* __restrict__ err) {
  const int per = H * (PG_E / 8);                                  // threads of a row
  const long at = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const int i = (int)(at / per), c = (int)(at % per);
  if (i >= M) return;                                              // (whole blocks of 32: per is a multiple of four)
  const int h = c / (PG_E / 8), e = c % (PG_E / 8) * 8;
  float kx[8], vx[8];
  pg8_get<T>(k + i * krow + h * khead + e, kx);
  pg8_get<T>(v + i * vrow + h * vhead + e, vx);
  __builtin_amdgcn_sched_barrier(0);                               // in flight while the place is looked up
  size_t row;
  bool inside;
  unsigned bad, sk, sv;
  const bool to = pg8_place(row, i, h, pages, shift, table, N, starts, lengths, B, M, H, inside, bad);
  const vh_u32x2 kw = pg8_hold(kx, sk), vw = pg8_hold(vx, sv);
  if (to) {
    *(vh_u32x2*)(kp + row * PG_E + e) = kw;
    *(vh_u32x2*)(vp + row * PG_E + e) = vw;
    if (e % 32 == 0) {
      ks[row * (PG_E / 32) + e / 32] = (unsigned char)sk;
      vs[row * (PG_E / 32) + e / 32] = (unsigned char)sv;
    }
  }
  if (bad) pg_raise(err, bad);
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
template <typename T>
__device__ __forceinline__ void pg8_put(T* p, vh_u32x4 v);
template <>
__device__ __forceinline__ void pg8_put<unsigned short>(unsigned short* p, vh_u32x4 v) { *(vh_u32x4*)p = v; }
template <>
__device__ __forceinline__ void pg8_put<float>(float* p, vh_u32x4 v) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = pg_to_f((unsigned short)(v[j] & 0xffffu));
    x[2 * j + 1] = pg_to_f((unsigned short)(v[j] >> 16));
  }
  *(vh_f32x4*)p = vh_f32x4{x[0], x[1], x[2], x[3]};
  *(vh_f32x4*)(p + 4) = vh_f32x4{x[4], x[5], x[6], x[7]};
}
template <typename T>
__device__ __forceinline__ void pg8_read_body(T* __restrict__ k, T* __restrict__ v, long krow, long khead, long vrow,
                                              long vhead, PG_POOL, int pages, int shift, const int* __restrict__ table,
                                              int N, const int* __restrict__ starts, const int* __restrict__ lengths,
                                              int B, int M, int H, unsigned* __restrict__ err) {
  const int per = H * (PG_E / 8);
  const long at = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const int i = (int)(at / per), c = (int)(at % per);
  if (i >= M) return;
  const int h = c / (PG_E / 8), e = c % (PG_E / 8) * 8;
  size_t row;
  bool inside;
  unsigned bad;
  vh_u32x4 kx = {0u, 0u, 0u, 0u}, vx = kx;
  if (pg8_place(row, i, h, pages, shift, table, N, starts, lengths, B, M, H, inside, bad)) {
    const vh_u32x2 kw = *(const vh_u32x2*)(kp + row * PG_E + e), vw = *(const vh_u32x2*)(vp + row * PG_E + e);
    kx = pg_open(kw[0], kw[1], pg_power(ks[row * (PG_E / 32) + e / 32]));
    vx = pg_open(vw[0], vw[1], pg_power(vs[row * (PG_E / 32) + e / 32]));
  }
  if (inside) {
    pg8_put<T>(k + i * krow + h * khead + e, kx);
    pg8_put<T>(v + i * vrow + h * vhead + e, vx);
  }
  if (bad) pg_raise(err, bad);
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
