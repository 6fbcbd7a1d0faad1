// A key/value cache in pages for gfx950: rows appended to pages, attention of
// ragged chunks of new tokens over them, the weight each position receives,
// and eviction by that weight. Appended to the prelude (hip/prelude.h,
// VBLOCK 256) and compiled at run time by hipRTC, once per head width PG_E
// (64, 128) and kind PG_KIND:
//   0  fp16 cache, fp16 queries       1  bf16 cache, bf16 queries
//   2  fp16 cache, fp32 queries (results in fp32)
//
// One layer's pool is [pages, page, H, E]; row s of sequence b lies in page
// table[b, s / page], slot s % page (page = 2^shift). starts[b] .. starts[b + 1]
// are the rows of sequence b's new tokens in the call's [M, ..] tensors,
// lengths[b] its positions with them: new token j is at position
// lengths[b] - count + j and sees positions 0 .. that. A token at a negative
// position (a padded sequence of length 0) sees nothing and is not stored.
//
// Everything that comes from the device (page ids, starts, lengths) is checked
// where it is used: an impossible one raises the error word and is replaced
// by a possible one, so that no access leaves its tensor.

#define PG_F16 0
#define PG_BF16 1
#define PG_F32 2
#define PG_ERR_PAGE 1u          // a page id outside the pool
#define PG_ERR_STARTS 2u        // starts not ascending, or past the rows
#define PG_ERR_LENGTH 4u        // a length past the table
#define PG_ERR_MOST 8u          // a sequence with more new tokens than `most`

typedef __bf16 pg_b8 __attribute__((ext_vector_type(8)));
typedef float pg_f8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ void pg_raise(unsigned* err, unsigned bits) {
  __hip_atomic_fetch_or(err, bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sequence b: its first row, new tokens and length.
struct PgSeq {
  int first, count, len;
  unsigned bad;
};
__device__ __forceinline__ PgSeq pg_seq(const int* __restrict__ starts, const int* __restrict__ lengths, int b, int M,
                                        int cap) {
  PgSeq s;
  const int a = starts[b], e = starts[b + 1], n = lengths[b];
  s.first = min(max(a, 0), M);
  const int end = min(max(e, s.first), M);
  s.count = end - s.first;
  s.len = min(max(n, 0), cap);
  s.bad = (s.first != a || end != e ? PG_ERR_STARTS : 0u) | (s.len != n ? PG_ERR_LENGTH : 0u);
  return s;
}

// One element of a 16-bit word pair as fp32, and eight floats as 16-bit values
// (round to nearest even).
__device__ __forceinline__ float pg_to_f(unsigned short h) {
#if PG_KIND == PG_BF16
  return __builtin_bit_cast(float, (unsigned)h << 16);
#else
  return h2f(h);
#endif
}
__device__ __forceinline__ vh_u32x4 pg_pack8(pg_f8 v) {
#if PG_KIND == PG_BF16
  return __builtin_bit_cast(vh_u32x4, __builtin_convertvector(v, pg_b8));
#else
  return __builtin_bit_cast(vh_u32x4, __builtin_convertvector(v, vh_h8));
#endif
}

// ---------------------------------------------------------------- append
// New key and value rows into their pages, eight elements a thread (fp32 ones
// rounded to the pool's type).
template <typename T>
__device__ __forceinline__ vh_u32x4 pg_load8(const T* p);
template <>
__device__ __forceinline__ vh_u32x4 pg_load8<unsigned short>(const unsigned short* p) { return ld16(p); }
template <>
__device__ __forceinline__ vh_u32x4 pg_load8<float>(const float* p) {
  const vh_f32x4 a = *(const vh_f32x4*)p, b = *(const vh_f32x4*)(p + 4);
  return pg_pack8(pg_f8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

template <typename T>
__device__ __forceinline__ void pg_append_body(const T* __restrict__ k, const T* __restrict__ v, long krow, long khead,
                                               long vrow, long vhead, unsigned short* __restrict__ kp,
                                               unsigned short* __restrict__ vp, int pages, int shift,
                                               const int* __restrict__ table, int N, const int* __restrict__ starts,
                                               const int* __restrict__ lengths, int B, int M, int H,
                                               unsigned* __restrict__ err) {
  const int per = H * (PG_E / 8);                       // threads of a row
  const long at = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const int i = (int)(at / per), c = (int)(at % per);
  if (i >= M) return;
  // the last sequence whose first row is at or before i
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= i) lo = mid; else hi = mid;
  }
  const PgSeq s = pg_seq(starts, lengths, lo, M, N << shift);
  unsigned bad = s.bad;
  const int j = i - s.first, pos = s.len - s.count + j;
  if (j >= 0 && j < s.count && pos >= 0) {
    const int page = table[(size_t)lo * N + (pos >> shift)];
    if ((unsigned)page < (unsigned)pages) {
      const int h = c / (PG_E / 8), e = c % (PG_E / 8) * 8;
      const size_t to = ((((size_t)page << shift) + (pos & ((1 << shift) - 1))) * H + h) * PG_E + e;
      const vh_u32x4 kx = pg_load8(k + i * krow + h * khead + e), vx = pg_load8(v + i * vrow + h * vhead + e);
      *(vh_u32x4*)(kp + to) = kx;
      *(vh_u32x4*)(vp + to) = vx;
    } else {
      bad |= PG_ERR_PAGE;
    }
  }
  if (bad) pg_raise(err, bad);
}
#define PG_APPEND(name, type)                                                                                      \
  extern "C" __global__ __launch_bounds__(256) void name(                                                          \
      const type* __restrict__ k, const type* __restrict__ v, long krow, long khead, long vrow, long vhead,        \
      unsigned short* __restrict__ kp, unsigned short* __restrict__ vp, int pages, int shift,                      \
      const int* __restrict__ table, int N, const int* __restrict__ starts, const int* __restrict__ lengths, int B, \
      int M, int H, unsigned* __restrict__ err) {                                                                  \
    pg_append_body<type>(k, v, krow, khead, vrow, vhead, kp, vp, pages, shift, table, N, starts, lengths, B, M, H, \
                         err);                                                                                     \
  }
PG_APPEND(pg_append16, unsigned short)
PG_APPEND(pg_append32, float)

// ---------------------------------------------------------------- attention
// Matrix-core products over 16-bit operands: lane l = 16 q + r holds row r,
// fold positions 8 q .. 8 q + 7 of a 16 x 32 operand tile; the result's column
// r, rows 4 q .. 4 q + 3.
__device__ __forceinline__ vh_f32x4 pg_mfma(vh_u32x4 a, vh_u32x4 b, vh_f32x4 c) {
#if PG_KIND == PG_BF16
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pg_b8, a), __builtin_bit_cast(pg_b8, b), c, 0, 0, 0);
#else
  return vh_mfma(a, b, c);
#endif
}

// fp32 values go through the matrix cores in three fp16 planes v = hi + (lo +
// tail) / 2^11, each what is left cut off after 11 bits: 24 bits. The two lower
// planes share an accumulator.
#if PG_KIND == PG_F32
#define PG_PLANES 3
typedef float pg_q;
#else
#define PG_PLANES 1
typedef unsigned short pg_q;
#endif
__device__ __forceinline__ void pg_split(const float* v, vh_u32x4* f) {
#if PG_KIND == PG_F32
  typedef __fp16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const h2 h = __builtin_amdgcn_cvt_pkrtz(v[2 * j], v[2 * j + 1]);
    const float r0 = fmaf((float)h[0], -VH_LO_SCALE, v[2 * j] * VH_LO_SCALE);
    const float r1 = fmaf((float)h[1], -VH_LO_SCALE, v[2 * j + 1] * VH_LO_SCALE);
    const h2 l = __builtin_amdgcn_cvt_pkrtz(r0, r1);
    const h2 t = __builtin_amdgcn_cvt_pkrtz(r0 - (float)l[0], r1 - (float)l[1]);
    f[0][j] = __builtin_bit_cast(unsigned, h);
    f[1][j] = __builtin_bit_cast(unsigned, l);
    f[2][j] = __builtin_bit_cast(unsigned, t);
  }
#else
  f[0] = pg_pack8(pg_f8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]});
#endif
}

// A wave's lanes hand each other values through LDS, whose operations a wave
// executes in order: this keeps the compiler to that order too.
__device__ __forceinline__ void pg_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// 16 query rows as the products' column operand: lane 16 q + r holds row r's
// dims 32 k + 8 q .. + 7, k < E / 32. fp32 rows are scaled by a power of two
// to below 1, so that any magnitude splits; k2 is the factor that makes scores
// powers of two: scale log2(e), times that power.
struct PgQuery {
  vh_u32x4 f[PG_E / 32][PG_PLANES];
  float k2;
};
__device__ __forceinline__ void pg_query(PgQuery& o, const pg_q* __restrict__ qp, int q, float scale2) {
#if PG_KIND == PG_F32
  float v[PG_E / 32][8];
  float mx = 0.0f;
#pragma unroll
  for (int k = 0; k < PG_E / 32; ++k) {
    const vh_f32x4 a = *(const vh_f32x4*)(qp + 32 * k + 8 * q), c = *(const vh_f32x4*)(qp + 32 * k + 8 * q + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[k][j] = a[j];
      v[k][4 + j] = c[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) mx = fmaxf(mx, __builtin_fabsf(v[k][j]));
  }
  mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
  mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
  int e = 0;
  if (mx > 0.0f && mx < INFINITY) e = max(__builtin_amdgcn_frexp_expf(mx), -100);
#pragma unroll
  for (int k = 0; k < PG_E / 32; ++k) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[k][j] = __builtin_ldexpf(v[k][j], -e);
    pg_split(v[k], o.f[k]);
  }
  o.k2 = __builtin_ldexpf(scale2, e);
#else
#pragma unroll
  for (int k = 0; k < PG_E / 32; ++k) o.f[k][0] = ld16(qp + 32 * k + 8 * q);
  o.k2 = scale2;
#endif
}

// Scores of 16 positions (their rows' pieces kf[k], the row operand) and the
// wave's 16 queries: lane 16 q + r gets positions 4 q + j of query r. In fp32,
// a score whose hi part is not finite (the cache may hold an infinity) is made
// again: 0 * inf of a plane that is 0 where the query is not would make an
// infinity a NaN.
__device__ __forceinline__ void pg_scores(const vh_u32x4* kf, const PgQuery& qf, const pg_q* __restrict__ qp, int lane,
                                          float* s) {
  vh_f32x4 h = {0.0f, 0.0f, 0.0f, 0.0f};
#if PG_KIND == PG_F32
  vh_f32x4 g = h, l = h;
#pragma unroll
  for (int k = 0; k < PG_E / 32; ++k) {
    if (k & 1) g = pg_mfma(kf[k], qf.f[k][0], g);
    else h = pg_mfma(kf[k], qf.f[k][0], h);
    l = pg_mfma(kf[k], qf.f[k][1], l);
    l = pg_mfma(kf[k], qf.f[k][2], l);
  }
  float fin = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[j] += g[j];
    s[j] = vh_hilo(h[j], l[j]);
    fin = fmaf(h[j], 0.0f, fin);
  }
  if (__any(fin != fin)) {
#pragma nounroll
    for (int j = 0; j < 4; ++j) {
      float acc = 0.0f;
      const int pr = 4 * (lane >> 4) + j;              // the position's row of the operand tile
#pragma unroll
      for (int k = 0; k < PG_E / 32; ++k)
#pragma nounroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const unsigned x = (unsigned)__shfl((int)kf[k][w], 16 * c + pr, 64);
            acc = fmaf(qp[32 * k + 8 * c + 2 * w], h2f_lo(x), acc);
            acc = fmaf(qp[32 * k + 8 * c + 2 * w + 1], h2f_hi(x), acc);
          }
      if (!(__builtin_fabsf(h[j]) < INFINITY)) s[j] = acc;
    }
  }
#else
#pragma unroll
  for (int k = 0; k < PG_E / 32; ++k) h = pg_mfma(kf[k], qf.f[k][0], h);
#pragma unroll
  for (int j = 0; j < 4; ++j) s[j] = h[j];
#endif
}

// Whether a 16-bit value is an infinity or a NaN (its exponent bits all set),
// and the same of a word's two: a unit added to the exponents carries into the
// halves' top bits.
#define PG_EXP (PG_KIND == PG_BF16 ? 0x7f80u : 0x7c00u)
__device__ __forceinline__ bool pg_wild(unsigned short h) { return (h & PG_EXP) == PG_EXP; }
__device__ __forceinline__ unsigned pg_wild2(unsigned x) {
  return ((x & (PG_EXP << 16 | PG_EXP)) + (0x80008000u - (PG_EXP << 16 | PG_EXP))) & 0x80008000u;
}

// A block makes 16 rows of one (sequence, key head): row x stands for new
// token x / G, query head G h + x % G. Its four waves take every fourth step
// of PG_STEP positions each and combine at the end. Scores are K Q^T, outputs
// V^T P^T, so that a lane holds values of one row (lane % 16) in both, and the
// weights feed the second product from the registers the first left them in:
// the instruction's fold position 8 q + e stands for position 4 q + e (e < 4)
// or 16 + 4 q + e - 4 of 32. Value rows go through LDS and are read transposed
// (ds_read_b64_tr_b16: 16 lanes read four rows of 16 values and get a column
// of four each). The softmax is a running one in powers of two, statistics in
// fp32; weights are rounded to the cache's type for the second product, as
// their values are (fp32 queries: 24 bits in three planes).
#define PG_STEP (PG_E == 64 ? 64 : 32)
#define PG_VROW (PG_E + 16)                // halves of a value row in LDS: 16 past a multiple of 32 banks
extern "C" __global__ __launch_bounds__(256, 2) void pg_attn(
    const pg_q* __restrict__ Q, long qrow, long qhead, const unsigned short* __restrict__ kp,
    const unsigned short* __restrict__ vp, int pages, int shift, const int* __restrict__ table, int N,
    const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M, int H, int G, int tiles, int most,
    float scale2, pg_q* __restrict__ out, long orow, long ohead, float* __restrict__ lse, unsigned* __restrict__ err) {
  constexpr int KS = PG_E / 32, NG = PG_STEP / 16, NV = PG_STEP * PG_E / 512, DT = PG_E / 16;
  __shared__ __attribute__((aligned(16))) unsigned short lv[4][PG_STEP * PG_VROW];
  __shared__ float om[4][2][16];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, q = lane >> 4;
  const int T = B * H * tiles, per = (T + 7) / 8, id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || id >= T) return;
  const int h = id / tiles % H, b = id / tiles / H;
  const PgSeq sq = pg_seq(starts, lengths, b, M, N << shift);
  const int R = sq.count * G, x0 = (tiles - 1 - id % tiles) * 16;  // the longest first
  unsigned bad = sq.bad | (sq.count > most ? PG_ERR_MOST : 0u);
  if (x0 == 0 && bad && tid == 0) pg_raise(err, bad);
  bad = 0;
  if (x0 >= R) return;
  const int x = min(x0 + r, R - 1), tok = x / G, head = h * G + x % G;
  const bool live = x0 + r < R;
  const int lim = sq.len - sq.count + tok;                         // this lane's last position
  const int last = sq.len - sq.count + min(x0 + 15, R - 1) / G, first = sq.len - sq.count + x0 / G;
  const int nt = last < 0 ? 0 : last / PG_STEP + 1;
  const pg_q* qp = Q + (sq.first + tok) * qrow + head * qhead;
  PgQuery qf;
  pg_query(qf, qp, q, scale2);
  const size_t rowlen = (size_t)H * PG_E;
  const int* tb = table + (size_t)b * N;
  auto row = [&](int s) -> size_t {                                // element offset of position s's row
    const int page = tb[s >> shift];
    const bool in = (unsigned)page < (unsigned)pages;
    if (!in) bad = PG_ERR_PAGE;
    return (((size_t)(in ? page : 0) << shift) + (s & ((1 << shift) - 1))) * rowlen + h * PG_E;
  };
  float o[DT][4] = {};
  float m2 = -INFINITY, sum = 0.0f;
  unsigned short* V = lv[wave];
  for (int t = wave; t < nt; t += 4) {
    const int p0 = t * PG_STEP;
    vh_u32x4 vr[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) {                                 // positions past the last: zeros
      const int s = p0 + n * (512 / PG_E) + lane / (PG_E / 8);
      vr[n] = ld16(vp + row(min(s, last)) + lane % (PG_E / 8) * 8);
      if (s > last) vr[n] = vh_u32x4{0u, 0u, 0u, 0u};
    }
    float s[NG][4];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      vh_u32x4 kf[KS];
      const unsigned short* kr = kp + row(min(p0 + 16 * i + r, last)) + 8 * q;
#pragma unroll
      for (int k = 0; k < KS; ++k) kf[k] = ld16(kr + 32 * k);
      pg_scores(kf, qf, qp, lane, s[i]);
    }
    const bool part = p0 + PG_STEP - 1 > first;                    // some row sees it in part
    // values that are not finite are left out of the product where a row may
    // not see their position, or a plane of its weight may be 0: 0 * inf ...
    bool wild = false;
    if (part || PG_KIND == PG_F32) {
      unsigned any = 0u;
#pragma unroll
      for (int n = 0; n < NV; ++n) any |= pg_wild2(vr[n][0]) | pg_wild2(vr[n][1]) | pg_wild2(vr[n][2]) | pg_wild2(vr[n][3]);
      wild = __any(any != 0u);
    }
    if (part) {
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = p0 + 16 * i + 4 * q + j <= lim ? s[i][j] : -INFINITY;
    }
    pg_wave_sync();
#pragma unroll
    for (int n = 0; n < NV; ++n)
      *(vh_u32x4*)(V + (n * (512 / PG_E) + lane / (PG_E / 8)) * PG_VROW + lane % (PG_E / 8) * 8) = vr[n];
    pg_wave_sync();
    float bm = s[0][0];
#pragma unroll
    for (int n = 1; n < 4 * NG; ++n) bm = fmaxf(bm, s[n >> 2][n & 3]);
    bm = fmaxf(bm, __shfl_xor(bm, 16, 64));
    bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
    const float n2 = fmaxf(m2, bm * qf.k2);
    const float ref = n2 == -INFINITY ? 0.0f : n2;                 // no score above -inf yet: all weights 0
    const float c = __builtin_amdgcn_exp2f(m2 - ref);
    m2 = n2;
    vh_u32x4 pf[NG / 2][PG_PLANES];
    float ts = 0.0f;
#pragma unroll
    for (int k = 0; k < NG / 2; ++k) {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(fmaf(s[2 * k + (j >> 2)][j & 3], qf.k2, -ref));
      ts += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      pg_split(w, pf[k]);
    }
    sum = fmaf(sum, c, ts);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      vh_f32x4 th = {0.0f, 0.0f, 0.0f, 0.0f};
#if PG_KIND == PG_F32
      vh_f32x4 tl = th;
#endif
#pragma unroll
      for (int k = 0; k < NG / 2; ++k) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef short s8 __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) s4 lds4;
        unsigned short* vb = V + (32 * k + 4 * q + r / 4) * PG_VROW + 16 * d + 4 * (r & 3);
        const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)vb);
        const s4 e = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(vb + 16 * PG_VROW));
        s8 f = __builtin_shufflevector(a, e, 0, 1, 2, 3, 4, 5, 6, 7);
        if (wild) {
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = pg_wild((unsigned short)f[j]) ? 0 : f[j];
        }
        const vh_u32x4 vf = __builtin_bit_cast(vh_u32x4, f);
        th = pg_mfma(vf, pf[k][0], th);
#if PG_KIND == PG_F32
        tl = pg_mfma(vf, pf[k][1], tl);
        tl = pg_mfma(vf, pf[k][2], tl);
#endif
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#if PG_KIND == PG_F32
        o[d][j] = fmaf(o[d][j], c, vh_hilo(th[j], tl[j]));
#else
        o[d][j] = fmaf(o[d][j], c, th[j]);
#endif
      }
    }
    if (wild) {                                                    // ... and go to the rows that see them
      for (int s = p0; s <= min(p0 + PG_STEP - 1, last); ++s)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const unsigned short v = V[(s - p0) * PG_VROW + 16 * d + 4 * q + j];
            if (pg_wild(v) && s <= lim) o[d][j] += pg_to_f(v);
          }
    }
  }
  if (__any(bad != 0) && lane == 0) pg_raise(err, PG_ERR_PAGE);
  sum += __shfl_xor(sum, 16, 64);
  sum += __shfl_xor(sum, 32, 64);
  // each wave's maximum, sum and output, rescaled to the common maximum and
  // added in wave order; wave w then makes every fourth dim tile
  float* ow = (float*)lv;                                          // [wave][dim tile][j][lane]
  static_assert(sizeof(lv) >= 4 * DT * 4 * 64 * 4, "the value tiles hold the waves' outputs");
  __syncthreads();
  if (q == 0) {
    om[wave][0][r] = m2;
    om[wave][1][r] = sum;
  }
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) ow[((wave * DT + d) * 4 + j) * 64 + lane] = o[d][j];
  __syncthreads();
  float m = om[0][0][r];
#pragma unroll
  for (int w = 1; w < 4; ++w) m = fmaxf(m, om[w][0][r]);
  sum = 0.0f;
  float f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = om[w][0][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(om[w][0][r] - m);   // no score: 0
    sum = fmaf(om[w][1][r], f[w], sum);
  }
  if (!live) return;
  pg_q* op = out + (sq.first + tok) * orow + head * ohead;
#pragma unroll
  for (int d = wave; d < DT; d += 4) {
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = fmaf(ow[((w * DT + d) * 4 + j) * 64 + lane], f[w], v[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = lim < 0 ? 0.0f : v[j] / sum;
#if PG_KIND == PG_F32
    *(vh_f32x4*)(op + 16 * d + 4 * q) = vh_f32x4{v[0], v[1], v[2], v[3]};
#else
    const vh_u32x4 w = pg_pack8(pg_f8{v[0], v[1], v[2], v[3], 0.0f, 0.0f, 0.0f, 0.0f});
    *(vh_u32x2*)(op + 16 * d + 4 * q) = vh_u32x2{w[0], w[1]};
#endif
  }
  // log2 of the row's sum of 2^score: +inf for a row that sees nothing, so
  // that all its weights are 0
  if (lse && wave == 0 && q == 0)
    lse[(size_t)(sq.first + tok) * (H * G) + head] = lim < 0 ? INFINITY : m + __builtin_amdgcn_logf(sum);
}

// ---------------------------------------------------------------- weights
// out[b, h, s] = old[b, h, s] (0 for the chunk's own positions) + the sum over
// the sequence's rows (tokens and the group's heads) of the softmax weight at
// s; 0 past the length. A block takes 128 positions of one (sequence, key
// head), 32 to a wave, their key rows in registers, and goes through the rows
// that see them, 16 at a time, in order: no atomics, the same sums each time.
// Scores are made again (as in pg_attn), the weight is 2^(score - lse).
extern "C" __global__ __launch_bounds__(256, 2) void pg_weigh(
    const pg_q* __restrict__ Q, long qrow, long qhead, const unsigned short* __restrict__ kp, int pages, int shift,
    const int* __restrict__ table, int N, const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M,
    int H, int G, float scale2, const float* __restrict__ lse, const float* __restrict__ old, int S,
    float* __restrict__ out, int So, int blocks) {
  constexpr int KS = PG_E / 32;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, q = lane >> 4;
  const int T = B * H * blocks, per = (T + 7) / 8, id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || id >= T) return;
  const int h = id / blocks % H, b = id / blocks / H, p0 = id % blocks * 128 + 32 * wave;
  if (p0 >= So) return;
  const PgSeq sq = pg_seq(starts, lengths, b, M, N << shift);
  const int new0 = sq.len - sq.count, R = sq.count * G;
  float acc[2][4] = {};
  if (p0 < sq.len) {
    vh_u32x4 kf[2][KS];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int s = min(p0 + 16 * i + r, sq.len - 1), page = table[(size_t)b * N + (s >> shift)];
      const size_t at = (((size_t)((unsigned)page < (unsigned)pages ? page : 0) << shift) + (s & ((1 << shift) - 1)));
#pragma unroll
      for (int k = 0; k < KS; ++k) kf[i][k] = ld16(kp + (at * H + h) * PG_E + 32 * k + 8 * q);
    }
    // from the first token that sees the wave's first position
    for (int x0 = max(p0 - new0, 0) * G / 16 * 16; x0 < R; x0 += 16) {
      const int x = min(x0 + r, R - 1), tok = x / G, head = h * G + x % G;
      const int lim = x0 + r < R ? new0 + tok : -1;
      const pg_q* qp = Q + (sq.first + tok) * qrow + head * qhead;
      PgQuery qf;
      pg_query(qf, qp, q, scale2);
      const float z = lse[(size_t)(sq.first + tok) * (H * G) + head];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float s[4];
        pg_scores(kf[i], qf, qp, lane, s);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] += p0 + 16 * i + 4 * q + j <= lim ? __builtin_amdgcn_exp2f(fmaf(s[j], qf.k2, -z)) : 0.0f;
      }
    }
  }
  const size_t bh = (size_t)b * H + h;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float w = acc[i][j];
      w += __shfl_xor(w, 1, 64);
      w += __shfl_xor(w, 2, 64);
      w += __shfl_xor(w, 4, 64);
      w += __shfl_xor(w, 8, 64);
      const int s = p0 + 16 * i + 4 * q + j;
      if (r == 0 && s < So) out[bh * So + s] = w + (s < new0 ? old[bh * S + s] : 0.0f);
    }
}

// ---------------------------------------------------------------- eviction
// pg_select: a block per (layer, sequence, head) finds which positions stay:
// the `recent` last and, of the others, those of largest weight, ties to the
// lowest position, min(keep, length) in all. The weight of the last one to stay
// is found eight bits at a time (histograms of an order-preserving integer
// key), then the positions are listed in order. A NaN counts as the largest.
__device__ __forceinline__ unsigned pg_key(float w) {
  const unsigned u = __builtin_bit_cast(unsigned, w + 0.0f);       // -0 as 0
  if (w != w) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

extern "C" __global__ __launch_bounds__(1024) void pg_select(const float* __restrict__ weight, int S,
                                                             const int* __restrict__ lengths, int cap, int B, int H,
                                                             int keep, int recent, int* __restrict__ kept,
                                                             float* __restrict__ wout, int So,
                                                             int* __restrict__ lout, unsigned* __restrict__ err) {
  __shared__ int hist[256];
  __shared__ int wsum[16][2];
  __shared__ unsigned s_prefix;
  __shared__ int s_need;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / H % B;                                // grid: layers * B * H
  const int len = lengths[b], n = min(max(len, 0), cap);
  const int m = min(keep, n), last = min(recent, m), C = n - last, take = m - last;
  if (blockIdx.x < (unsigned)(B * H) && blockIdx.x % H == 0 && tid == 0) {
    lout[b] = m;
    if (n != len) pg_raise(err, PG_ERR_LENGTH);
  }
  const float* w = weight + (size_t)blockIdx.x * S;
  unsigned prefix = 0;
  int need = take;                                                 // of those with the prefix so far
  for (int bit = 24; bit >= 0; bit -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int s = tid; s < C; s += 1024) {
      const unsigned k = pg_key(w[s]);
      if (bit == 24 || (k >> (bit + 8)) == prefix) atomicAdd(&hist[(k >> bit) & 255u], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int v = 255, left = need;
      while (v > 0 && left > hist[v]) left -= hist[v--];
      s_prefix = prefix << 8 | (unsigned)v;
      s_need = left;
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
  }
  // positions in order: those above the key stay, and the first `need` that equal it
  int* kp = kept + (size_t)blockIdx.x * keep;
  float* wp = wout + (size_t)blockIdx.x * So;
  int above0 = 0, same0 = 0;
  for (int base = 0; base < n; base += 1024) {
    const int s = base + tid;
    float x = 0.0f;
    bool above = false, same = false;
    if (s < n) {
      x = w[s];
      const unsigned k = pg_key(x);
      above = s >= C || (take > 0 && k > prefix);
      same = s < C && take > 0 && k == prefix;
    }
    const unsigned long long am = __ballot(above), sm = __ballot(same), below = (1ull << lane) - 1ull;
    if (lane == 0) {
      wsum[wave][0] = __popcll(am);
      wsum[wave][1] = __popcll(sm);
    }
    __syncthreads();
    int a = above0, e = same0;
    for (int i = 0; i < 16; ++i) {
      if (i < wave) {
        a += wsum[i][0];
        e += wsum[i][1];
      }
      above0 += wsum[i][0];
      same0 += wsum[i][1];
    }
    a += __popcll(am & below);
    e += __popcll(sm & below);
    if (above || (same && e < need)) {
      const int to = a + min(e, need);
      if (to < keep) {
        kp[to] = s;
        wp[to] = x;
      }
    }
    __syncthreads();
  }
  for (int s = m + tid; s < keep; s += 1024) kp[s] = -1;
  for (int s = m + tid; s < So; s += 1024) wp[s] = 0.0f;
}

// pg_move: the kept rows of all layers into the pages of the other table, 16
// bytes of a key and of a value row a thread.
extern "C" __global__ __launch_bounds__(256) void pg_move(unsigned short* __restrict__ kp, unsigned short* __restrict__ vp,
                                                          int pages, int shift, const int* __restrict__ table, int N,
                                                          const int* __restrict__ to, int No,
                                                          const int* __restrict__ kept, int keep, int B, int H,
                                                          int blocks, unsigned* __restrict__ err) {
  const int lb = blockIdx.x / blocks, b = lb % B, layer = lb / B;  // grid: layers * B * blocks
  const long at = (long)(blockIdx.x % blocks) * 256 + threadIdx.x;
  const int per = H * (PG_E / 8), d = (int)(at / per), c = (int)(at % per), h = c / (PG_E / 8);
  if (d >= keep) return;
  const int s = kept[((size_t)lb * H + h) * keep + d];
  if (s < 0) return;
  const int sp = table[(size_t)b * N + (s >> shift)], dp = to[(size_t)b * No + (d >> shift)];
  if ((unsigned)sp >= (unsigned)pages || (unsigned)dp >= (unsigned)pages) {
    pg_raise(err, PG_ERR_PAGE);
    return;
  }
  const int mask = (1 << shift) - 1;
  const size_t pool = ((size_t)layer * pages) << shift;
  const size_t from = (pool + ((size_t)sp << shift) + (s & mask)) * per + c;
  const size_t into = (pool + ((size_t)dp << shift) + (d & mask)) * per + c;
  const vh_u32x4 kx = *((const vh_u32x4*)kp + from), vx = *((const vh_u32x4*)vp + from);
  *((vh_u32x4*)kp + into) = kx;
  *((vh_u32x4*)vp + into) = vx;
}
