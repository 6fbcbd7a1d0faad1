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
// by a possible one, so that no access leaves its tensor; nothing is appended
// for a sequence that has one.

#define PG_F16 0
#define PG_BF16 1
#define PG_F32 2
#define PG_ERR_PAGE 1u          // a page id outside the pool
#define PG_ERR_STARTS 2u        // starts not ascending, or past the rows
#define PG_ERR_LENGTH 4u        // a length past the table
#define PG_ERR_MOST 8u          // a sequence with more new tokens than `most`
#define PG_ERR_POSITION 16u     // a position past the model's learned ones
#define PG_ERR_TOKEN 32u        // a token id outside the vocabulary

typedef __bf16 pg_b8 __attribute__((ext_vector_type(8)));
typedef float pg_f8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ void pg_raise(unsigned* err, unsigned bits) {
  __hip_atomic_fetch_or(err, bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The error word, read and cleared at once.
extern "C" __global__ __launch_bounds__(64) void pg_take(unsigned* __restrict__ err, unsigned* __restrict__ took) {
  if (threadIdx.x == 0) *took = __hip_atomic_exchange(err, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// x / d of whole numbers, x >= 0 and d > 0: the compiler's 32-bit division is
// some 35 dependent operations, and a small call waits for half a dozen. Below
// 2^22 the reciprocal's quotient is off by one at most.
__device__ __forceinline__ int pg_div(int x, int d) {
  if (x >= 1 << 22) return x / d;
  const int q = (int)((float)x * __builtin_amdgcn_rcpf((float)d)), r = x - q * d;
  return q + (r >= d ? 1 : 0) - (r < 0 ? 1 : 0);
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

// Row i's sequence: the last whose first row is at or before it.
__device__ __forceinline__ int pg_owner(const int* __restrict__ starts, int B, int i) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
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
// rounded to the pool's type). Bound by memory: 12,900 rows of 8 heads of 128,
// 106 MB read and written, 18.8 us (5.6 TB/s); eight rows 2.8 us, a launch. The
// stores pass by the cache: with other data in it the same call is 19.3 us, 23.7
// with plain ones, and the attention that follows takes the same time.
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
  const int h = c / (PG_E / 8), e = c % (PG_E / 8) * 8;
  const vh_u32x4 kx = pg_load8(k + i * krow + h * khead + e), vx = pg_load8(v + i * vrow + h * vhead + e);
  __builtin_amdgcn_sched_barrier(0);                    // in flight while the place is looked up
  const int lo = pg_owner(starts, B, i);
  const PgSeq s = pg_seq(starts, lengths, lo, M, N << shift);
  unsigned bad = s.bad;
  const int j = i - s.first, pos = s.len - s.count + j;
  if (!s.bad && j >= 0 && j < s.count && pos >= 0) {   // (a place made possible would be another row's)
    const int page = table[(size_t)lo * N + (pos >> shift)];
    if ((unsigned)page < (unsigned)pages) {
      const size_t to = ((((size_t)page << shift) + (pos & ((1 << shift) - 1))) * H + h) * PG_E + e;
      __builtin_nontemporal_store(kx, (vh_u32x4*)(kp + to));
      __builtin_nontemporal_store(vx, (vh_u32x4*)(vp + to));
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

// What a model's pass over the cache begins with: the tokens' ids, and the rows
// of their learned positions (ids and positions outside their tables clamped
// into them, the ids by the embedding), eight elements a thread. An error where
// a row that is a sequence's has such a one; padded rows may hold anything.
extern "C" __global__ __launch_bounds__(256) void pg_input(const int* __restrict__ tokens,
                                                           const int* __restrict__ positions,
                                                           const unsigned short* __restrict__ wpe, int npos, int D, int V,
                                                           const int* __restrict__ starts,
                                                           const int* __restrict__ lengths, int B, int M, int cap,
                                                           int* __restrict__ tok, unsigned short* __restrict__ rows,
                                                           unsigned* __restrict__ err) {
  const int per = D / 8;
  const long at = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const int i = (int)(at / per), c = (int)(at % per);
  if (i >= M) return;
  const int p = positions[i];
  *(vh_u32x4*)(rows + (size_t)i * D + 8 * c) = ld16(wpe + (size_t)min(max(p, 0), npos - 1) * D + 8 * c);
  if (c) return;
  const int id = tokens[i];
  tok[i] = id;
  const unsigned bad = ((unsigned)p >= (unsigned)npos ? PG_ERR_POSITION : 0u)
                       | ((unsigned)id >= (unsigned)V ? PG_ERR_TOKEN : 0u);
  if (!bad) return;
  const int b = pg_owner(starts, B, i);
  const PgSeq s = pg_seq(starts, lengths, b, M, cap);
  const int j = i - s.first;
  if (j >= 0 && j < s.count && s.len - s.count + j >= 0) pg_raise(err, bad);
}

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
// tail) / 2^LO, each what is left cut off after 11 bits: 24 bits. The two lower
// planes share an accumulator. LO is 11, as the second plane begins there; 25 for
// weights, of which there may be many small ones: a largest of 1, or just above,
// leaves less than 2^15 to the second plane, and those below 2^-14, where the
// first has fp16's fixed step, have bits down to 2^-49 (LO 11: 2^-35).
#if PG_KIND == PG_F32
#define PG_PLANES 3
typedef float pg_q;
#else
#define PG_PLANES 1
typedef unsigned short pg_q;
#endif
#define PG_WEIGHT_LO 25
template <int LO = 11>
__device__ __forceinline__ void pg_split(const float* v, vh_u32x4* f) {
#if PG_KIND == PG_F32
  typedef __fp16 h2 __attribute__((ext_vector_type(2)));
  constexpr float S = (float)(1 << LO);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const h2 h = __builtin_amdgcn_cvt_pkrtz(v[2 * j], v[2 * j + 1]);
    const float r0 = fmaf((float)h[0], -S, v[2 * j] * S);
    const float r1 = fmaf((float)h[1], -S, v[2 * j + 1] * S);
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

// A weighted value from its products with the weights' planes.
__device__ __forceinline__ float pg_weighted(float h, float l) { return fmaf(l, 1.0f / (1 << PG_WEIGHT_LO), h); }

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

// Weights are 2^(score - reference), the reference a running one at or below the
// row's largest score: fp16, which holds the second product's operand, has full
// precision down to 2^-14 only and nothing below 2^-25, so the largest weight is
// 2^PG_ATTN_BIAS and a long tail of small ones keeps its mass down to 2^-40 of it
// (with a largest of 1, positions 2^-25.5 below one lost all of theirs, while the
// sum counted it). pg_wide's may grow by 2^PG_SLACK before it rescales (fp16, 4 x
// 600 after 500 of width 128, slack 4 / 6 / 8: 58.0 / 56.7 / 56.7 us), so its
// largest is 2^9 at first and its tail reaches to 2^-34. bf16 has the range, and
// fp32's planes (pg_split): their weights' exponents stay near 0, where they have
// most bits (with a largest weight of 2^14, 8 x 128 was off by 1.9e-7, not 1.5e-7).
// Sums, weighted values and the parts' maxima are all against the reference, so
// that it cancels.
#define PG_SLACK (PG_KIND == PG_BF16 ? 8 : 6)
#define PG_ATTN_BIAS (PG_KIND == PG_F16 ? 15 : 0)
#define PG_WIDE_BIAS (PG_KIND == PG_F16 ? 15 - PG_SLACK : 0)
// The reference of a largest score bm k2: rounded up where the nearest would
// give a weight that its type cannot hold (scores of 2^24 and more).
template <int BIAS>
__device__ __forceinline__ float pg_reference(float bm, float k2) {
  if constexpr (PG_KIND == PG_BF16) return bm * k2;
  float n = BIAS ? fmaf(bm, k2, -(float)BIAS) : bm * k2;
  if (fmaf(bm, k2, -n) > (PG_KIND == PG_F32 ? 1.0f : (float)BIAS)) n = fmaf(__builtin_fabsf(n), 0x1p-23f, n);
  return n;
}
// log2 of a row's sum of 2^score, from its sum against reference m. (The bias is
// taken out of both first: log2 of a small number has more bits behind the point.)
template <int BIAS>
__device__ __forceinline__ float pg_lse(float m, float sum) {
  return (m + (float)BIAS) + __builtin_amdgcn_logf(__builtin_ldexpf(sum, -BIAS));
}

// Whether a 16-bit value is an infinity or a NaN (its exponent bits all set),
// and the same of a word's two: a unit added to the exponents carries into the
// halves' top bits.
#define PG_EXP (PG_KIND == PG_BF16 ? 0x7f80u : 0x7c00u)
__device__ __forceinline__ bool pg_wild(unsigned short h) { return (h & PG_EXP) == PG_EXP; }
__device__ __forceinline__ unsigned pg_wild2(unsigned x) {
  return ((x & (PG_EXP << 16 | PG_EXP)) + (0x80008000u - (PG_EXP << 16 | PG_EXP))) & 0x80008000u;
}

// Eight values with 0 for those that are not finite.
__device__ __forceinline__ vh_u32x4 pg_tame(vh_u32x4 v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned w = pg_wild2(v[j]);
    v[j] &= ~((w & 0x8000u ? 0xffffu : 0u) | (w >> 31 ? 0xffff0000u : 0u));
  }
  return v;
}
// What pg_tame took out of row s of a head's values (rows of `rowlen`, the
// table's and the pool's as the kernels have them), added to a row's outputs
// that see it: dim `dim` of it.
__device__ __forceinline__ float pg_taken(const unsigned short* __restrict__ vh, size_t rowlen,
                                          const int* __restrict__ tb, int pages, int shift, int s, int dim) {
  const int page = tb[s >> shift];
  const size_t at = (((size_t)((unsigned)page < (unsigned)pages ? page : 0)) << shift) + (s & ((1 << shift) - 1));
  const unsigned short v = vh[at * rowlen + dim];
  return pg_wild(v) ? pg_to_f(v) : 0.0f;
}

// A block makes 16 rows of one (sequence, key head): row x stands for new
// token x / G, query head G h + x % G. Its W waves take every W-th step of
// PG_STEP positions each and combine at the end. Scores are K Q^T, outputs
// V^T P^T, so that a lane holds values of one row (lane % 16) in both, and the
// weights feed the second product from the registers the first left them in:
// the instruction's fold position 8 q + e stands for position 4 q + e (e < 4)
// or 16 + 4 q + e - 4 of 32. Value rows go through LDS and are read transposed
// (ds_read_b64_tr_b16: 16 lanes read four rows of 16 values and get a column
// of four each). The softmax is a running one in powers of two, statistics in
// fp32; weights are rounded to the cache's type for the second product, as
// their values are (fp32 queries: 24 bits in three planes).
//
// A block that has a part of the positions only (pg_work) leaves its rows'
// maxima, sums and weighted values in `ws` for pg_join.
//
// What bounds it: over long contexts the cache's bytes: two tokens of 32 heads
// after 100,003 positions of 8 heads of 128, 818 MB in 158 us (5.15 TB/s, a
// copy's rate), 64 ragged sequences of up to 4000 603 MB in 125 (4.8 TB/s);
// over short ones the chain of dependent loads (lengths, pages, rows: 5.5 us
// with one position, 1.4 us for each further step of a wave). A wave's next
// step is in flight while it uses one: 16 KB, 128 KB a CU at two waves a SIMD
// (three waves a SIMD spill: 134 -> 200 us).
#define PG_STEP (PG_E == 64 ? 64 : 32)
#define PG_VROW (PG_E + 16)                // halves of a value row in LDS: 16 past a multiple of 32 banks
#define PG_WS(rows) ((rows) * (PG_E + 2))  // floats of a tile's part: maxima, sums, rows of E

// How the work is dealt to blocks. A sequence's rows come in tiles of ROWS, its
// positions in steps of STEP; a part is `each` steps of one (sequence, key
// head, tile), `each` such that there are about `target` parts in all (0: one
// part a tile). So parts are of one size whatever the lengths, and a block of
// the grid is a part: the grid holds target + H (M G / ROWS + B) + 64, every
// number of parts that can come out (a multiple of 8 runs), and is dealt to the
// eight XCDs in runs of `run`, which share an L2. A sequence's parts follow
// each other; in each come its tiles from the longest, all heads of a tile, or
// (few tiles, or runs of many) its heads, all tiles of a head, which read the
// same rows. Starts that do not ascend can ask for more parts than there can
// be: those past `limit`, the places of ws, are left out.
struct PgWork {
  PgSeq sq;
  int b, h, R, x0, tile, tiles, part, each, at;   // x0: the tile's first row of R; at: the part's place in ws
};
__device__ __forceinline__ int pg_deal(int block, int run) {       // the block's place: blocks go to XCD block % 8
  const int j = block >> 3;
  const int n = pg_div(j, run);
  return (n * 8 + (block & 7)) * run + j - n * run;
}
template <int ROWS, int STEP>
__device__ __forceinline__ void pg_count(const PgSeq& s, int G, int& tiles, int& steps) {
  tiles = (s.count * G + ROWS - 1) / ROWS;
  steps = max((s.len + STEP - 1) / STEP, 1);
}
// Sums over the lanes up to each.
template <int CTRL, int ROWS>
__device__ __forceinline__ int pg_dpp(int v) {                     // a lane of another row or column, 0 where there is none
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true);
}
__device__ __forceinline__ int pg_scan(int v) {                    // (row_shr 1, 2, 4, 8, then row_bcast 15, 31)
  v += pg_dpp<0x111, 0xF>(v);
  v += pg_dpp<0x112, 0xF>(v);
  v += pg_dpp<0x114, 0xF>(v);
  v += pg_dpp<0x118, 0xF>(v);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}
// The steps of a part: the same in every wave that asks.
template <int ROWS, int STEP>
__device__ __forceinline__ int pg_each(const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M,
                                       int cap, int H, int G, int target, int least) {
  if (target == 0) return 0x7fffffff;
  const int lane = threadIdx.x & 63;
  float w = 0.0f;
  for (int b = lane; b < B; b += 64) {
    int tiles, steps;
    pg_count<ROWS, STEP>(pg_seq(starts, lengths, b, M, cap), G, tiles, steps);
    w += (float)tiles * (float)steps;
  }
  w = wave_red_sum(w);
  return max((int)fminf(w * (float)H / (float)target, 1e9f) + 1, least);
}
// Once a call, by one wave: what is wrong with any sequence.
__device__ __forceinline__ void pg_faults(const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M,
                                          int cap, int most, unsigned* __restrict__ err) {
  unsigned bad = 0u;
  for (int b = threadIdx.x & 63; b < B; b += 64) {
    const PgSeq s = pg_seq(starts, lengths, b, M, cap);
    bad |= s.bad | (s.count > most ? PG_ERR_MOST : 0u);
  }
  if (bad) pg_raise(err, bad);
}
// Block `at`'s part, where `joined` one of all (sequence, head, tile)s of a
// grid of those instead (its parts' first place in ws is then `at`).
template <int ROWS, int STEP>
__device__ __forceinline__ bool pg_work(PgWork& o, int block, int run, bool joined, const int* __restrict__ starts,
                                        const int* __restrict__ lengths, int B, int M, int cap, int H, int G,
                                        int target, int least, int limit, unsigned* __restrict__ err, int most) {
  const int lane = threadIdx.x & 63;
  // A tile a sequence and key head at most, which the program has said: no
  // block has to look through the sequences (one token after 700, 12 heads: 9.7
  // -> 9.2 us), but one behind the tiles, for what is wrong with them.
  if (!joined && target == 0 && most * G <= ROWS) {
    const int at = pg_deal(block, run);
    if (at < B * H) {
      o.b = pg_div(at, H);
      o.h = at - o.b * H;
      o.sq = pg_seq(starts, lengths, o.b, M, cap);
      o.each = 0x7fffffff;
      o.part = o.tile = o.x0 = 0;
      o.tiles = 1;
      o.at = at;
      o.R = o.sq.count * G;
      return o.R > 0;
    }
    if (at == B * H && threadIdx.x < 64) pg_faults(starts, lengths, B, M, cap, most, err);
    return false;
  }
  // Where sequences have several tiles of many rows, all tiles longest first: a
  // CU has few of them, and a long one that starts late is waited for (sequence
  // by sequence / longest first: 16 x 1024 of 12 heads of 64 68 / 50 us, 32 x
  // 700 63 / 57; four tiles a sequence: 6 x up to 512 26.0 / 28.0; 1 x 9000 of 12
  // heads a head's tiles to an XCD 269 / 208, of two of 128 keyed, 4096 after
  // 20,000, 3050 / 900, of eight 1885 / 1850 after 27,001).
  if (ROWS >= 128 && !joined && target == 0 && B <= 64 && most * G >= 5 * ROWS) {
    if (block == 0 && threadIdx.x < 64) pg_faults(starts, lengths, B, M, cap, most, err);
    PgSeq s = {};
    if (lane < B) s = pg_seq(starts, lengths, lane, M, cap);
    const int R = s.count * G, T = (R + ROWS - 1) / ROWS, first = s.len - s.count;
    const int at = pg_deal(block, run), x = pg_div(at, H);
    if (x >= __builtin_amdgcn_readlane(pg_scan(T), 63) || at >= limit) return false;
    auto longer = [&](int n) -> int {                              // the lane's tiles of n steps or more
      const long y = ((long)(n - 1) * STEP - first) * G;           // their last row is y or later
      return n <= 0 || y < 0 ? T : y >= R ? 0 : T - (int)y / ROWS;
    };
    int lo = 0, hi = cap / STEP + 2;                               // more than x tiles have lo steps, not so hi
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__builtin_amdgcn_readlane(pg_scan(longer(mid)), 63) > x) lo = mid; else hi = mid;
    }
    const int a = longer(hi), n = longer(lo) - a, sum = pg_scan(n);
    const int rest = x - __builtin_amdgcn_readlane(pg_scan(a), 63);
    const int l = __builtin_ctzll(__ballot(sum > rest));
    o.b = l;
    o.h = at - x * H;
    o.sq.first = __builtin_amdgcn_readlane(s.first, l);
    o.sq.count = __builtin_amdgcn_readlane(s.count, l);
    o.sq.len = __builtin_amdgcn_readlane(s.len, l);
    o.tiles = __builtin_amdgcn_readlane(T, l);
    o.tile = o.tiles - 1 - __builtin_amdgcn_readlane(a, l) - (rest - __builtin_amdgcn_readlane(sum - n, l));
    o.each = 0x7fffffff;
    o.part = 0;
    o.at = at;
    o.R = o.sq.count * G;
    o.x0 = o.tile * ROWS;
    return true;
  }
  o.each = pg_each<ROWS, STEP>(starts, lengths, B, M, cap, H, G, target, least);
  auto mine = [&](int b, PgSeq& s, int& tiles, int& parts) -> int {
    tiles = parts = 0;
    if (b >= B) return 0;
    s = pg_seq(starts, lengths, b, M, cap);
    int steps;
    pg_count<ROWS, STEP>(s, G, tiles, steps);
    parts = target ? pg_div(steps - 1, o.each) + 1 : 1;
    return tiles * H * (joined ? 1 : parts);
  };
  PgSeq s = {};
  int tiles, parts, n = mine(lane, s, tiles, parts), sum = pg_scan(n);
  int total = __builtin_amdgcn_readlane(sum, 63);
  for (int base = 64; base < B; base += 64) {
    PgSeq u;
    int x, y;
    total += __builtin_amdgcn_readlane(pg_scan(mine(base + lane, u, x, y)), 63);
  }
  if (err && block == 0 && threadIdx.x < 64) pg_faults(starts, lengths, B, M, cap, most, err);
  const int at = joined ? block : pg_deal(block, run);
  if (at >= total || (!joined && at >= limit)) return false;
  int before = 0, places = 0;                                      // in the chunks of 64 sequences already passed
  for (int base = 0; base < B; base += 64) {
    if (base) {
      n = mine(base + lane, s, tiles, parts);
      sum = pg_scan(n);
    }
    const int all = __builtin_amdgcn_readlane(sum, 63);
    if (at < before + all) {
      const int l = __builtin_ctzll(__ballot(before + sum > at));  // the sequence's lane
      o.b = base + l;
      o.sq.first = __builtin_amdgcn_readlane(s.first, l);
      o.sq.count = __builtin_amdgcn_readlane(s.count, l);
      o.sq.len = __builtin_amdgcn_readlane(s.len, l);
      o.tiles = __builtin_amdgcn_readlane(tiles, l);
      const int rest = at - before - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(n, l));
      const bool by_head = o.tiles <= 8;
      o.part = target ? pg_div(rest, o.tiles * H) : 0;
      const int ht = rest - o.part * (o.tiles * H), inner = by_head ? o.tiles : H;
      const int major = pg_div(ht, inner), minor = ht - major * inner;
      o.h = by_head ? major : minor;
      o.tile = o.tiles - 1 - (by_head ? minor : major);            // the longest first
      o.at = at;
      if (joined) {
        const int p = pg_scan(n * parts);
        o.at = places + __builtin_amdgcn_readlane(p, l) - __builtin_amdgcn_readlane(n * parts, l) + rest;
        if (o.at < 0 || o.at + (__builtin_amdgcn_readlane(parts, l) - 1) * (o.tiles * H) >= limit) return false;
      }
      o.R = o.sq.count * G;
      o.x0 = o.tile * ROWS;
      return true;
    }
    before += all;
    if (joined) places += __builtin_amdgcn_readlane(pg_scan(n * parts), 63);
  }
  return false;
}
// A tile's last position (-1: its rows see none), its steps and its parts that have steps.
template <int ROWS, int STEP>
__device__ __forceinline__ void pg_span(const PgWork& w, int G, int& last, int& steps, int& parts) {
  last = w.sq.len - w.sq.count + pg_div(min(w.x0 + ROWS - 1, w.R - 1), G);
  steps = last < 0 ? 0 : last / STEP + 1;
  parts = steps > w.each ? pg_div(steps - 1, w.each) + 1 : 1;
}

// Four consecutive results of a row, rounded to the queries' type.
__device__ __forceinline__ void pg_store4(pg_q* p, const float* v) {
#if PG_KIND == PG_F32
  *(vh_f32x4*)p = vh_f32x4{v[0], v[1], v[2], v[3]};
#else
  const vh_u32x4 w = pg_pack8(pg_f8{v[0], v[1], v[2], v[3], 0.0f, 0.0f, 0.0f, 0.0f});
  *(vh_u32x2*)p = vh_u32x2{w[0], w[1]};
#endif
}

template <int W>
__device__ __forceinline__ void pg_attn_body(
    const pg_q* __restrict__ Q, long qrow, long qhead, const unsigned short* __restrict__ kp,
    const unsigned short* __restrict__ vp, int pages, int shift, const int* __restrict__ table, int N,
    const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M, int H, int G, int target, int least,
    int run, int limit, int most, float scale2, pg_q* __restrict__ out, long orow, long ohead, float* __restrict__ lse,
    float* __restrict__ ws, float* __restrict__ sc, long pitch, unsigned* __restrict__ err) {
  constexpr int KS = PG_E / 32, NG = PG_STEP / 16, NV = PG_STEP * PG_E / 512, DT = PG_E / 16;
  constexpr int VL = PG_E / 8, VR = 64 / VL;                       // lanes of a value row; rows of a wave's load
  __shared__ __attribute__((aligned(16))) unsigned short lv[W][PG_STEP * PG_VROW];
  __shared__ float om[W][2][16];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, q = lane >> 4;
  PgWork wk;
  if (!pg_work<16, PG_STEP>(wk, blockIdx.x, run, false, starts, lengths, B, M, N << shift, H, G, target, least, limit,
                            err, most))
    return;
  int last, steps, parts;
  pg_span<16, PG_STEP>(wk, G, last, steps, parts);
  if (wk.part >= parts) return;
  const PgSeq sq = wk.sq;
  const int R = wk.R, x0 = wk.x0, h = wk.h;
  const int t0 = min(wk.part * wk.each, steps), t1 = wk.each < steps - t0 ? t0 + wk.each : steps;
  unsigned bad = 0;
  const int x = min(x0 + r, R - 1), tok = pg_div(x, G), head = h * G + x - tok * G;
  const bool live = x0 + r < R;
  const int lim = sq.len - sq.count + tok;                         // this lane's last position
  const int first = sq.len - sq.count + pg_div(x0, G);                    // the first row's
  const pg_q* qp = Q + (sq.first + tok) * qrow + head * qhead;
  const size_t rowlen = (size_t)H * PG_E;
  const int* tb = table + (size_t)wk.b * N;
  const unsigned short *kh = kp + h * PG_E + 8 * q, *vh = vp + h * PG_E + lane % VL * 8;
  // the page of a step's positions, one a lane: looked up a step ahead of its
  // rows, and looked at only then (a wait for it would be one for the rows
  // asked for before it)
  auto look = [&](int t) { return tb[min(t * PG_STEP + lane % PG_STEP, last) >> shift]; };
  vh_u32x4 kr[NG][KS], vr[NV];
  auto load = [&](int t, int page) {
    const bool in = (unsigned)page < (unsigned)pages;
    if (!in) bad = PG_ERR_PAGE;
    const unsigned rw = ((unsigned)(in ? page : 0) << shift)
                        + (unsigned)(min(t * PG_STEP + lane % PG_STEP, last) & ((1 << shift) - 1));
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const unsigned short* p = kh + (unsigned)__shfl((int)rw, 16 * i + r, 64) * rowlen;
#pragma unroll
      for (int k = 0; k < KS; ++k) kr[i][k] = ld16(p + 32 * k);
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) vr[n] = ld16(vh + (unsigned)__shfl((int)rw, n * VR + lane / VL, 64) * rowlen);
  };
  float o[DT][4] = {};
  float m2 = -INFINITY, sum = 0.0f;
  unsigned short* V = lv[wave];
  int page = 0;
  if (t0 + wave < t1) page = look(t0 + wave);
  PgQuery qf;
  pg_query(qf, qp, q, scale2);
  if (t0 + wave < t1) {
    load(t0 + wave, page);
    page = look(min(t0 + wave + W, t1 - 1));
  }
  for (int t = t0 + wave; t < t1; t += W) {
    const int p0 = t * PG_STEP;
    float s[NG][4];
#pragma unroll
    for (int i = 0; i < NG; ++i) pg_scores(kr[i], qf, qp, lane, s[i]);
    const bool seen = p0 + PG_STEP - 1 > first;                    // not the whole step by every row
    // values past the last position are 0; ones that are not finite are left
    // out of the product where a row may not see their position, or a plane of
    // its weight may be 0: 0 * inf ...
    bool wild = false;
    if (p0 + PG_STEP - 1 > last) {
#pragma unroll
      for (int n = 0; n < NV; ++n)
        if (p0 + n * VR + lane / VL > last) vr[n] = vh_u32x4{0u, 0u, 0u, 0u};
    }
    if (seen || PG_KIND == PG_F32) {
      unsigned any = 0u;
#pragma unroll
      for (int n = 0; n < NV; ++n) any |= pg_wild2(vr[n][0]) | pg_wild2(vr[n][1]) | pg_wild2(vr[n][2]) | pg_wild2(vr[n][3]);
      wild = __any(any != 0u);
      if (wild) {
#pragma unroll
        for (int n = 0; n < NV; ++n) vr[n] = pg_tame(vr[n]);
      }
    }
    pg_wave_sync();                                                // the step before is read
#pragma unroll
    for (int n = 0; n < NV; ++n) *(vh_u32x4*)(V + (n * VR + lane / VL) * PG_VROW + lane % VL * 8) = vr[n];
    pg_wave_sync();
    if (t + W < t1) {
      load(t + W, page);
      page = look(min(t + 2 * W, t1 - 1));
    }
    if (seen) {
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = p0 + 16 * i + 4 * q + j <= lim ? s[i][j] : -INFINITY;
    }
    if (sc && live) {                                              // for pg_given, in powers of 2
      float* to = sc + ((long)(sq.first + tok) * (H * G) + head) * pitch + p0 + 4 * q;
#pragma unroll
      for (int i = 0; i < NG; ++i)
        *(vh_f32x4*)(to + 16 * i) = vh_f32x4{s[i][0] * qf.k2, s[i][1] * qf.k2, s[i][2] * qf.k2, s[i][3] * qf.k2};
    }
    float bm = s[0][0];
#pragma unroll
    for (int n = 1; n < 4 * NG; ++n) bm = fmaxf(bm, s[n >> 2][n & 3]);
    bm = vh_pair32(vh_pair16(bm, op_max), op_max);
    const float n2 = fmaxf(m2, pg_reference<PG_ATTN_BIAS>(bm, qf.k2));
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
      pg_split<PG_WEIGHT_LO>(w, pf[k]);
    }
    sum = fmaf(sum, c, ts);
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds4;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      vh_f32x4 th = {0.0f, 0.0f, 0.0f, 0.0f};
#if PG_KIND == PG_F32
      vh_f32x4 tw = th;
#endif
#pragma unroll
      for (int k = 0; k < NG / 2; ++k) {
        unsigned short* vb = V + (32 * k + 4 * q + r / 4) * PG_VROW + 16 * d + 4 * (r & 3);
        const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)vb);
        const s4 e = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(vb + 16 * PG_VROW));
        const vh_u32x4 vf = __builtin_bit_cast(vh_u32x4, __builtin_shufflevector(a, e, 0, 1, 2, 3, 4, 5, 6, 7));
        th = pg_mfma(vf, pf[k][0], th);
#if PG_KIND == PG_F32
        tw = pg_mfma(vf, pf[k][1], tw);
        tw = pg_mfma(vf, pf[k][2], tw);
#endif
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#if PG_KIND == PG_F32
        o[d][j] = fmaf(o[d][j], c, pg_weighted(th[j], tw[j]));
#else
        o[d][j] = fmaf(o[d][j], c, th[j]);
#endif
      }
    }
    if (wild) {                                                    // ... and go to the rows that see them
#pragma nounroll
      for (int s = p0; s <= min(p0 + PG_STEP - 1, last); ++s)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float v = pg_taken(vp + h * PG_E, rowlen, tb, pages, shift, s, 16 * d + 4 * q + j);
            o[d][j] += s <= lim ? v : 0.0f;
          }
    }
  }
  if (__any(bad != 0) && lane == 0) pg_raise(err, PG_ERR_PAGE);
  sum = vh_pair32(vh_pair16(sum, op_sum), op_sum);
  // each wave's maximum, sum and output, rescaled to the common maximum and
  // added in wave order; wave w then makes every fourth dim tile
  float* ow = (float*)lv;                                          // [wave][dim tile][j][lane]
  static_assert(sizeof(lv) >= W * DT * 4 * 64 * 4, "the value tiles hold the waves' outputs");
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
  for (int w = 1; w < W; ++w) m = fmaxf(m, om[w][0][r]);
  sum = 0.0f;
  float f[W];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    f[w] = om[w][0][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(om[w][0][r] - m);   // no score: 0
    sum = fmaf(om[w][1][r], f[w], sum);
  }
  if (!live) return;
  const bool whole = parts == 1;
  pg_q* op = out + (sq.first + tok) * orow + head * ohead;
  float* wp = ws + (size_t)wk.at * PG_WS(16);
#pragma unroll
  for (int d = wave; d < DT; d += W) {
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = fmaf(ow[((w * DT + d) * 4 + j) * 64 + lane], f[w], v[j]);
    if (whole) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = lim < 0 ? 0.0f : v[j] / sum;
      pg_store4(op + 16 * d + 4 * q, v);
    } else {
      *(vh_f32x4*)(wp + 32 + r * PG_E + 16 * d + 4 * q) = vh_f32x4{v[0], v[1], v[2], v[3]};
    }
  }
  if (wave == 0 && q == 0) {
    if (!whole) {
      wp[r] = m;
      wp[16 + r] = sum;
    } else if (lse) {
      // log2 of the row's sum of 2^score: +inf for a row that sees nothing, so
      // that all its weights are 0
      lse[(size_t)(sq.first + tok) * (H * G) + head] = lim < 0 ? INFINITY : pg_lse<PG_ATTN_BIAS>(m, sum);
    }
  }
}

#define PG_ATTN(name, waves) \
  extern "C" __global__ __launch_bounds__(64 * waves, 2) void name( \
      const pg_q* __restrict__ Q, long qrow, long qhead, const unsigned short* __restrict__ kp, \
      const unsigned short* __restrict__ vp, int pages, int shift, const int* __restrict__ table, int N, \
      const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M, int H, int G, int target, int least, \
      int run, int limit, int most, float scale2, pg_q* __restrict__ out, long orow, long ohead, float* __restrict__ lse, \
      float* __restrict__ ws, float* __restrict__ sc, long pitch, unsigned* __restrict__ err) { \
    pg_attn_body<waves>(Q, qrow, qhead, kp, vp, pages, shift, table, N, starts, lengths, B, M, H, \
                        G, target, least, run, limit, most, scale2, out, orow, ohead, lse, ws, sc, pitch, err); \
  }
PG_ATTN(pg_attn2, 2)
PG_ATTN(pg_attn, 4)
PG_ATTN(pg_attn8, 8)

// Waits for loads whose registers a loop reads: left to the first use inside it,
// the wait is for all loads issued since as well, each time round (pg_wide, six
// chunks of up to 512 tokens: 27.8 -> 25.8 us).
template <int N>
__device__ __forceinline__ void pg_here(vh_u32x4 (&f)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) asm volatile("" : "+v"(f[k]));
}

// Attention of many rows. A block makes 128 rows of one (sequence, key head),
// or 256 (W: its waves, 32 rows each), over steps of 64 positions that its
// waves share: key and value rows lie in LDS (double-buffered; the loads of the
// step after next are in flight while one is used). Products in tiles of
// 32 x 32 x 16: lane 32 g + r holds row r, fold positions 8 g .. + 7 of an
// operand; column r, rows 8 (i / 4) + 4 g + i % 4 of the result, i < 16. As in
// pg_attn, scores are K Q^T, outputs V^T P^T, and the weights feed the second
// product from the registers they are in: fold position 8 g + e stands for
// position 4 g + e (e < 4) or 8 + 4 g + e - 4 of 16. The weighted values
// accumulate in the matrix cores' own registers; they are rescaled only when a
// row's reference has grown by more than PG_SLACK since (weights up to 2^PG_SLACK
// times the largest are exact in the sums and rounded as finely). fp32 queries and weights go in
// three planes, 32 positions at a time, and each 32 positions' weighted values
// are summed on their own and added in fp32, so that no sum is a chain over all
// positions; they take this kernel at width 64 only (at 128 their planes leave
// one block a CU, no faster than pg_attn: 32 x 768 1169 us against 1171).
//
// What bounds it at width 128: a wave's step takes 1024 cycles of the matrix
// cores, 1000 to 1300 of the vector units (the softmax) and, as each operand
// read from LDS serves 32 rows, 360 of the CU's LDS, 1440 for its four SIMDs.
// Two blocks of four waves drift into step and do each in turn (4700 cycles for
// a step of both; 4096 tokens after 27,001, 1.95 TFLOP in 2050-2100 us). In
// blocks of eight, two groups of four waves, one of each on a SIMD, are kept
// apart by barriers: while one has the matrix cores, the other has the vector
// units. The same 4096 tokens in 1800 us (1085 TFLOP/s, 80% of a large library
// product's rate). At width 64 the softmax on the vector units (about 1400
// cycles a step against 512), and for short chunks the blocks' starts and ends
// (4 us): six chunks of up to 512 tokens 23 us (240 TFLOP/s).
#if PG_KIND != PG_F32 || PG_E == 64
#define PG_WROW (PG_E + 32)                // halves of a value row in LDS: 64 bytes past a multiple of all banks
typedef float pg_f16v __attribute__((ext_vector_type(16)));
__device__ __forceinline__ pg_f16v pg_mfma32(vh_u32x4 a, vh_u32x4 b, pg_f16v c) {
#if PG_KIND == PG_BF16
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pg_b8, a), __builtin_bit_cast(pg_b8, b), c, 0, 0, 0);
#else
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vh_h8, a), __builtin_bit_cast(vh_h8, b), c, 0, 0, 0);
#endif
}

template <int W>
__device__ __forceinline__ void pg_wide_body(
    const pg_q* __restrict__ Q, long qrow, long qhead, const unsigned short* __restrict__ kp,
    const unsigned short* __restrict__ vp, int pages, int shift, const int* __restrict__ table, int N,
    const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M, int H, int G, int target, int least,
    int run, int limit, int most, float scale2, pg_q* __restrict__ out, long orow, long ohead, float* __restrict__ lse,
    float* __restrict__ ws, unsigned* __restrict__ err) {
  constexpr int KS = PG_E / 16, DT = PG_E / 32, CH = PG_E / 8;     // k-steps, dim tiles, 16-byte pieces of a row
  constexpr int TILE = 32 * W, RS = 64 * W / CH, NL = 64 / RS;     // rows; a thread's rows of a step apart, its pieces
  __shared__ __attribute__((aligned(16))) vh_u32x4 lk[2][64 * (CH + 1)];
  __shared__ __attribute__((aligned(16))) unsigned short lv[2][64 * PG_WROW];
  __shared__ int lwild[2];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 31, g = lane >> 5;
  PgWork wk;
  if (!pg_work<TILE, 64>(wk, blockIdx.x, run, false, starts, lengths, B, M, N << shift, H, G, target, least, limit, err,
                        most))
    return;
  int last, steps, parts;
  pg_span<TILE, 64>(wk, G, last, steps, parts);
  if (wk.part >= parts) return;
  const PgSeq sq = wk.sq;
  const int R = wk.R, x0 = wk.x0 + 32 * wave, h = wk.h, new0 = sq.len - sq.count;
  const int t0 = min(wk.part * wk.each, steps), t1 = wk.each < steps - t0 ? t0 + wk.each : steps;
  const int x = min(x0 + r, R - 1), tok = pg_div(x, G), head = h * G + x - tok * G;
  const bool live = x0 + r < R;
  const int lim = new0 + tok;                                      // this lane's last position
  const int bfirst = new0 + pg_div(wk.x0, G);                             // the block's first row's
  const int wfirst = new0 + pg_div(min(x0, R - 1), G), wlast = new0 + pg_div(min(x0 + 31, R - 1), G);
  unsigned bad = 0;
  const pg_q* qp = Q + (sq.first + tok) * qrow + head * qhead;
#if PG_KIND == PG_F32
  vh_u32x4 qf[KS][3];
  float k2;                                                        // as in pg_query
  {
    float v[KS][8], mx = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const vh_f32x4 a = *(const vh_f32x4*)(qp + 16 * k + 8 * g), c = *(const vh_f32x4*)(qp + 16 * k + 8 * g + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[k][j] = a[j];
        v[k][4 + j] = c[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) mx = fmaxf(mx, __builtin_fabsf(v[k][j]));
    }
    mx = vh_pair32(mx, op_max);
    int e = 0;
    if (mx > 0.0f && mx < INFINITY) e = max(__builtin_amdgcn_frexp_expf(mx), -100);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] = __builtin_ldexpf(v[k][j], -e);
      pg_split(v[k], qf[k]);
    }
    k2 = __builtin_ldexpf(scale2, e);
  }
#else
  vh_u32x4 qf[KS];
#pragma unroll
  for (int k = 0; k < KS; ++k) qf[k] = ld16(qp + 16 * k + 8 * g);
#endif
  // staging: thread t takes piece t % CH of rows t / CH + RS n
  const size_t rowlen = (size_t)H * PG_E;
  const int* tb = table + (size_t)wk.b * N;
  const int c8 = tid % CH, r8 = tid / CH;
  const unsigned short *kh = kp + h * PG_E + 8 * c8, *vh = vp + h * PG_E + 8 * c8;
  int page[NL];
  auto look = [&](int t) {                                         // as in pg_attn
#pragma unroll
    for (int n = 0; n < NL; ++n) page[n] = tb[min(64 * t + r8 + RS * n, last) >> shift];
  };
  vh_u32x4 kr[NL], vr[NL];
  unsigned at[NL];
  auto where = [&](int t) {
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const bool in = (unsigned)page[n] < (unsigned)pages;
      if (!in) bad = PG_ERR_PAGE;
      at[n] = ((unsigned)(in ? page[n] : 0) << shift) + (unsigned)(min(64 * t + r8 + RS * n, last) & ((1 << shift) - 1));
    }
  };
  auto load_k = [&]() {
#pragma unroll
    for (int n = 0; n < NL; ++n) kr[n] = ld16(kh + (size_t)at[n] * (unsigned)rowlen);
  };
  auto load_v = [&]() {
#pragma unroll
    for (int n = 0; n < NL; ++n) vr[n] = ld16(vh + (size_t)at[n] * (unsigned)rowlen);
  };
  // Key rows are 16 bytes past a multiple of all banks apart, so that a column
  // of their pieces falls on all of them.
  auto put_k = [&](int t) {
#pragma unroll
    for (int n = 0; n < NL; ++n) lk[t & 1][(r8 + RS * n) * (CH + 1) + c8] = kr[n];
  };
  // Values past the last position are 0, and where some row sees a step in part
  // so are those that are not finite (0 * inf); that there are such is noted.
  auto put_v = [&](int t) {
    if (64 * t + 63 > last) {
#pragma unroll
      for (int n = 0; n < NL; ++n)
        if (64 * t + r8 + RS * n > last) vr[n] = vh_u32x4{0u, 0u, 0u, 0u};
      asm volatile("" ::: "memory");                               // kept a branch
    }
    if (PG_KIND == PG_F32 || 64 * t + 63 > bfirst) {               // (fp32: a plane of a weight may be 0)
      unsigned any = 0u;
#pragma unroll
      for (int n = 0; n < NL; ++n) any |= pg_wild2(vr[n][0]) | pg_wild2(vr[n][1]) | pg_wild2(vr[n][2]) | pg_wild2(vr[n][3]);
      if (any) {
        lwild[t & 1] = t + 1;
#pragma unroll
        for (int n = 0; n < NL; ++n) vr[n] = pg_tame(vr[n]);
      }
    }
#pragma unroll
    for (int n = 0; n < NL; ++n) *(vh_u32x4*)(lv[t & 1] + (r8 + RS * n) * PG_WROW + 8 * c8) = vr[n];
  };
  pg_f16v o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[d][j] = 0.0f;
  float m2 = -INFINITY, sum = 0.0f;
  if (tid < 2) lwild[tid] = 0;
  vh_lds_sync();                                                   // noted as none before a step may be noted
  typedef short s4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s4 lds4;
  auto value = [&](int t, int i, int k, int d) {
    const unsigned short* vb = lv[t & 1] + (32 * i + 16 * k + 4 * g + ((lane & 15) >> 2)) * PG_WROW + 32 * d
                               + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)vb);
    const s4 e = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(vb + 8 * PG_WROW));
    return __builtin_bit_cast(vh_u32x4, __builtin_shufflevector(a, e, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto sees = [&](int t) { return x0 < R && 64 * t <= wlast; };    // whether the wave has a row that sees step t
  // the values of a step that are not finite, to the rows that see them
  auto add_wild = [&](int t) {
#pragma nounroll
    for (int s = 64 * t; s <= min(64 * t + 63, last); ++s)
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float v = pg_taken(vp + h * PG_E, rowlen, tb, pages, shift, s, 32 * d + 8 * (j >> 2) + 4 * g + (j & 3));
          o[d][j] += s <= lim ? v : 0.0f;
        }
  };
#if PG_KIND != PG_F32
  pg_f16v s[2];
  vh_u32x4 pf[2][2];
  auto scores = [&](int t) {
    const vh_u32x4* K = lk[t & 1];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) s[i][j] = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) s[i] = pg_mfma32(K[(32 * i + r) * (CH + 1) + 2 * k + g], qf[k], s[i]);
  };
  auto soften = [&](int t) {
    const int p0 = 64 * t;
    if (p0 + 63 > wfirst) {                                        // not the whole step by every row
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[i][j] = p0 + 32 * i + 8 * (j >> 2) + 4 * g + (j & 3) <= lim ? s[i][j] : -INFINITY;
    }
    // The largest as a whole number of the same bits, right wherever one is
    // positive (fmaxf asks for a canonical form of every score first: 48
    // operations more); where none is, in floats.
    int bi = 0x80000000;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float a = s[0][j], e = s[1][j];                        // (a bit_cast of a vector's element takes its first)
      bi = max(max(bi, __builtin_bit_cast(int, a)), __builtin_bit_cast(int, e));
    }
    float bm = __builtin_bit_cast(float, bi);
    if (__any(bi < 0)) {
      bm = fmaxf(s[0][0], s[1][0]);
#pragma unroll
      for (int j = 1; j < 16; ++j) bm = fmaxf(bm, fmaxf(s[0][j], s[1][j]));
    }
    bm = vh_pair32(bm, op_max);
    // (a first one too: m2 is -inf; what pg_reference may add to it counts, and is added where it is taken)
    const float n2 = fmaf(bm, scale2, -(float)PG_WIDE_BIAS);
    if (__any(fmaf(__builtin_fabsf(n2), 0x1p-23f, n2 - m2) > (float)PG_SLACK)) {
      const float m = fmaxf(m2, pg_reference<PG_WIDE_BIAS>(bm, scale2));
      const float c = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m2 - m);
      m2 = m;
      sum *= c;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[d][j] *= c;
    }
    const float ref = m2 == -INFINITY ? 0.0f : m2;                 // no score above -inf yet: all weights 0
    float ts[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(fmaf(s[i][8 * k + j], scale2, -ref));
        ts[2 * i + k] = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
        pf[i][k] = pg_pack8(pg_f8{w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]});
      }
    sum += (ts[0] + ts[1]) + (ts[2] + ts[3]);
  };
  auto gather = [&](int t) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = pg_mfma32(value(t, i, k, d), pf[i][k], o[d]);
  };
#endif
  if (t0 < t1) {
    look(t0);
    where(t0);
    load_k();
    load_v();
    look(min(t0 + 1, t1 - 1));
  }
#if PG_KIND == PG_F32
#pragma unroll
  for (int k = 0; k < KS; ++k) pg_here(qf[k]);
#else
  pg_here(qf);
#endif
#if PG_KIND != PG_F32
  // Two groups of four waves take turns. In its turn at the products a wave
  // also puts its share of the next step's keys and of this one's values into
  // LDS, where nobody reads them before both groups have done so.
  if constexpr (W == 8) {
    unsigned av[NL];                     // rows of the values to be asked for next: the keys' of a step before
    auto place = [&](int t) {
#pragma unroll
      for (int n = 0; n < NL; ++n) av[n] = at[n];
      if (t < t1) {
        where(t);
        look(min(t + 1, t1 - 1));
      }
    };
    auto ask = [&](int t) {              // the values of step t, the keys of the next
      if (t >= t1) return;
#pragma unroll
      for (int n = 0; n < NL; ++n) vr[n] = ld16(vh + (size_t)av[n] * (unsigned)rowlen);
      if (t + 1 < t1) load_k();
    };
    auto stage = [&](int t) {
      if (t + 1 < t1) put_k(t + 1);
      put_v(t);
    };
    if (t0 < t1) {
      put_k(t0);
      place(t0 + 1);
      if (t0 + 1 < t1) load_k();         // (its values are there)
      place(t0 + 2);
    }
    vh_lds_sync();
    if (wave >= 4) vh_lds_sync();        // half a step behind
    if (t0 < t1) {
      stage(t0);
      if (sees(t0)) scores(t0);
      vh_lds_sync();
    }
    for (int t = t0; t < t1; ++t) {
      ask(t + 1);
      if (sees(t)) soften(t);
      place(t + 3);
      vh_lds_sync();
      __builtin_amdgcn_s_setprio(1);     // (1935 us without)
      if (t + 1 < t1) stage(t + 1);
      const int noted = lwild[t & 1];
      if (sees(t)) {
        gather(t);
        // LDS reads run ahead of the products that take them (1920 us as the compiler has it)
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
        for (int n = 0; n < 13; ++n) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 3, 0);
        if (noted == t + 1) add_wild(t);
      }
      if (t + 1 < t1 && sees(t + 1)) {
        scores(t + 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int n = 0; n < 12; ++n) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
      }
      __builtin_amdgcn_s_setprio(0);
      if (t + 1 < t1) vh_lds_sync();
    }
    if (wave < 4) vh_lds_sync();         // as many barriers as the other group
  }
#endif
  if constexpr (W == 4) {
    if (t0 < t1) {
      put_k(t0);
      put_v(t0);
      if (t0 + 1 < t1) {
        where(t0 + 1);
        load_k();
        load_v();
        look(min(t0 + 2, t1 - 1));
      }
    }
    for (int t = t0; t < t1; ++t) {
      vh_lds_sync();                       // step t is staged; the other buffer's step is read
      if (t + 1 < t1) {
        put_k(t + 1);
        put_v(t + 1);
        if (t + 2 < t1) {
          where(t + 2);
          load_k();
          load_v();
          look(min(t + 3, t1 - 1));
        }
      }
      if (!sees(t)) continue;
      const int noted = lwild[t & 1];
#if PG_KIND != PG_F32
      scores(t);
      soften(t);
      gather(t);
#else
      const int p0 = 64 * t;
      const bool seen = p0 + 63 > wfirst;
      const vh_u32x4* K = lk[t & 1];
#pragma nounroll
      for (int i = 0; i < 2; ++i) {
        pg_f16v hi, lo;
#pragma unroll
        for (int j = 0; j < 16; ++j) hi[j] = lo[j] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const vh_u32x4 kf = K[(32 * i + r) * (CH + 1) + 2 * k + g];
          hi = pg_mfma32(kf, qf[k][0], hi);
          lo = pg_mfma32(kf, qf[k][1], lo);
          lo = pg_mfma32(kf, qf[k][2], lo);
        }
        float s[16], fin = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          s[j] = vh_hilo(hi[j], lo[j]);
          fin = fmaf(hi[j], 0.0f, fin);
        }
        if (__any(fin != fin)) {                                     // as in pg_scores
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float acc = 0.0f;
#pragma nounroll
            for (int c = 0; c < CH; ++c) {
              float kv[8];
              unpack8(K[(32 * i + 8 * (j >> 2) + 4 * g + (j & 3)) * (CH + 1) + c], kv);
#pragma unroll
              for (int d = 0; d < 8; ++d) acc = fmaf(qp[8 * c + d], kv[d], acc);
            }
            if (!(__builtin_fabsf(hi[j]) < INFINITY)) s[j] = acc;
          }
        }
        if (seen) {
#pragma unroll
          for (int j = 0; j < 16; ++j) s[j] = p0 + 32 * i + 8 * (j >> 2) + 4 * g + (j & 3) <= lim ? s[j] : -INFINITY;
        }
        float bm = s[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) bm = fmaxf(bm, s[j]);
        bm = vh_pair32(bm, op_max);
        const float n2 = fmaxf(m2, pg_reference<PG_WIDE_BIAS>(bm, k2));
        const float ref = n2 == -INFINITY ? 0.0f : n2;               // no score above -inf yet: all weights 0
        const float c = __builtin_amdgcn_exp2f(m2 - ref);
        m2 = n2;
        vh_u32x4 pf[2][3];
        float ts[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(fmaf(s[8 * k + j], k2, -ref));
          ts[k] = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
          pg_split<PG_WEIGHT_LO>(w, pf[k]);
        }
        sum = fmaf(sum, c, ts[0] + ts[1]);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          pg_f16v th, tw;
#pragma unroll
          for (int j = 0; j < 16; ++j) th[j] = tw[j] = 0.0f;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const vh_u32x4 vf = value(t, i, k, d);
            th = pg_mfma32(vf, pf[k][0], th);
            tw = pg_mfma32(vf, pf[k][1], tw);
            tw = pg_mfma32(vf, pf[k][2], tw);
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) o[d][j] = fmaf(o[d][j], c, pg_weighted(th[j], tw[j]));
        }
      }
#endif
      if (noted == t + 1) add_wild(t);
    }
  }
  if (__any(bad != 0) && lane == 0) pg_raise(err, PG_ERR_PAGE);
  if (!live) return;
  sum = vh_pair32(sum, op_sum);
  const bool whole = W == 8 || parts == 1;                         // (eight waves are not launched for parts)
  const float inv = 1.0f / sum;        // (exact enough for results of 16 bits: a division each was 0.5 us of a block's end)
  pg_q* op = out + (sq.first + tok) * orow + head * ohead;
  float* wp = ws + (size_t)wk.at * PG_WS(TILE);
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = !whole ? o[d][4 * i + j] : lim < 0 ? 0.0f : PG_KIND == PG_F32 ? o[d][4 * i + j] / sum : o[d][4 * i + j] * inv;
      if (whole) pg_store4(op + 32 * d + 8 * i + 4 * g, v);
      else *(vh_f32x4*)(wp + 2 * TILE + (32 * wave + r) * PG_E + 32 * d + 8 * i + 4 * g) = vh_f32x4{v[0], v[1], v[2], v[3]};
    }
  if (g == 0) {
    if (!whole) {
      wp[32 * wave + r] = m2;
      wp[TILE + 32 * wave + r] = sum;
    } else if (lse) {
      lse[(size_t)(sq.first + tok) * (H * G) + head] = lim < 0 ? INFINITY : pg_lse<PG_WIDE_BIAS>(m2, sum);
    }
  }
}
#define PG_WIDE(name, waves)                                                                                       \
  extern "C" __global__ __launch_bounds__(64 * waves, 2) void name(                                                \
      const pg_q* __restrict__ Q, long qrow, long qhead, const unsigned short* __restrict__ kp,                    \
      const unsigned short* __restrict__ vp, int pages, int shift, const int* __restrict__ table, int N,           \
      const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M, int H, int G, int target,     \
      int least, int run, int limit, int most, float scale2, pg_q* __restrict__ out, long orow, long ohead,        \
      float* __restrict__ lse, float* __restrict__ ws, unsigned* __restrict__ err) {                               \
    pg_wide_body<waves>(Q, qrow, qhead, kp, vp, pages, shift, table, N, starts, lengths, B, M, H, G, target,       \
                        least, run, limit, most, scale2, out, orow, ohead, lse, ws, err);                          \
  }
PG_WIDE(pg_wide, 4)
#if PG_KIND != PG_F32 && PG_E == 128
PG_WIDE(pg_wide8, 8)
#endif
#endif

// The parts of a tile of ROWS rows put together: a block of 512 threads makes
// up to `each_rows` (1, 4 or 16) rows of it, E / 4 lanes a row; where there are
// fewer rows their parts are dealt to the lane groups left, whose results are
// added in order. What bounds it is the chain of loads (128 parts of four rows,
// one group a row: 60 us; four rows a block, four groups a row: 11.7; a row a
// block: 8.5).
template <int ROWS, int STEP>
__device__ __forceinline__ void pg_join_body(const int* __restrict__ starts, const int* __restrict__ lengths, int B,
                                             int cap, int M, int H, int G, int target, int least, int run, int limit,
                                             int each_rows, const float* __restrict__ ws, pg_q* __restrict__ out, long orow,
                                             long ohead, float* __restrict__ lse) {
  constexpr int LR = PG_E / 4, NGR = 512 / LR;
  __shared__ float jm[NGR], js[NGR];
  __shared__ vh_f32x4 jv[512];
  const int tid = threadIdx.x, c = tid % LR, grp = tid / LR, cut = ROWS / each_rows;
  const int tile = pg_div(blockIdx.x, cut), y0 = ((int)blockIdx.x - tile * cut) * each_rows;
  PgWork wk;                                                       // grid: H (M G / ROWS + B) tiles or more
  if (!pg_work<ROWS, STEP>(wk, tile, run, true, starts, lengths, B, M, cap, H, G, target, least, limit,
                           nullptr, 0))
    return;
  int last, steps, parts;
  pg_span<ROWS, STEP>(wk, G, last, steps, parts);
  const int n = min(each_rows, wk.R - wk.x0 - y0);                 // rows
  if (parts == 1 || n <= 0) return;
  const int n2 = n == 1 ? 1 : 1 << (32 - __builtin_clz(n - 1)), slices = NGR / n2;
  const int y = y0 + grp % n2, slice = grp / n2;
  const size_t next = (size_t)H * wk.tiles * PG_WS(ROWS);          // the tile's next part
  const float* wp = ws + (size_t)wk.at * PG_WS(ROWS);
  float m = -INFINITY, sum = 0.0f;
  vh_f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (grp % n2 < n) {
    for (int p0 = slice; p0 < parts; p0 += 8 * slices) {
      float pm[8], ps[8];
      vh_f32x4 pv[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {                                // past the last: the last again, not counted
        const int p = p0 + u * slices;
        const float* w = wp + min(p, parts - 1) * next;
        pm[u] = p < parts ? w[y] : -INFINITY;
        ps[u] = w[ROWS + y];
        pv[u] = *(const vh_f32x4*)(w + 2 * ROWS + y * PG_E + 4 * c);
      }
      float mm = m;
#pragma unroll
      for (int u = 0; u < 8; ++u) mm = fmaxf(mm, pm[u]);
      const float old = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mm);       // no score: 0
      m = mm;
      sum *= old;
      v *= old;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        // a part without a score, or far below the largest, has no weight; a NaN in it stays one (0 * NaN)
        const float f = pm[u] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(pm[u] - mm);
        if (p0 + u * slices < parts) {
          sum = fmaf(ps[u], f, sum);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = fmaf(pv[u][j], f, v[j]);
        }
      }
    }
  }
  if (slices > 1) {
    if (c == 0) {
      jm[grp] = m;
      js[grp] = sum;
    }
    jv[tid] = v;
    __syncthreads();
    if (slice > 0) return;
    float mm = m;
    for (int k = 1; k < slices; ++k) mm = fmaxf(mm, jm[grp + k * n2]);
    const float old = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mm);
    sum *= old;
    v *= old;
    for (int k = 1; k < slices; ++k) {
      const float km = jm[grp + k * n2], ks = js[grp + k * n2];
      const float f = km == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(km - mm);
      sum = fmaf(ks, f, sum);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = fmaf(jv[tid + k * n2 * LR][j], f, v[j]);
    }
    m = mm;
  }
  if (grp % n2 >= n || slice > 0) return;
  const int x = wk.x0 + y, tok = pg_div(x, G), head = wk.h * G + x - tok * G, lim = wk.sq.len - wk.sq.count + tok;
  float w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = lim < 0 ? 0.0f : v[j] / sum;
  pg_store4(out + (wk.sq.first + tok) * orow + head * ohead + 4 * c, w);
  constexpr int BIAS = ROWS == 16 ? PG_ATTN_BIAS : PG_WIDE_BIAS;
  if (lse && c == 0) lse[(size_t)(wk.sq.first + tok) * (H * G) + head] = lim < 0 ? INFINITY : pg_lse<BIAS>(m, sum);
}
#define PG_JOIN(name, rows, step)                                                                                  \
  extern "C" __global__ __launch_bounds__(512) void name(                                                          \
      const int* __restrict__ starts, const int* __restrict__ lengths, int B, int cap, int M, int H, int G,        \
      int target, int least, int run, int limit, int each_rows, const float* __restrict__ ws,                      \
      pg_q* __restrict__ out, long orow, long ohead, float* __restrict__ lse) {                                    \
    pg_join_body<rows, step>(starts, lengths, B, cap, M, H, G, target, least, run, limit, each_rows, ws, out, orow, \
                             ohead, lse);                                                                          \
  }
PG_JOIN(pg_join, 16, PG_STEP)
#if PG_KIND != PG_F32 || PG_E == 64
PG_JOIN(pg_wide_join, 128, 64)
#endif

// ---------------------------------------------------------------- weights
// out[b, h, s] = old[b, h, s] (0 for the chunk's own positions) + the sum over
// the sequence's rows (tokens and the group's heads) of the softmax weight at
// s; 0 past the length. A block takes 128 positions of one (sequence, key
// head), 32 to a wave, their key rows in registers, and goes through the rows
// that see them, 16 at a time, in order: no atomics, the same sums each time. In
// slices of the rows, where there are few blocks, as pg_weigh_wide.
// `out` may be `old`: a thread reads an element before it writes it.
// Scores are made again (as in pg_attn), the weight is 2^(score - lse). Where
// pg_attn made few rows, and for fp32 queries of width 128.
extern "C" __global__ __launch_bounds__(256, 2) void pg_weigh(
    const pg_q* __restrict__ Q, long qrow, long qhead, const unsigned short* __restrict__ kp, int pages, int shift,
    const int* __restrict__ table, int N, const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M,
    int H, int G, float scale2, const float* __restrict__ lse, const float* old, int S, float* out, int So,
    int blocks, int run, int slices, float* __restrict__ part) {
  constexpr int KS = PG_E / 32;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, q = lane >> 4;
  const int id = pg_deal(blockIdx.x, run);
  if (id >= B * H * blocks * slices) return;
  const int slice = id % slices, task = id / slices;
  const int h = task / blocks % H, b = task / blocks / H, b0 = task % blocks * 128, p0 = b0 + 32 * wave;
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
    // the slice's share of the rows from the first token that sees the block's
    // first position, from the first that sees the wave's
    const int tile0 = max(b0 - new0, 0) * G / 16, share = (max((R + 15) / 16 - tile0, 0) + slices - 1) / slices;
    const int end = min((tile0 + (slice + 1) * share) * 16, R);
    for (int x0 = max((tile0 + slice * share) * 16, max(p0 - new0, 0) * G / 16 * 16); x0 < end; x0 += 16) {
      const int x = min(x0 + r, R - 1), tok = pg_div(x, G), head = h * G + x - tok * G;
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
      if (r != 0 || s >= So) continue;
      if (slices > 1) part[((size_t)slice * B * H + bh) * So + s] = w;
      else out[bh * So + s] = w + (s < new0 ? old[bh * S + s] : 0.0f);
    }
}

// The same where pg_attn left its scores (rows of `pitch` in `sc`): a thread
// takes every 256th of 1024 positions.
extern "C" __global__ __launch_bounds__(256) void pg_given(const float* __restrict__ sc, long pitch,
                                                           const int* __restrict__ starts,
                                                           const int* __restrict__ lengths, int cap, int M, int H, int G,
                                                           const float* __restrict__ lse, const float* old, int S,
                                                           float* out, int So, int blocks) {
  const int bh = blockIdx.x / blocks, b = bh / H, h = bh % H;      // grid: B * H * blocks
  const int p0 = blockIdx.x % blocks * 1024 + threadIdx.x;
  const PgSeq sq = pg_seq(starts, lengths, b, M, cap);
  const int new0 = sq.len - sq.count;
  float acc[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) acc[u] = p0 + 256 * u < min(new0, So) ? old[(size_t)bh * S + p0 + 256 * u] : 0.0f;
  for (int j = max(p0 - (int)threadIdx.x - new0, 0); j < sq.count; ++j)   // tokens that see some of the 1024
    for (int g = 0; g < G; ++g) {
      const long row = (long)(sq.first + j) * (H * G) + h * G + g;
      const float z = lse[row];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = p0 + 256 * u;
        if (s <= new0 + j) acc[u] += __builtin_amdgcn_exp2f(sc[row * pitch + s] - z);
      }
    }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (p0 + 256 * u < So) out[(size_t)bh * So + p0 + 256 * u] = acc[u];
}

// The same for many rows (fp32: of width 64): a block takes 256 positions of one
// (sequence, key head), 64 to a wave, their key rows in registers, and a slice
// of the rows that see them, 64 at a time through LDS (double-buffered, with
// the rows' lse, fp32 rows scaled and in three planes as in pg_query), on tiles
// of 32 x 32 x 16 as in pg_wide. A wave's sums stay in registers over all rows. Several slices (few positions, many rows) leave
// their sums in `part` [slice][B H So] for pg_total. 4 x 1999 tokens of 32 heads
// (8 of 128 keyed): 79.5 us, of which 45 the rows and the rest the blocks' starts
// and ends; slices of one size for all positions instead: 99. fp32: 32 x 768 of 12
// heads of 64, with the attention, 333 us in pg_weigh, 240 here.
#if PG_KIND != PG_F32 || PG_E == 64
extern "C" __global__ __launch_bounds__(256, 2) void pg_weigh_wide(
    const pg_q* __restrict__ Q, long qrow, long qhead, const unsigned short* __restrict__ kp, int pages, int shift,
    const int* __restrict__ table, int N, const int* __restrict__ starts, const int* __restrict__ lengths, int B, int M,
    int H, int G, float scale2, const float* __restrict__ lse, const float* old, int S,
    float* out, int So, int blocks, int run, int slices, float* __restrict__ part) {
  constexpr int KS = PG_E / 16, CH = PG_E / 8, NL = 64 * CH / 256, RS = 256 / CH;
  __shared__ __attribute__((aligned(16))) vh_u32x4 lq[2][PG_PLANES][64 * (CH + 1)];
  __shared__ float lz[2][64], lk2[2][64];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 31, g = lane >> 5;
  const int id = pg_deal(blockIdx.x, run);
  if (id >= B * H * blocks * slices) return;
  // the first positions of all heads first: most rows see them
  const int slice = id % slices, bh = id / slices % (B * H), b = bh / H, h = bh % H;
  const int b0 = id / slices / (B * H) * 256, p0 = b0 + 64 * wave;
  const PgSeq sq = pg_seq(starts, lengths, b, M, N << shift);
  const int new0 = sq.len - sq.count, R = sq.count * G;
  // the slice's rows: its share of the 64-row tiles from the first token that sees the block's first position
  const int tile0 = max(b0 - new0, 0) * G / 64, tiles = b0 < sq.len ? max((R + 63) / 64 - tile0, 0) : 0;
  const int share = (tiles + slices - 1) / slices;
  const int x0 = (tile0 + min(slice * share, tiles)) * 64, x1 = (tile0 + min((slice + 1) * share, tiles)) * 64;
  float acc[2][16] = {};
  vh_u32x4 kf[2][KS];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = min(p0 + 32 * i + r, sq.len - 1), page = x0 < x1 ? table[(size_t)b * N + (max(s, 0) >> shift)] : 0;
    const size_t at = ((size_t)((unsigned)page < (unsigned)pages ? page : 0) << shift) + (max(s, 0) & ((1 << shift) - 1));
#pragma unroll
    for (int k = 0; k < KS; ++k) kf[i][k] = ld16(kp + (at * H + h) * PG_E + 16 * k + 8 * g);
  }
  // Staging: row x + r8 + RS n is head `gr`, token `tr` of the sequence, both
  // carried on from 64 rows before (a division each cost a third of the loop).
  const int c8 = tid % CH, r8 = tid / CH, step_t = 64 / G, step_g = 64 % G;
  int tr[NL + 1], gr[NL + 1];                                      // the last: of the lse's row, x + tid
#pragma unroll
  for (int n = 0; n <= NL; ++n) {
    const int y = x0 + (n < NL ? r8 + RS * n : tid & 63);
    tr[n] = pg_div(y, G);
    gr[n] = y - tr[n] * G;
  }
#if PG_KIND == PG_F32
  vh_f32x4 qr[NL][2];
#else
  vh_u32x4 qr[NL];
#endif
  float zr = 0.0f;
  auto load = [&]() {                                              // past the last row: the last token, without weight
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const pg_q* qp = Q + (sq.first + min(tr[n], sq.count - 1)) * qrow + (h * G + gr[n]) * qhead + 8 * c8;
#if PG_KIND == PG_F32
      qr[n][0] = *(const vh_f32x4*)qp;
      qr[n][1] = *(const vh_f32x4*)(qp + 4);
#else
      qr[n] = ld16(qp);
#endif
    }
    if (tid < 64)
      zr = tr[NL] < sq.count ? lse[(size_t)(sq.first + tr[NL]) * (H * G) + h * G + gr[NL]] : INFINITY;
#pragma unroll
    for (int n = 0; n <= NL; ++n) {
      gr[n] += step_g;
      tr[n] += step_t;
      if (gr[n] >= G) {
        gr[n] -= G;
        ++tr[n];
      }
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int row = r8 + RS * n;
#if PG_KIND == PG_F32
      float v[8], mx = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = qr[n][j >> 2][j & 3];
        mx = fmaxf(mx, __builtin_fabsf(v[j]));
      }
#pragma unroll
      for (int m = 1; m < CH; m <<= 1) mx = fmaxf(mx, __shfl_xor(mx, m, 64));
      int e = 0;
      if (mx > 0.0f && mx < INFINITY) e = max(__builtin_amdgcn_frexp_expf(mx), -100);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __builtin_ldexpf(v[j], -e);
      vh_u32x4 f[3];
      pg_split(v, f);
#pragma unroll
      for (int p = 0; p < 3; ++p) lq[buf][p][row * (CH + 1) + c8] = f[p];
      if (c8 == 0) lk2[buf][row] = __builtin_ldexpf(scale2, e);
#else
      lq[buf][0][row * (CH + 1) + c8] = qr[n];
#endif
    }
    if (tid < 64) lz[buf][tid] = zr;
  };
  if (x0 < x1) load();
#pragma unroll
  for (int i = 0; i < 2; ++i) pg_here(kf[i]);
  if (x0 < x1) {
    put(0);
    if (x0 + 64 < x1) load();
  }
  for (int x = x0, buf = 0; x < x1; x += 64, buf ^= 1) {
    vh_lds_sync();
    if (x + 64 < x1) {
      put(buf ^ 1);
      if (x + 128 < x1) load();
    }
    if (new0 + pg_div(min(x + 63, R - 1), G) < p0) continue;              // no row sees the wave's positions
    const bool part = p0 + 63 > new0 + pg_div(x, G);                      // not all of them by every row
#if PG_KIND == PG_F32
#pragma nounroll
#else
#pragma unroll
#endif
    for (int u = 0; u < 2; ++u) {
      const float z = lz[buf][32 * u + r];
      pg_f16v s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[i][j] = 0.0f;
#if PG_KIND == PG_F32
      const float k2 = lk2[buf][32 * u + r];
      pg_f16v lo[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) lo[i][j] = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int at = (32 * u + r) * (CH + 1) + 2 * k + g;
        const vh_u32x4 q0 = lq[buf][0][at], q1 = lq[buf][1][at], q2 = lq[buf][2][at];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[i] = pg_mfma32(kf[i][k], q0, s[i]);
          lo[i] = pg_mfma32(kf[i][k], q1, lo[i]);
          lo[i] = pg_mfma32(kf[i][k], q2, lo[i]);
        }
      }
      float fin = 0.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) fin = fmaf(s[i][j], 0.0f, fin);
      if (__any(fin != fin)) {                                     // as in pg_scores
        const int y = min(x + 32 * u + r, R - 1), tok = pg_div(y, G);
        const pg_q* qp = Q + (sq.first + tok) * qrow + (h * G + y - tok * G) * qhead;
#pragma nounroll
        for (int e = 0; e < 32; ++e) {
          const int at = min(p0 + 32 * (e >> 4) + 8 * ((e & 15) >> 2) + 4 * g + (e & 3), sq.len - 1);
          const int page = table[(size_t)b * N + (at >> shift)];
          const unsigned short* kq = kp + ((((size_t)((unsigned)page < (unsigned)pages ? page : 0) << shift)
                                            + (at & ((1 << shift) - 1))) * H + h) * PG_E;
          float whole = 0.0f;
#pragma nounroll
          for (int c = 0; c < CH; ++c) {
            float kv[8];
            unpack8(ld16(kq + 8 * c), kv);
#pragma unroll
            for (int d = 0; d < 8; ++d) whole = fmaf(qp[8 * c + d], kv[d], whole);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float hi = s[i][j];
              if (e == 16 * i + j && !(__builtin_fabsf(hi) < INFINITY)) {
                s[i][j] = whole;
                lo[i][j] = 0.0f;
              }
            }
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) s[i][j] = vh_hilo(s[i][j], lo[i][j]);
#else
      const float k2 = scale2;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const vh_u32x4 qf = lq[buf][0][(32 * u + r) * (CH + 1) + 2 * k + g];
#pragma unroll
        for (int i = 0; i < 2; ++i) s[i] = pg_mfma32(kf[i][k], qf, s[i]);
      }
#endif
      if (part) {
        const int lim = new0 + pg_div(min(x + 32 * u + r, R - 1), G);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[i][j] = p0 + 32 * i + 8 * (j >> 2) + 4 * g + (j & 3) <= lim ? s[i][j] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] += __builtin_amdgcn_exp2f(fmaf(s[i][j], k2, -z));
    }
  }
  // Over the rows: lane 32 g + r keeps position 32 (r / 16) + 8 (r % 16 / 4) + 4 g + r % 4.
  // Lanes that differ in a bit of r each take over the sums that differ in it
  // alike, 31 exchanges (a sum at a time: 160).
  float sums[32];
#pragma unroll
  for (int k = 0; k < 32; ++k) sums[k] = acc[k >> 4][k & 15];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1)
#pragma unroll
    for (int k = 0; k < m; ++k) {
      const float give = r & m ? sums[k] : sums[k + m], keep = r & m ? sums[k + m] : sums[k];
      sums[k] = keep + __shfl_xor(give, m, 64);
    }
  const float w = sums[0];
  const int s = p0 + 32 * (r >> 4) + 8 * ((r & 15) >> 2) + 4 * g + (r & 3);
  if (s >= So) return;
  if (slices > 1) part[((size_t)slice * B * H + bh) * So + s] = w;
  else out[(size_t)bh * So + s] = w + (s < new0 ? old[(size_t)bh * S + s] : 0.0f);
}
#endif

// The slices' sums added to the old ones, in order.
extern "C" __global__ __launch_bounds__(256) void pg_total(const float* __restrict__ part, int slices,
                                                           const int* __restrict__ starts,
                                                           const int* __restrict__ lengths, int cap, int B, int M, int H,
                                                           const float* old, int S, float* out, int So, int blocks) {
  const int bh = blockIdx.x / blocks, s = blockIdx.x % blocks * 256 + threadIdx.x;     // grid: B * H * blocks
  if (s >= So) return;
  const PgSeq sq = pg_seq(starts, lengths, bh / H, M, cap);
  float w = 0.0f;
  for (int k = 0; k < slices; ++k) w += part[((size_t)k * B * H + bh) * So + s];
  out[(size_t)bh * So + s] = w + (s < sq.len - sq.count ? old[(size_t)bh * S + s] : 0.0f);
}

// ---------------------------------------------------------------- eviction
// pg_select: a block per (layer, sequence, head) finds which positions stay:
// the `recent` last and, of the others, those of largest weight, ties to the
// lowest position, min(keep, length) in all. The weight of the last one to stay
// is found 11, 11 and 10 bits at a time (histograms in LDS of an
// order-preserving whole number: with fewer bits at once the first digit, an
// exponent, takes few values, whose adds wait for each other), ending early
// where all that share a prefix stay; then the positions are listed in order,
// four consecutive ones a thread. A NaN counts as the largest. What bounds it:
// LDS adds, about one a cycle and CU whatever their addresses (four or eight
// copies of the histogram are no faster): 30,000 positions 31 us, of which 14
// the first digit's; 1152 times 1024 positions 13 us.
#define PG_BINS 2048
__device__ __forceinline__ unsigned pg_key(float w) {
  const unsigned u = __builtin_bit_cast(unsigned, w + 0.0f);       // -0 as 0
  if (w != w) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

#define PG_HELD 8                          // groups of four consecutive weights a thread holds in registers

extern "C" __global__ __launch_bounds__(1024) void pg_select(const float* __restrict__ weight, int S,
                                                             const int* __restrict__ lengths, int cap, int B, int H,
                                                             int keep, int recent, int* __restrict__ kept,
                                                             float* __restrict__ wout, int So,
                                                             int* __restrict__ lout, unsigned* __restrict__ err) {
  __shared__ int hist[PG_BINS];
  __shared__ int part[PG_HELD][16];
  __shared__ int found[3];                                         // the digit, how many of it stay, how many have it
  const int tid = threadIdx.x, threads = blockDim.x;               // 256 or 1024
  const int lane = tid & 63, wave = tid >> 6, waves = threads >> 6;
  const int b = blockIdx.x / H % B;                                // grid: layers * B * H
  const int len = lengths[b], n = min(max(len, 0), cap);
  const int m = min(keep, n), last = min(recent, m), C = n - last, take = m - last;
  if (blockIdx.x < (unsigned)(B * H) && blockIdx.x % H == 0 && tid == 0) {
    lout[b] = m;
    if (n != len) pg_raise(err, PG_ERR_LENGTH);
  }
  const float* w = weight + (size_t)blockIdx.x * S;
  // Group c of a thread: positions 4 (c threads + tid) .. + 3. The first
  // PG_HELD groups are loaded once, the rest (a long sequence's) in each pass.
  const int block = 4 * threads, held = PG_HELD * block;
  float x[PG_HELD][4];
  auto get = [&](int base) {
#pragma unroll
    for (int c = 0; c < PG_HELD; ++c)
      if (base + c * block < n)
#pragma unroll
        for (int u = 0; u < 4; ++u) x[c][u] = w[min(base + c * block + 4 * tid + u, n - 1)];
  };
  get(0);
  // of those whose key's bits from `bit` on are `prefix`, the first `need` stay,
  // and all above
  unsigned prefix = 0;
  int need = take, bit = 32;
  while (bit > 0 && take > 0 && take < C) {                        // the same for all threads
    const int bits = bit == 10 ? 10 : 11, low = bit - bits;
    for (int v = tid; v < PG_BINS; v += threads) hist[v] = 0;
    __syncthreads();
    for (int base = 0; base < C; base += held) {
      if (n > held) get(base);
#pragma unroll
      for (int c = 0; c < PG_HELD; ++c)
        if (base + c * block < C)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const unsigned k = pg_key(x[c][u]);
            if (base + c * block + 4 * tid + u < C && (bit == 32 || k >> (bit & 31) == prefix))
              atomicAdd(&hist[(k >> low) & ((1u << bits) - 1u)], 1);
          }
    }
    __syncthreads();
    // thread t takes the bins from the top, PG_BINS / threads each
    const int each = PG_BINS / threads, top = PG_BINS - 1 - tid * each;
    int mine = 0;
    for (int v = 0; v < each; ++v) mine += hist[top - v];
    const int upto = pg_scan(mine);
    if (lane == 63) part[0][wave] = upto;
    __syncthreads();
    int above = upto - mine;
    for (int i = 0; i < wave; ++i) above += part[0][i];
    if (above < need && need <= above + mine) {                    // one thread's
      int v = top;
      while (above + hist[v] < need) above += hist[v--];
      found[0] = v;
      found[1] = need - above;
      found[2] = hist[v];
    }
    __syncthreads();
    prefix = prefix << bits | (unsigned)found[0];
    need = found[1];
    bit = low;
    if (need == found[2]) break;
    __syncthreads();                                               // found is read
  }
  if (take >= C) need = C;                                         // all of them
  // positions in order
  int* kp = kept + (size_t)blockIdx.x * keep;
  float* wp = wout + (size_t)blockIdx.x * So;
  int above0 = 0, same0 = 0;                                       // in the groups before
  for (int base = 0; base < n; base += held) {
    if (n > held) get(base);
    unsigned stay[PG_HELD];                                        // bits u: above, 4 + u: same
    int upto[PG_HELD];                                             // above: low half, same: high half
    __syncthreads();                                               // part is read
#pragma unroll
    for (int c = 0; c < PG_HELD; ++c) {
      stay[c] = 0;
      upto[c] = 0;
      if (base + c * block < n) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int s = base + c * block + 4 * tid + u;
          const unsigned k = bit == 32 ? 0u : pg_key(x[c][u]) >> bit;
          if (s < n && (s >= C || (take > 0 && k > prefix))) stay[c] |= 1u << u;
          if (s < C && take > 0 && k == prefix) stay[c] |= 16u << u;
        }
        upto[c] = pg_scan(__builtin_popcount(stay[c] & 15u) + (__builtin_popcount(stay[c] & 240u) << 16));
        if (lane == 63) part[c][wave] = upto[c];
      }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < PG_HELD; ++c) {
      if (base + c * block >= n) continue;
      int before = 0, total = 0;
      for (int i = 0; i < waves; ++i) {
        if (i < wave) before += part[c][i];
        total += part[c][i];
      }
      before += upto[c] - __builtin_popcount(stay[c] & 15u) - (__builtin_popcount(stay[c] & 240u) << 16);
      int a = above0 + (before & 0xffff), e = same0 + (before >> 16);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool above = stay[c] >> u & 1u, same = stay[c] >> (4 + u) & 1u;
        if (above || (same && e < need)) {
          const int to = a + min(e, need);
          if (to < keep) {
            kp[to] = base + c * block + 4 * tid + u;
            wp[to] = x[c][u];
          }
        }
        a += above ? 1 : 0;
        e += same ? 1 : 0;
      }
      above0 += total & 0xffff;
      same0 += total >> 16;
    }
  }
  for (int s = m + tid; s < keep; s += threads) kp[s] = -1;
  for (int s = m + tid; s < So; s += threads) wp[s] = 0.0f;
}

// pg_move: the kept rows of all layers into the pages of the other table, 16
// bytes of a key and of a value row a thread: 393 MB in 72 us (5.5 TB/s; 79 with
// plain stores, which leave the rows in a cache that nothing reads them from).
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
  __builtin_nontemporal_store(kx, (vh_u32x4*)kp + into);
  __builtin_nontemporal_store(vx, (vh_u32x4*)vp + into);
}
