// Rows of a cache in 8 bits: each 32 values of a row are 8-bit elements and one
// power of two, in the OCP microscaling formats' layout (a byte a block):
//   PG_FORM 1  whole numbers of +-127: element q of a block with byte s stands for q 2^(s - 133)
//   PG_FORM 2  e4m3 floats (up to 448): element x for x 2^(s - 127)
// The power is the least with which a block's largest value is below 127.5 or 464
// steps of it, within limits that make every value one of fp16 (bf16 where PG_KIND is),
// so that opening an element is exact and what attention multiplies is what the
// cache holds. (Whole numbers read as bf16 end at 127 2^119, two powers below the
// type's end: they are opened as (q + 128) f - 128 f, which the last power would make
// an infinity.) A power of two costs e4m3 nothing and whole numbers half a bit on
// average against any factor; a block of its own for 32 dims gains about as
// much, and keeps the head's small dims apart from its large ones.
//
// Attention over such rows is hip/paged.hip's: rows are loaded as they are held and
// opened on their way to registers or LDS. Long decodes take what the cache's bytes
// take, half as many (two sequences after 120,001 of 8 heads of 128, 485 MB, in 96
// us, 5.1 TB/s, where 16 bits take 180). Chunks of many rows are bound as 16-bit
// ones are, with the opening on top: 4096 tokens after 18,001 in bf16 16 bits 1237 us,
// e4m3 1240 (two operations for four values), whole numbers 1350 (eleven); in fp16
// 1290, 1272 and 1355 (seven).
//
// A byte of 255 stands for a block of NaNs (whole numbers have none); e4m3 has a
// NaN itself, which is also what an infinity is held as.
#define PG_PAIR_BF16 (PG_KIND == 1)
#define PG8_MOST (PG_FORM == 1 ? 127.0f : 448.0f)
// a block's bytes, the least and the most; what is added to the largest value's
// bits so that its exponent counts the power that it needs (it goes up from
// 127.5 / 64 or 464 / 256 times a power of two on), and what that exceeds the byte by
#define PG8_LOW (PG_FORM == 1 ? (PG_PAIR_BF16 ? 7 : 109) : (PG_PAIR_BF16 ? 10 : 112))
#define PG8_HIGH (PG_FORM == 1 ? (PG_PAIR_BF16 ? 252 : 142) : (PG_PAIR_BF16 ? 246 : 134))
#define PG8_ROUND (PG_FORM == 1 ? 0x10000u : 0x180000u)
#define PG8_BELOW (PG_FORM == 1 ? 0 : 8)
#define PG8_NAN 255u

// A row's powers, one load.
#if PG_E == 64
typedef unsigned short pg_powers;
#else
typedef unsigned pg_powers;
#endif

typedef _Float16 pg_h2 __attribute__((ext_vector_type(2)));
typedef __bf16 pg_bf2 __attribute__((ext_vector_type(2)));

// What a block's elements are multiplied by, from its byte: 2^(s - 127), of
// whole numbers 2^(s - 133), as the opening wants it.
#if PG_FORM == 1 && !PG_PAIR_BF16
typedef pg_h2 pg_factor;
__device__ __forceinline__ pg_factor pg_power(unsigned s) {
  const _Float16 f = s == PG8_NAN ? (_Float16)__builtin_nanf("") : (_Float16)__builtin_bit_cast(float, (s - 6u) << 23);
  return pg_factor{f, f};
}
#else
typedef float pg_factor;
__device__ __forceinline__ pg_factor pg_power(unsigned s) {
#if PG_FORM == 1
  return s == PG8_NAN ? __builtin_nanf("") : __builtin_bit_cast(float, (s - 6u) << 23);
#else
  return __builtin_bit_cast(float, s << 23);
#endif
}
#endif

// Whether any of 16 elements, or of a row's powers, stands for a NaN.
__device__ __forceinline__ unsigned pg_odd(vh_u32x4 w) {
  unsigned any = 0u;
#if PG_FORM == 2
#pragma unroll
  for (int j = 0; j < 4; ++j) any |= (w[j] & 0x7f7f7f7fu) + 0x01010101u;
#endif
  return any & 0x80808080u;
}
__device__ __forceinline__ unsigned pg_odd_powers(pg_powers s) {
#if PG_FORM == 1
  return ((s & 0x7f7f7f7fu) + 0x01010101u) & s & 0x80808080u;
#else
  return 0u;
#endif
}

// Four elements as two words of 16-bit values, exactly.
// Whole numbers: fp16: q + 128 is put behind the exponent of 1024, and 1152 taken
// off again; bf16, whose fraction is too short for that: through fp32.
__device__ __forceinline__ vh_u32x2 pg_open4(unsigned w, pg_factor f) {
#if PG_FORM == 2 && PG_PAIR_BF16
  return vh_u32x2{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, f, false)),
                  __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, f, true))};
#elif PG_FORM == 2
  return vh_u32x2{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, f, false)),
                  __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, f, true))};
#elif PG_PAIR_BF16
  w ^= 0x80808080u;
  const float c = -128.0f * f;
  unsigned u[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) u[j] = __builtin_bit_cast(unsigned, fmaf((float)(w >> 8 * j & 255u), f, c));
  return vh_u32x2{__builtin_amdgcn_perm(u[1], u[0], 0x07060302u), __builtin_amdgcn_perm(u[3], u[2], 0x07060302u)};
#else
  w ^= 0x80808080u;
  const pg_h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
  const pg_h2 a = __builtin_bit_cast(pg_h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off;
  const pg_h2 b = __builtin_bit_cast(pg_h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off;
  return vh_u32x2{__builtin_bit_cast(unsigned, a * f), __builtin_bit_cast(unsigned, b * f)};
#endif
}
__device__ __forceinline__ vh_u32x4 pg_open(unsigned lo, unsigned hi, pg_factor f) {
  const vh_u32x2 a = pg_open4(lo, f), b = pg_open4(hi, f);
  return vh_u32x4{a[0], a[1], b[0], b[1]};
}
