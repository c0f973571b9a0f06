// kf_frag.h -- 16-wide fragments of matrix products in two arithmetics with one layout, and how they leave LDS.
//
// A fragment is one operand of a 16 x 16 product over a depth of 32: lane (i = lane % 16, g = lane / 16) holds the 8 elements of
// row (column) i at 8 depths.  Which depths is free as long as both operands agree; two maps are used:
//   depth C:  8 g + e             -- 8 consecutive elements of a row-major [i][depth] tile: one (two) 16-byte LDS reads
//   depth T:  16 (e / 4) + 4 g + e % 4 -- what 4 accumulator registers of two 16 x 16 tiles hold, and what the transposing LDS
//             read (ds_read_b64_tr_b16: 4 rows x 16 columns to 4 values for each of 16 lanes) takes out of a [depth][i] tile
// so a product's result enters the next one as an operand without leaving its registers.
// bf16: one v_mfma_f32_16x16x32_bf16.  fp32: eight v_mfma_f32_16x16x4_f32, element e of both operands in each (their depth is the
// lane's g, so any map works).  Both leave D with column = lane % 16, rows 4 g + r.
#pragma once
#include "kf_sequence.h"

typedef __bf16 kf_bf16x8 __attribute__((ext_vector_type(8)));
typedef short kf_s16x4 __attribute__((ext_vector_type(4)));
typedef short kf_s16x8 __attribute__((ext_vector_type(8)));
typedef float kf_f32x4 __attribute__((ext_vector_type(4)));
typedef float kf_f32x8 __attribute__((ext_vector_type(8)));
typedef unsigned kf_u32x4 __attribute__((ext_vector_type(4)));

// x, but computed anew here as far as the compiler can tell: keeps addresses built from it out of registers held across a loop
static __device__ __forceinline__ int kf_fresh(int x) {
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("" : "+v"(x));
#endif
  return x;
}

// sums over the 16 lanes of a row, in all of them
template <int CTRL> static __device__ __forceinline__ float kf_dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
static __device__ __forceinline__ float kf_row_sum(float x) {
  x += kf_dpp<0x128>(x);  // row_ror 8, 4, 2, 1
  x += kf_dpp<0x124>(x);
  x += kf_dpp<0x122>(x);
  return x + kf_dpp<0x121>(x);
}

static __device__ __forceinline__ unsigned kf_bits(float x) { return __builtin_bit_cast(unsigned, x); }
static __device__ __forceinline__ float kf_float_of(unsigned x) { return __builtin_bit_cast(float, x); }
static __device__ __forceinline__ bool kf_finite(float x) { return (kf_bits(x) & 0x7f800000u) != 0x7f800000u; }
// two floats rounded to nearest even, packed (v_cvt_pk_bf16_f32)
typedef __bf16 kf_bf16x2 __attribute__((ext_vector_type(2)));
typedef float kf_f32x2 __attribute__((ext_vector_type(2)));
static __device__ __forceinline__ unsigned kf_pack_bf16(float lo, float hi) {
  const kf_f32x2 x = {lo, hi};
  return __builtin_bit_cast(unsigned, __builtin_convertvector(x, kf_bf16x2));
}

struct KfBf16 {
  typedef unsigned short elem;
  typedef kf_bf16x8 frag;
  static __device__ __forceinline__ kf_f32x4 mma(frag a, frag b, kf_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ frag from(kf_f32x4 x, kf_f32x4 y) {
    return __builtin_bit_cast(frag, kf_u32x4{kf_pack_bf16(x[0], x[1]), kf_pack_bf16(x[2], x[3]), kf_pack_bf16(y[0], y[1]), kf_pack_bf16(y[2], y[3])});
  }
  static __device__ __forceinline__ float value(frag a, int e) {
    const unsigned w = __builtin_bit_cast(kf_u32x4, a)[e >> 1];
    return kf_float_of((e & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ frag finite(frag a) {  // infinities and NaN as zeros
    kf_s16x8 x = __builtin_bit_cast(kf_s16x8, a);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (x[e] & 0x7f80) == 0x7f80 ? (short)0 : x[e];
    return __builtin_bit_cast(frag, x);
  }
  static __device__ __forceinline__ float get(const elem* p) { return kf_float_of((unsigned)*p << 16); }
};

struct KfF32 {
  typedef float elem;
  typedef kf_f32x8 frag;
  static __device__ __forceinline__ kf_f32x4 mma(frag a, frag b, kf_f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ frag from(kf_f32x4 x, kf_f32x4 y) { return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7); }
  static __device__ __forceinline__ float value(frag a, int e) { return a[e]; }
  static __device__ __forceinline__ frag finite(frag a) {
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = kf_finite(a[e]) ? a[e] : 0.f;
    return a;
  }
  static __device__ __forceinline__ float get(const elem* p) { return *p; }
};

// Rows of COLS elements in LDS, 64 banks of 4 bytes.  The 16-byte pieces of a row are permuted (by exclusive or) so that what is read
// or written at a time meets different banks: a piece of 16 neighbouring rows, of which rows 4 to 11 read the next lane group's depth
// (16-byte reads take the lanes in that order: measured by their conflicts), and 32 bytes of 8 rows for columns.  32-bit elements: only 8
// pieces are permuted among each other.  16 would leave a sixth of the conflicts, but the reads of columns then need twice as many
// addresses, and that costs more: gradient of 3 x 333 tokens 59.5 us instead of 58.
//
// A lane's part of an address is computed once (KfLanes, in bytes); row, column and depth of the tile come in as constants: rows (a
// multiple of 16) and whole TURNS pieces as an offset, the pieces inside by exclusive or.
struct KfLanes { int row, row_t, col; };
static __device__ __forceinline__ KfLanes kf_fresh(const KfLanes& x) { return {kf_fresh(x.row), kf_fresh(x.row_t), kf_fresh(x.col)}; }
template <typename A, int COLS> struct KfTile {
  typedef typename A::elem E;
  typedef typename A::frag F;
  static constexpr int SZ = sizeof(E), PIECE = 16 / SZ, PIECES = COLS / PIECE;
  static_assert(PIECES >= 4, "a row of 64 bytes at least");
  static constexpr int TURNS = SZ == 4 ? 8 : 16;  // pieces that are permuted among each other
  static constexpr int turn(int r) {
    const int b1 = (r >> 1) & 1, b2 = (r >> 2) & 1, b3 = (r >> 3) & 1;
    if (SZ == 4) return ((r & 3) << 1) | b2;
    return PIECES >= 16 ? (b2 ^ b3) * 8 + (r & 3) * 2 + b3 : PIECES == 8 ? (b2 ^ b3) * 4 + b1 * 2 + b3 : (b2 ^ b3) * 2 + b3;
  }
  static __device__ __forceinline__ int at(int r, int c) {  // element
    return r * COLS + (((c / PIECE) ^ turn(r)) * PIECE) + c % PIECE;
  }
  static __device__ __forceinline__ KfLanes lanes(int i, int g) {
    return {at(i, 8 * g) * SZ, at(i, 4 * g) * SZ, (SZ == 2 ? at(4 * g + (i >> 2), 4 * (i & 3)) : at(4 * g, i)) * SZ};
  }
  // byte address of a lane's part at row r (a multiple of 16) and column c (a multiple of what the lanes' parts span)
  static __device__ __forceinline__ int mix(int lane, int r, int c) {
    const int p = c / PIECE;
    return (lane ^ ((p & (TURNS - 1)) * 16)) + (p / TURNS) * (16 * TURNS) + r * (COLS * SZ);
  }
  template <typename X> static __device__ __forceinline__ X read(const E* p, int byte) { return *reinterpret_cast<const X*>(reinterpret_cast<const char*>(p) + byte); }
  template <typename X> static __device__ __forceinline__ void write(E* p, int byte, X x) { *reinterpret_cast<X*>(reinterpret_cast<char*>(p) + byte) = x; }

  // 8 bytes by an instruction of their own: two of them merged into one ds_read2st64_b64 take 16 cycles instead of 4 (volatile reads
  // are not merged; gradient of 4 x 2048 tokens, bf16: LDS busy 95 thousand cycles merged, 51 apart; 190 and 187 us)
  static __device__ __forceinline__ kf_s16x4 read8(const E* p, int byte) {
    typedef const volatile __attribute__((address_space(3))) kf_s16x4* lds;
    return *(lds)(reinterpret_cast<const char*>(p) + byte);
  }

  // operand: row r + i, depths c .. c + 31 in order C (c a multiple of 32)
  static __device__ __forceinline__ F row(const E* p, const KfLanes& L, int r, int c) {
    const int b = mix(L.row, r, c);
    if constexpr (SZ == 2) return read<F>(p, b);
    else return A::from(read<kf_f32x4>(p, b), read<kf_f32x4>(p, b ^ 16));
  }
  // the same in order T
  static __device__ __forceinline__ F row_t(const E* p, const KfLanes& L, int r, int c) {
    if constexpr (SZ == 2) {
      const kf_s16x4 x = read8(p, mix(L.row_t, r, c)), y = read8(p, mix(L.row_t, r, c + 16));
      return __builtin_bit_cast(F, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      return A::from(read<kf_f32x4>(p, mix(L.row_t, r, c)), read<kf_f32x4>(p, mix(L.row_t, r, c + 16)));
    }
  }
  // operand: column c + i, depths r .. r + 31 of the rows in order T
  static __device__ __forceinline__ F col(const E* p, const KfLanes& L, int r, int c) {
    if constexpr (SZ == 2) {
      typedef __attribute__((address_space(3))) kf_s16x4* lds;
      const char* q = reinterpret_cast<const char*>(p);
      const kf_s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(q + mix(L.col, r, c))),
                     y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(q + mix(L.col, r + 16, c)));
      return __builtin_bit_cast(F, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      F f;
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = read<float>(p, (mix(L.col, r, c) ^ (16 * turn(e & 3))) + (16 * (e >> 2) + (e & 3)) * COLS * SZ);
      return f;
    }
  }
  // four accumulators of row r + i at columns c + 4 g .. + 3 (c a multiple of 16)
  static __device__ __forceinline__ void put4(E* p, const KfLanes& L, int r, int c, kf_f32x4 x) {
    if constexpr (SZ == 2) write(p, mix(L.row_t, r, c), make_uint2(kf_pack_bf16(x[0], x[1]), kf_pack_bf16(x[2], x[3])));
    else write(p, mix(L.row_t, r, c), x);
  }
  static __device__ __forceinline__ kf_f32x4 get4(const E* p, const KfLanes& L, int r, int c) {
    if constexpr (SZ == 2) {
      const uint2 x = __builtin_bit_cast(uint2, read8(p, mix(L.row_t, r, c)));
      return kf_f32x4{kf_float_of(x.x << 16), kf_float_of(x.x & 0xffff0000u), kf_float_of(x.y << 16), kf_float_of(x.y & 0xffff0000u)};
    } else {
      return read<kf_f32x4>(p, mix(L.row_t, r, c));
    }
  }
  // eight elements of any row r at column c (a multiple of 8)
  static __device__ __forceinline__ void put8(E* p, int r, int c, F x) {
    const int b = at(r, c) * SZ;
    if constexpr (SZ == 2) {
      write(p, b, x);
    } else {
      write(p, b, __builtin_shufflevector(x, x, 0, 1, 2, 3));
      write(p, b ^ 16, __builtin_shufflevector(x, x, 4, 5, 6, 7));
    }
  }
  // with the columns of each 32 so ordered that a lane's four values of two neighbouring 16-wide tiles are 8 neighbours: column
  // 8 a + 4 y + b at 16 y + 4 a + b
  static __device__ __forceinline__ void put8_paired(E* p, int r, int c, F x) {
    const int to = (c & ~31) + (c & 31) / 2;
    if constexpr (SZ == 2) {
      const kf_u32x4 w = __builtin_bit_cast(kf_u32x4, x);
      write(p, at(r, to) * SZ, make_uint2(w[0], w[1]));
      write(p, at(r, to + 16) * SZ, make_uint2(w[2], w[3]));
    } else {
      write(p, at(r, to) * SZ, __builtin_shufflevector(x, x, 0, 1, 2, 3));
      write(p, at(r, to + 16) * SZ, __builtin_shufflevector(x, x, 4, 5, 6, 7));
    }
  }
};
// the column that stands at place c of such rows
static __device__ __forceinline__ int kf_paired(int c) { return (c & ~31) + 8 * ((c >> 2) & 3) + 4 * ((c >> 4) & 1) + (c & 3); }

// fp32 numbers as one operand (accumulators of two 16 x 16 tiles, or a fragment times a weight for each depth), exactly: fp32 as they
// are; bf16 cut into three parts of 8 bits each (cut, not rounded: what is left is exact and keeps the sign), three products.  Two parts
// would leave 2^-18 of each value out and states and their gradients 2.4e-6 off where fp32 sums leave 1.5e-7.
template <typename A> struct KfSplit;
template <> struct KfSplit<KfF32> {
  kf_f32x8 p;
  __device__ __forceinline__ void set(kf_f32x4 x, kf_f32x4 y) { p = KfF32::from(x, y); }
  __device__ __forceinline__ void set(kf_f32x8 a, const float (&w)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = a[e] * w[e];
  }
  __device__ __forceinline__ kf_f32x4 mma(kf_f32x8 b, kf_f32x4 c) const { return KfF32::mma(p, b, c); }
  __device__ __forceinline__ kf_f32x4 mma_right(kf_f32x8 a, kf_f32x4 c) const { return KfF32::mma(a, p, c); }
};
template <> struct KfSplit<KfBf16> {
  kf_bf16x8 p0, p1, p2;
  static __device__ __forceinline__ kf_bf16x8 high(const float (&x)[8]) {  // the high halves
    kf_u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = __builtin_amdgcn_perm(kf_bits(x[2 * e + 1]), kf_bits(x[2 * e]), 0x07060302u);
    return __builtin_bit_cast(kf_bf16x8, r);
  }
  static __device__ __forceinline__ void rest(float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] -= kf_float_of(kf_bits(x[e]) & 0xffff0000u);
  }
  __device__ __forceinline__ void cut(float (&x)[8]) {
    p0 = high(x);
    rest(x);
    p1 = high(x);
    rest(x);
    p2 = high(x);
  }
  __device__ __forceinline__ void set(kf_f32x4 x, kf_f32x4 y) {
    float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    cut(v);
  }
  __device__ __forceinline__ void set(kf_bf16x8 a, const float (&w)[8]) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = KfBf16::value(a, e) * w[e];
    cut(v);
  }
  __device__ __forceinline__ kf_f32x4 mma(kf_bf16x8 b, kf_f32x4 c) const { return KfBf16::mma(p0, b, KfBf16::mma(p1, b, KfBf16::mma(p2, b, c))); }
  __device__ __forceinline__ kf_f32x4 mma_right(kf_bf16x8 a, kf_f32x4 c) const { return KfBf16::mma(a, p0, KfBf16::mma(a, p1, KfBf16::mma(a, p2, c))); }
};

// 16 bytes at any element's address (global accesses need no alignment beyond the element's)
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) KfAny16 { kf_u32x4 v; };

// Elements col .. col + 7 of a global row of `dim` elements as the arithmetic's own, zeros from dim on and where !ok (`row` is
// readable all the same), in two steps: `raw` only loads, so that nothing waits for it until `finish` is called (PLAIN: it is known that
// nothing is to be zero).  No branches:
//   KF_ROWS_WHOLE   dim % 8 == 0
//   KF_ROWS_CUT     dim >= 8: the last piece is read from where it still ends inside the row, and moved down by the elements too many
//                   (a number that is the same for all lanes)
//   KF_ROWS_NARROW  dim < 8 occurs: element by element
enum { KF_ROWS_WHOLE, KF_ROWS_CUT, KF_ROWS_NARROW };
static inline int kf_rows_mode(int K, int V) { return K < 8 || V < 8 ? KF_ROWS_NARROW : K % 8 || V % 8 ? KF_ROWS_CUT : KF_ROWS_WHOLE; }
static __device__ __forceinline__ kf_u32x4 kf_keep(kf_u32x4 x, bool keep) {
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = keep ? x[e] : 0u;
  return x;
}
// eight 16-bit elements moved down by s (0 .. 7)
static __device__ __forceinline__ kf_u32x4 kf_down16(kf_u32x4 x, int s) {
  const kf_u32x4 a = {s & 4 ? x[2] : x[0], s & 4 ? x[3] : x[1], s & 4 ? 0 : x[2], s & 4 ? 0 : x[3]};
  const kf_u32x4 b = {s & 2 ? a[1] : a[0], s & 2 ? a[2] : a[1], s & 2 ? a[3] : a[2], s & 2 ? 0 : a[3]};
  const int h = 16 * (s & 1);
  return kf_u32x4{__builtin_amdgcn_alignbit(b[1], b[0], h), __builtin_amdgcn_alignbit(b[2], b[1], h), __builtin_amdgcn_alignbit(b[3], b[2], h), b[3] >> h};
}
template <int MODE> struct KfRow16 {
  typedef kf_u32x4 Raw;
  // the row at `row` elements behind `base` (the same for all lanes)
  template <typename T> static __device__ __forceinline__ Raw raw(const T* base, unsigned row, int col, int dim) {
    if constexpr (MODE == KF_ROWS_NARROW) {
      kf_s16x8 r;
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = col + e < dim ? reinterpret_cast<const short*>(base)[row + col + e] : (short)0;
      return __builtin_bit_cast(Raw, r);
    } else {
      const unsigned off = (row + (unsigned)(col < dim - 8 ? col : dim - 8)) * (unsigned)sizeof(T);
      return reinterpret_cast<const KfAny16<T>*>(reinterpret_cast<const char*>(base) + off)->v;
    }
  }
  template <bool PLAIN = false> static __device__ __forceinline__ Raw bits(Raw x, int col, int dim, bool ok) {
    if constexpr (PLAIN) return x;
    if constexpr (MODE == KF_ROWS_CUT) x = kf_down16(x, col + 8 > dim && col < dim ? col + 8 - dim : 0);
    return kf_keep(x, ok && col < dim);
  }
};
template <typename A, typename T, int MODE> struct KfRow;
template <int MODE> struct KfRow<KfBf16, __hip_bfloat16, MODE> : KfRow16<MODE> {
  template <bool PLAIN = false> static __device__ __forceinline__ kf_bf16x8 finish(kf_u32x4 x, int col, int dim, bool ok) {
    return __builtin_bit_cast(kf_bf16x8, KfRow16<MODE>::template bits<PLAIN>(x, col, dim, ok));
  }
};
template <int MODE> struct KfRow<KfF32, __half, MODE> : KfRow16<MODE> {
  template <bool PLAIN = false> static __device__ __forceinline__ kf_f32x8 finish(kf_u32x4 x, int col, int dim, bool ok) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    return __builtin_convertvector(__builtin_bit_cast(h8, KfRow16<MODE>::template bits<PLAIN>(x, col, dim, ok)), kf_f32x8);
  }
};
template <int MODE> struct KfRow<KfF32, float, MODE> {
  typedef kf_f32x8 Raw;
  static __device__ __forceinline__ Raw raw(const float* base, unsigned row, int col, int dim) {
    Raw r;
    if constexpr (MODE == KF_ROWS_NARROW) {
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = col + e < dim ? base[row + col + e] : 0.f;
    } else {
      const char* p = reinterpret_cast<const char*>(base) + (row + (unsigned)(col < dim - 8 ? col : dim - 8)) * 4u;
      r = KfF32::from(__builtin_bit_cast(kf_f32x4, reinterpret_cast<const KfAny16<float>*>(p)->v),
                      __builtin_bit_cast(kf_f32x4, reinterpret_cast<const KfAny16<float>*>(p + 16)->v));
    }
    return r;
  }
  template <bool PLAIN = false> static __device__ __forceinline__ kf_f32x8 finish(Raw x, int col, int dim, bool ok) {
    if constexpr (PLAIN) return x;
    if constexpr (MODE == KF_ROWS_CUT) {
      const int s = col + 8 > dim && col < dim ? col + 8 - dim : 0;
      kf_f32x8 y;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = s & 4 ? (e < 4 ? x[(e + 4) & 7] : 0.f) : x[e];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s & 2 ? (e < 6 ? y[(e + 2) & 7] : 0.f) : y[e];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = s & 1 ? (e < 7 ? x[(e + 1) & 7] : 0.f) : x[e];
      x = y;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = ok && col < dim ? x[e] : 0.f;
    return x;
  }
};

// Four consecutive outputs, the first n of them.
template <typename T>
static __device__ __forceinline__ void kf_store4(T* p, kf_f32x4 x, int n) {
  if (n >= 4) {
    typedef unsigned W __attribute__((ext_vector_type(sizeof(T))));
    struct __attribute__((packed, aligned(sizeof(T)))) Any { W v; };
    struct { T v[4]; } r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r.v[e] = kf_from_float<T>(x[e]);
    reinterpret_cast<Any*>(p)->v = __builtin_bit_cast(W, r);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) p[e] = kf_from_float<T>(x[e]);
  }
}

// Eight of them, made ready and stored.
template <typename T> struct alignas(16) KfOut8 {
  T v[8];
  __device__ __forceinline__ void set(kf_f32x4 x, kf_f32x4 y) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = kf_from_float<T>(x[e]);
      v[4 + e] = kf_from_float<T>(y[e]);
    }
  }
  __device__ __forceinline__ void store(T* p, int n) const {
    if (n >= 8) {
      struct Half { kf_u32x4 v[sizeof(T) / 2]; };
      const Half h = __builtin_bit_cast(Half, *this);
#pragma unroll
      for (unsigned e = 0; e < sizeof(T) / 2; ++e) reinterpret_cast<KfAny16<T>*>(p + 8 * e / (sizeof(T) / 2))->v = h.v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) p[e] = v[e];
    }
  }
};
