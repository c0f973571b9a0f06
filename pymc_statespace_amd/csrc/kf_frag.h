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

static __device__ __forceinline__ unsigned kf_bits(float x) { return __builtin_bit_cast(unsigned, x); }
static __device__ __forceinline__ float kf_float_of(unsigned x) { return __builtin_bit_cast(float, x); }
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
  static constexpr int PAD = 8;  // elements after a row in LDS: 16 bytes, so that 16 rows start in different banks
  static __device__ __forceinline__ kf_f32x4 mma(frag a, frag b, kf_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ frag zero() { return __builtin_bit_cast(frag, kf_u32x4{0, 0, 0, 0}); }
  // row i of a [i][depth] tile, p at its first depth of this lane
  static __device__ __forceinline__ frag row(const elem* p) { return *reinterpret_cast<const frag*>(p); }
  // the same row at depth T, p at 4 g
  static __device__ __forceinline__ frag row_t(const elem* p) {
    const kf_s16x4 x = *reinterpret_cast<const kf_s16x4*>(p), y = *reinterpret_cast<const kf_s16x4*>(p + 16);
    return __builtin_bit_cast(frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  // column i of a [depth][i] tile, p at its corner
  static __device__ __forceinline__ frag col(const elem* p, int ld, int i, int g) {
    const elem* a = p + (4 * g + (i >> 2)) * ld + 4 * (i & 3);
    typedef __attribute__((address_space(3))) kf_s16x4* lds;
    const kf_s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)a), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(a + 16 * ld));
    return __builtin_bit_cast(frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
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
  // four consecutive elements
  static __device__ __forceinline__ void put4(elem* p, kf_f32x4 x) {
    *reinterpret_cast<uint2*>(p) = make_uint2(kf_pack_bf16(x[0], x[1]), kf_pack_bf16(x[2], x[3]));
  }
  static __device__ __forceinline__ void put8(elem* p, frag x) { *reinterpret_cast<frag*>(p) = x; }
  static __device__ __forceinline__ float get(const elem* p) { return kf_float_of((unsigned)*p << 16); }
  static __device__ __forceinline__ kf_f32x4 get4(const elem* p) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    return kf_f32x4{kf_float_of(x.x << 16), kf_float_of(x.x & 0xffff0000u), kf_float_of(x.y << 16), kf_float_of(x.y & 0xffff0000u)};
  }
};

struct KfF32 {
  typedef float elem;
  typedef kf_f32x8 frag;
  static constexpr int PAD = 4;
  static __device__ __forceinline__ kf_f32x4 mma(frag a, frag b, kf_f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ frag zero() { return frag{0, 0, 0, 0, 0, 0, 0, 0}; }
  static __device__ __forceinline__ frag row(const elem* p) {
    const kf_f32x4 x = *reinterpret_cast<const kf_f32x4*>(p), y = *reinterpret_cast<const kf_f32x4*>(p + 4);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ frag row_t(const elem* p) {
    const kf_f32x4 x = *reinterpret_cast<const kf_f32x4*>(p), y = *reinterpret_cast<const kf_f32x4*>(p + 16);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ frag col(const elem* p, int ld, int i, int g) {
    frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = p[(16 * (e >> 2) + 4 * g + (e & 3)) * ld + i];
    return f;
  }
  static __device__ __forceinline__ frag from(kf_f32x4 x, kf_f32x4 y) { return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7); }
  static __device__ __forceinline__ float value(frag a, int e) { return a[e]; }
  static __device__ __forceinline__ frag finite(frag a) {
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = (kf_bits(a[e]) & 0x7f800000u) == 0x7f800000u ? 0.f : a[e];
    return a;
  }
  static __device__ __forceinline__ void put4(elem* p, kf_f32x4 x) { *reinterpret_cast<kf_f32x4*>(p) = x; }
  static __device__ __forceinline__ void put8(elem* p, frag x) {
    put4(p, __builtin_shufflevector(x, x, 0, 1, 2, 3));
    put4(p + 4, __builtin_shufflevector(x, x, 4, 5, 6, 7));
  }
  static __device__ __forceinline__ float get(const elem* p) { return *p; }
  static __device__ __forceinline__ kf_f32x4 get4(const elem* p) { return *reinterpret_cast<const kf_f32x4*>(p); }
};

// An operand times a weight for each depth, exact to 24 bits: in fp32 the product itself; in bf16 the fp32 product is cut into three
// parts of 8 bits each (cut, not rounded: the rest is exact and keeps the sign) and takes three matrix products.
template <typename A> struct KfWeighted;
template <> struct KfWeighted<KfF32> {
  kf_f32x8 p;
  __device__ __forceinline__ void set(kf_f32x8 a, const float (&w)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = a[e] * w[e];
  }
  __device__ __forceinline__ kf_f32x4 mma(kf_f32x8 b, kf_f32x4 c) const { return KfF32::mma(p, b, c); }
  __device__ __forceinline__ kf_f32x4 mma_right(kf_f32x8 a, kf_f32x4 c) const { return KfF32::mma(a, p, c); }
};
template <> struct KfWeighted<KfBf16> {
  kf_bf16x8 p0, p1, p2;
  __device__ __forceinline__ void set(kf_bf16x8 a, const float (&w)[8]) {
    unsigned x0[8], x1[8], x2[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = KfBf16::value(a, e) * w[e];
      x0[e] = kf_bits(x);
      const float r = x - kf_float_of(x0[e] & 0xffff0000u);
      x1[e] = kf_bits(r);
      x2[e] = kf_bits(r - kf_float_of(x1[e] & 0xffff0000u));
    }
    p0 = pack(x0); p1 = pack(x1); p2 = pack(x2);
  }
  static __device__ __forceinline__ kf_bf16x8 pack(const unsigned (&x)[8]) {  // the high halves
    kf_u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = __builtin_amdgcn_perm(x[2 * e + 1], x[2 * e], 0x07060302u);
    return __builtin_bit_cast(kf_bf16x8, r);
  }
  __device__ __forceinline__ kf_f32x4 mma(kf_bf16x8 b, kf_f32x4 c) const {
    return KfBf16::mma(p0, b, KfBf16::mma(p1, b, KfBf16::mma(p2, b, c)));
  }
  __device__ __forceinline__ kf_f32x4 mma_right(kf_bf16x8 a, kf_f32x4 c) const {
    return KfBf16::mma(a, p0, KfBf16::mma(a, p1, KfBf16::mma(a, p2, c)));
  }
};

// Accumulators of two 16 x 16 tiles as one operand: fp32 as they are; bf16 in two rounded parts, 2 x 8 bits and a sign each
// (2^-18 of each value is lost), two products.
template <typename A> struct KfSplit;
template <> struct KfSplit<KfF32> {
  static constexpr int PARTS = 2;  // 16-byte pieces
  kf_f32x8 p;
  __device__ __forceinline__ void set(kf_f32x4 x, kf_f32x4 y) { p = KfF32::from(x, y); }
  __device__ __forceinline__ kf_f32x4 mma(kf_f32x8 b, kf_f32x4 c) const { return KfF32::mma(p, b, c); }
  __device__ __forceinline__ float value(int e) const { return p[e]; }
  __device__ __forceinline__ kf_u32x4 piece(int k) const {
    return k ? __builtin_bit_cast(kf_u32x4, __builtin_shufflevector(p, p, 4, 5, 6, 7)) : __builtin_bit_cast(kf_u32x4, __builtin_shufflevector(p, p, 0, 1, 2, 3));
  }
  __device__ __forceinline__ void pieces(kf_u32x4 x, kf_u32x4 y) { p = KfF32::from(__builtin_bit_cast(kf_f32x4, x), __builtin_bit_cast(kf_f32x4, y)); }
};
template <> struct KfSplit<KfBf16> {
  static constexpr int PARTS = 2;
  kf_bf16x8 hi, lo;
  __device__ __forceinline__ void set(kf_f32x4 x, kf_f32x4 y) {
    hi = KfBf16::from(x, y);
    kf_f32x4 u, v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u[e] = x[e] - KfBf16::value(hi, e);
      v[e] = y[e] - KfBf16::value(hi, 4 + e);
    }
    lo = KfBf16::from(u, v);
  }
  __device__ __forceinline__ kf_f32x4 mma(kf_bf16x8 b, kf_f32x4 c) const { return KfBf16::mma(hi, b, KfBf16::mma(lo, b, c)); }
  __device__ __forceinline__ float value(int e) const { return KfBf16::value(hi, e) + KfBf16::value(lo, e); }
  __device__ __forceinline__ kf_u32x4 piece(int k) const { return __builtin_bit_cast(kf_u32x4, k ? lo : hi); }
  __device__ __forceinline__ void pieces(kf_u32x4 x, kf_u32x4 y) { hi = __builtin_bit_cast(kf_bf16x8, x); lo = __builtin_bit_cast(kf_bf16x8, y); }
};

// Eight consecutive elements of a global row as the arithmetic's own (the first `n` of them; n <= 0: none), zeros behind them.
// vec: the address is 16-byte aligned whenever n >= 8 (decided once for a tensor, on the host).
template <typename A, typename T> struct KfLoad8;
template <> struct KfLoad8<KfBf16, __hip_bfloat16> {
  static __device__ __forceinline__ kf_bf16x8 load(const __hip_bfloat16* p, int n, bool vec) {
    if (vec && n >= 8) return *reinterpret_cast<const kf_bf16x8*>(p);
    kf_s16x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = e < n ? reinterpret_cast<const short*>(p)[e] : (short)0;
    return __builtin_bit_cast(kf_bf16x8, r);
  }
};
template <> struct KfLoad8<KfF32, float> {
  static __device__ __forceinline__ kf_f32x8 load(const float* p, int n, bool vec) {
    if (vec && n >= 8) return KfF32::row(p);
    kf_f32x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = e < n ? p[e] : 0.f;
    return r;
  }
};
template <> struct KfLoad8<KfF32, __half> {
  static __device__ __forceinline__ kf_f32x8 load(const __half* p, int n, bool vec) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    if (vec && n >= 8) return __builtin_convertvector(*reinterpret_cast<const h8*>(p), kf_f32x8);
    kf_f32x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = e < n ? (float)reinterpret_cast<const _Float16*>(p)[e] : 0.f;
    return r;
  }
};

// Four consecutive outputs, the first n of them; vec: the address is aligned to four elements.
template <typename T>
static __device__ __forceinline__ void kf_store4(T* p, kf_f32x4 x, int n, bool vec) {
  if (vec && n >= 4) {
    struct alignas(4 * sizeof(T)) V4 { T v[4]; } r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r.v[e] = kf_from_float<T>(x[e]);
    *reinterpret_cast<V4*>(p) = r;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) p[e] = kf_from_float<T>(x[e]);
  }
}
