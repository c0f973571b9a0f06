// kf_orthogonalise.hip -- a batch of matrices moved towards their orthogonal factors by Newton-Schulz products:
//     X = M / (|M|_F + eps);   per step   A = X X',   X <- a X + (b A + c A A) X
// on the transpose where there are more rows than columns: X is d x L with d <= L.  Four ways, by size and type:
//   * d <= 16, L <= 64: one wave for each matrix, all steps in its registers
//   * d <= 80 and X in LDS: one workgroup for each matrix, all steps on chip, in 32 bits (64 for fp64)
//   * larger, up to 32 bits: tiled products on v_mfma_f32_16x16x32_f16, numbers held in fp16 parts (below)
//   * larger, fp64: tiled products on v_mfma_f64_16x16x4
//
// Numbers in fp16 parts.  The singular values stay below 2 (checked on the host), so entries of X, A = X X' and B = b A + c A A are
// bounded and a power of two for each brings them to the top of fp16's range: hi = fp16(x), lo = fp16(x - hi) hold 22 bits and
// nothing overflows.  fp32 and fp16 data take three products, hi hi + hi lo + lo hi (2^-22 of the terms is lost), at 1/3 of fp16's rate,
// five times fp32's.  bf16 data keep X in both parts, which is what the term a X and every later step build on, but multiply hi parts
// only: the products' rounding (2^-12 a factor) then stays below that of the bf16 result, 1.1e-3 to 1.8e-3 against 1.7e-3 of |X|, also
// where M is of low rank (X in one part grows its rounding by a for each step in the missing directions: 4e-2 there).
//
// Where |M|_F is far below eps, X starts far below 1 and its parts would leave fp16's range at the lower end (|M| = 1e-7 eps, 150 x 200 in
// fp32: 1.8e-3 off).  Each matrix then carries 2^k X, with k >= 0 from its norm, and k falls by what a step can grow X by until it is 0: with
// Y = 2^k X a step is a Y + (4^-k b (YY') + 16^-k c (YY')^2) Y.  k = 0 multiplies by 1: no bit of other matrices changes.
//
// Measured: one 4096 x 4096 in fp32 3.7 ms, at 1101 TFLOP/s (the fp16 rate of a large library product) its 4.1 TFLOP take 3.75 ms; its fp32
// library products 14.5 ms.  Four of 768 x 2048 in fp32 or fp16 387 us, in bf16 224, 74 at that rate: with 312 tiles of 64 (A, B) and 384 of 128 (X) for 256
// compute units, the units that have two bound each product by the 64 bytes a cycle they can read, 15 + 8 + 22 us a step.
#include "kf_sequence.h"

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

template <typename T> struct Acc { typedef float type; };
template <> struct Acc<double> { typedef double type; };
static __device__ __forceinline__ double to_acc(double x) { return x; }
static __device__ __forceinline__ float to_acc(float x) { return x; }
static __device__ __forceinline__ float to_acc(__half x) { return __half2float(x); }
static __device__ __forceinline__ float to_acc(__hip_bfloat16 x) { return __bfloat162float(x); }
template <typename T> static __device__ __forceinline__ T from_acc(typename Acc<T>::type x) { return kf_from_float<T>(x); }
template <> __device__ __forceinline__ double from_acc<double>(double x) { return x; }

template <typename X> static __device__ __forceinline__ X block_sum(X s, X* red) {  // red: one for each wave
#pragma unroll
  for (int m = 1; m < 64; m *= 2) s += __shfl_xor(s, m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  s = X(0);
  for (unsigned i = 0; i < blockDim.x / 64; ++i) s += red[i];
  return s;
}

// ------------------------------------------------------------------------------------- in the registers of one wave
// d <= 16, L <= 16 NT.  Tiles of 16 x 16 as v_mfma_*_16x16x4 leave them: lane (g, c) holds column c of rows r(s, g), s = 0 .. 3.
// Measured against one workgroup for each matrix (below): 512 of 16 x 64 in fp32 9 and 27 us, 4096 of 16 x 64 in fp64 36 and 132.
// The same registers are the right operand of a product that runs over those rows, and the left operand's transpose: with y = X' (X's
// tiles transposed through LDS once a step), A = y'y, A A and B X = (B)'x need no other lane's values.  The fp64 instructions' 64 cycles
// bound it (each SIMD has four matrices of 4096): four of them only where the depth is above 12 (4096 matrices of 10 x 10: 14 us with
// four each time and X' by a product of its own, 10 now).
template <typename C> struct Tile;
template <> struct Tile<double> {
  typedef double type __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ int row(int s, int g) { return 4 * s + g; }
  static __device__ __forceinline__ type mma(type a, type b, type c, int depth) {  // (step s: depths 4 s .. 4 s + 3)
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (4 * s < depth) c = __builtin_amdgcn_mfma_f64_16x16x4f64(a[s], b[s], c, 0, 0, 0);
    return c;
  }
};
template <> struct Tile<float> {
  typedef f4 type;
  static __device__ __forceinline__ int row(int s, int g) { return 4 * g + s; }
  static __device__ __forceinline__ type mma(type a, type b, type c, int) {  // (step s: depths s, 4 + s, 8 + s, 12 + s)
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
    return c;
  }
};

template <typename T, int NT>
__global__ __launch_bounds__(256) void orth_wave_kernel(KfOrthArgs a) {
  typedef typename Acc<T>::type C;
  typedef Tile<C> Q;
  typedef typename Q::type V;
  __shared__ C turn[4][16][17];  // one tile for each wave; 17: rows and columns meet different banks
  const long z = blockIdx.x * 4l + (threadIdx.x >> 6);
  if (z >= a.n) return;
  const int l = threadIdx.x & 63, g = l >> 4, c = l & 15;
  const bool tall = a.rows > a.cols;
  const int d = tall ? a.cols : a.rows, L = tall ? a.rows : a.cols;
  const int sr = tall ? 1 : a.cols, sc = tall ? a.cols : 1;  // strides of X's rows and columns in M
  const T* M = (const T*)a.M + z * d * L;
  V x[NT];
  double sum = 0.;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int r = Q::row(s, g);
      x[t][s] = r < d && 16 * t + c < L ? to_acc(M[r * sr + (16 * t + c) * sc]) : C(0);
      sum += (double)x[t][s] * (double)x[t][s];
    }
#pragma unroll
  for (int m = 1; m < 64; m *= 2) sum += __shfl_xor(sum, m);
  const double f = 1.0 / (sqrt(sum) + a.eps);
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int s = 0; s < 4; ++s) x[t][s] = (C)((double)x[t][s] * f);
  C(*const tile)[17] = turn[threadIdx.x >> 6];
  const V zero = {C(0), C(0), C(0), C(0)};
  for (int step = 0; step < a.steps; ++step) {
    const C ca = (C)a.coef[step][0], cb = (C)a.coef[step][1], cc = (C)a.coef[step][2];
    V A = zero;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      // (a wave's LDS operations are done in their order; the fences, which cost no instruction, keep the compiler to it)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int s = 0; s < 4; ++s) tile[Q::row(s, g)][c] = x[t][s];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      V y;
#pragma unroll
      for (int s = 0; s < 4; ++s) y[s] = tile[c][Q::row(s, g)];
      A = Q::mma(y, y, A, L - 16 * t);
    }
    const V B = cb * A + cc * Q::mma(A, A, zero, d);
#pragma unroll
    for (int t = 0; t < NT; ++t) x[t] = Q::mma(B, x[t], ca * x[t], d);
  }
  T* out = (T*)a.X + z * d * L;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int r = Q::row(s, g);
      if (r < d && 16 * t + c < L) out[r * sr + (16 * t + c) * sc] = from_acc<T>(x[t][s]);
    }
}

template <typename T>
int launch_wave(kf_handle* h, const KfOrthArgs& a, hipStream_t stream) {
  const int L = a.rows > a.cols ? a.rows : a.cols;
  const dim3 grid((unsigned)((a.n + 3) / 4));
  if (L <= 16) hipLaunchKernelGGL((orth_wave_kernel<T, 1>), grid, dim3(256), 0, stream, a);
  else if (L <= 32) hipLaunchKernelGGL((orth_wave_kernel<T, 2>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((orth_wave_kernel<T, 4>), grid, dim3(256), 0, stream, a);
  KF_HIP_CHECK(h, hipGetLastError());
  return KF_OK;
}
static inline bool fits_wave(const KfOrthArgs& a) { return (a.rows <= 16 && a.cols <= 64) || (a.cols <= 16 && a.rows <= 64); }

// ----------------------------------------------------------------------------------------------------- on chip
// d <= 80 and X, A and B in LDS, padded with zeros to whole tiles of 16 x 16; one workgroup for each matrix.  A product's
// operand is read along the depth, 4 numbers of one row for each lane (depth 4 g + s in step s, the same for both operands), or, X as the
// right operand of B X, 4 numbers of one column.  B X stays in registers until every wave has read X.  Rows are an odd number of 16-byte
// pieces apart: neighbouring rows meet different banks.  Where A has fewer tiles than there are waves the sum over L is cut into
// `slices`, which meet in LDS.  Measured against the tiled products below, fp32: 256 matrices of 24 x 24 11 and 143 us, 256 of 64 x 64 42 and
// 145, 256 of 64 x 250 79 and 189, one of 64 x 250 71 and 63, one of 80 x 150 69 and 75; fp64: 256 of 80 x 80 74 and 510 us.  Bound by the
// waits between its three products a step, each short: the matrix pipe is busy 10 us of a 64 x 64 matrix's 40.  (8 waves of 16 tiles, for
// more than 64 tiles of X in 32 bits, spill 5 of their 256 registers.)
template <typename C> struct ChipRow { static __host__ __device__ constexpr int stride(int n) { return sizeof(C) == 8 ? (n & ~1) | 2 : (n & ~3) | 4; } };

// WAVES x HELD tiles of X at most, HELD for each wave.
template <typename T, int WAVES, int HELD>
__global__ __launch_bounds__(64 * WAVES, HELD == 4 ? 4 : 2) void orth_chip_kernel(KfOrthArgs a, int slices) {
  typedef typename Acc<T>::type C;
  typedef Tile<C> Q;
  typedef typename Q::type V;
  constexpr int TH = 64 * WAVES;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ double red[WAVES];
  const bool tall = a.rows > a.cols;
  const int d = tall ? a.cols : a.rows, L = tall ? a.rows : a.cols;
  const int td = (d + 15) / 16, tl = (L + 15) / 16, ts = td * (td + 1) / 2;
  const int lx = ChipRow<C>::stride(16 * tl), la = ChipRow<C>::stride(16 * td);
  C* X = (C*)smem;
  C* A = X + 16 * td * lx;
  C* B = A + 16 * td * la;
  C* part = B + 16 * td * la;  // [slices][ts][256]
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, i = l & 15, g = l >> 4;
  const long size = (long)d * L;
  const T* M = (const T*)a.M + blockIdx.x * size;
  T* out = (T*)a.X + blockIdx.x * size;
  for (int e = tid; e < 16 * td * lx; e += TH) X[e] = C(0);
  __syncthreads();
  double sum = 0.;
  for (int e = tid; e < size; e += TH) {
    const C x = to_acc(M[e]);
    const int r = e / a.cols, c = e - r * a.cols;
    X[tall ? c * lx + r : r * lx + c] = x;
    sum += (double)x * (double)x;
  }
  const double f = 1.0 / (sqrt(block_sum(sum, red)) + a.eps);
  for (int e = tid; e < 16 * td * lx; e += TH) X[e] = (C)((double)X[e] * f);  // (f = inf of a matrix of zeros with eps = 0: NaN, as it should be)
  __syncthreads();
  typedef V V16 __attribute__((aligned(16)));
  auto row = [&](const C* p, int ld, int r, int k) { return (V)*reinterpret_cast<const V16*>(p + (r + i) * ld + k + 4 * g); };
  auto below = [](int t, int* r, int* c) {  // tile t on or below the diagonal
    int x = 0;
    while ((x + 1) * (x + 2) / 2 <= t) ++x;
    *r = 16 * x;
    *c = 16 * (t - x * (x + 1) / 2);
  };
  auto store = [&](C* p, int r0, int c0, V v) {  // and its mirror image
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int r = r0 + Q::row(s, g);
      p[r * la + c0 + i] = v[s];
      p[(c0 + i) * la + r] = v[s];
    }
  };
  const V zero = {C(0), C(0), C(0), C(0)};
  for (int step = 0; step < a.steps; ++step) {
    const C ca = (C)a.coef[step][0], cb = (C)a.coef[step][1], cc = (C)a.coef[step][2];
    // A = X X'
    for (int x = w; x < ts * slices; x += WAVES) {
      const int t = x % ts, sl = x / ts;
      int r0, c0;
      below(t, &r0, &c0);
      V acc = zero;
      for (int k = 16 * sl; k < 16 * tl; k += 16 * slices) acc = Q::mma(row(X, lx, r0, k), row(X, lx, c0, k), acc, 16);
      if (slices > 1) reinterpret_cast<V16*>(part)[x * 64 + l] = acc;
      else store(A, r0, c0, acc);
    }
    __syncthreads();
    if (slices > 1) {
      for (int t = w; t < ts; t += WAVES) {
        int r0, c0;
        below(t, &r0, &c0);
        V acc = zero;
        for (int sl = 0; sl < slices; ++sl) acc += reinterpret_cast<const V16*>(part)[(sl * ts + t) * 64 + l];
        store(A, r0, c0, acc);
      }
      __syncthreads();
    }
    // B = b A + c A A (A is symmetric: rows for columns)
    for (int t = w; t < ts; t += WAVES) {
      int r0, c0;
      below(t, &r0, &c0);
      V acc = zero;
      for (int k = 0; k < 16 * td; k += 16) acc = Q::mma(row(A, la, r0, k), row(A, la, c0, k), acc, 16);
#pragma unroll
      for (int s = 0; s < 4; ++s) acc[s] = cb * A[(r0 + Q::row(s, g)) * la + c0 + i] + cc * acc[s];
      store(B, r0, c0, acc);
    }
    __syncthreads();
    // a X + B X
    V held[HELD];
#pragma unroll
    for (int u = 0; u < HELD; ++u) {
      const int t = w + u * WAVES;
      held[u] = zero;
      if (t < td * tl) {
        const int r0 = t / tl * 16, c0 = t % tl * 16;
#pragma unroll
        for (int s = 0; s < 4; ++s) held[u][s] = ca * X[(r0 + Q::row(s, g)) * lx + c0 + i];
        for (int k = 0; k < 16 * td; k += 16) {
          V x;
#pragma unroll
          for (int s = 0; s < 4; ++s) x[s] = X[(k + 4 * g + s) * lx + c0 + i];
          held[u] = Q::mma(row(B, la, r0, k), x, held[u], 16);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < HELD; ++u) {
      const int t = w + u * WAVES;
      if (t < td * tl) {
        const int r0 = t / tl * 16, c0 = t % tl * 16;
#pragma unroll
        for (int s = 0; s < 4; ++s) X[(r0 + Q::row(s, g)) * lx + c0 + i] = held[u][s];
      }
    }
    __syncthreads();
  }
  for (int e = tid; e < size; e += TH) {
    const int r = e / a.cols, c = e - r * a.cols;
    out[e] = from_acc<T>(X[tall ? c * lx + r : r * lx + c]);
  }
}

struct ChipPlan { int waves, held, slices; size_t lds; bool fits; };
ChipPlan chip_plan(const KfOrthArgs& a) {
  ChipPlan p;
  const int d = a.rows < a.cols ? a.rows : a.cols, L = a.rows < a.cols ? a.cols : a.rows;
  p.fits = false;
  if (d > 80 || L > 10000) return p;
  const int td = (d + 15) / 16, tl = (L + 15) / 16, ts = td * (td + 1) / 2;
  const bool wide = a.dtype == KF_DTYPE_F64;
  auto stride = [&](int n) { return wide ? ChipRow<double>::stride(n) : ChipRow<float>::stride(n); };
  // as few registers as hold the tiles, so that several matrices share a compute unit (1024 of 24 x 100: 87 us with 8 waves that could hold
  // 16 tiles each, 39 with 4 of 4 tiles; 1024 of 40 x 100: 124 us, with 8 of 4 tiles 79)
  const int tiles = td * tl;
  p.waves = tiles <= 16 ? 4 : 8;
  p.held = tiles <= 32 ? 4 : tiles <= 64 ? 8 : 16;
  p.slices = p.waves / ts < 1 ? 1 : p.waves / ts;
  p.lds = (wide ? 8 : 4) * ((size_t)16 * td * (stride(16 * tl) + 2 * stride(16 * td)) + (p.slices > 1 ? p.slices * ts * 256 : 0));
  p.fits = p.lds <= 156 * 1024 && tiles <= 8 * (wide ? 8 : 16);
  return p;
}

template <typename T, int WAVES, int HELD>
int launch_chip(kf_handle* h, const KfOrthArgs& a, const ChipPlan& p, hipStream_t stream) {
  KF_HIP_CHECK(h, hipFuncSetAttribute(reinterpret_cast<const void*>(orth_chip_kernel<T, WAVES, HELD>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.lds));
  hipLaunchKernelGGL((orth_chip_kernel<T, WAVES, HELD>), dim3((unsigned)a.n), dim3(64 * WAVES), p.lds, stream, a, p.slices);
  KF_HIP_CHECK(h, hipGetLastError());
  return KF_OK;
}
template <typename T>
int launch_chip(kf_handle* h, const KfOrthArgs& a, const ChipPlan& p, hipStream_t stream) {
  if (p.waves == 4) return launch_chip<T, 4, 4>(h, a, p, stream);
  if (p.held == 4) return launch_chip<T, 8, 4>(h, a, p, stream);
  if constexpr (sizeof(typename Acc<T>::type) == 4)
    if (p.held == 16) return launch_chip<T, 8, 16>(h, a, p, stream);
  return launch_chip<T, 8, 8>(h, a, p, stream);
}

// ------------------------------------------------------------------------------------- |M|_F^2 in 64 bits, by parts
constexpr int NORM_PARTS = 1024;
template <typename T>
__global__ __launch_bounds__(256) void orth_norm_kernel(const T* M, long size, double* part) {
  constexpr int V = 16 / sizeof(T);
  struct alignas(16) Piece { T v[V]; };
  __shared__ double red[4];
  const T* m = M + (long)blockIdx.y * size;
  double s = 0.;
  const long step = gridDim.x * 256l, first = blockIdx.x * 256l + threadIdx.x;
  const long head = ((uintptr_t)m & 15) ? 0 : size / V;  // whole pieces
  for (long i = first; i < head; i += step) {
    const Piece p = reinterpret_cast<const Piece*>(m)[i];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const double x = (double)to_acc(p.v[e]);
      s += x * x;
    }
  }
  for (long i = head * V + first; i < size; i += step) {
    const double x = (double)to_acc(m[i]);
    s += x * x;
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) part[blockIdx.y * (long)gridDim.x + blockIdx.x] = s;
}
// by a whole workgroup, the same order everywhere
static __device__ __forceinline__ double norm_factor(const double* part, int parts, double eps, double* red, double* norm = nullptr) {
  double s = 0.;
  for (int x = threadIdx.x; x < parts; x += blockDim.x) s += part[x];
  s = sqrt(block_sum(s, red));
  if (norm) *norm = s;
  return 1.0 / (s + eps);
}
static inline int norm_parts(long size) {  // about 16 elements a thread
  const long p = (size + 4095) / 4096;
  return p < NORM_PARTS ? (int)p : NORM_PARTS;
}
static inline size_t norm_bytes(const KfOrthArgs& a) { return kf_seq_round((size_t)a.n * norm_parts((long)a.rows * a.cols) * 8); }

// ------------------------------------------------------------------------------------------------ fp16 parts
constexpr float SCALE_X = 16384.f;  // 2^14: |x| < 2 stays below 32768, half of what fp16 holds (what rounding adds has room)
constexpr float SCALE_A = 8192.f;   // 2^13: |a| < 4 stays below 32768

// Where entry (r, c) of a matrix with rows of ld entries has its hi part: alone (STORED 1), or with the lo parts of 32 columns
// behind the hi parts of the same 32, one 128-byte line (STORED 2).
template <int STORED> static __device__ __forceinline__ long place(long r, long c, long ld) {
  return STORED == 1 ? r * ld + c : r * 2 * ld + ((c >> 5) << 6) + (c & 31);
}

static __device__ __forceinline__ void parts_of(f4 x, h4* hi, h4* lo) {
  *hi = __builtin_convertvector(x, h4);
  *lo = __builtin_convertvector(x - __builtin_convertvector(*hi, f4), h4);
}

template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Eight { T v[8]; };  // at any element's address
// 8 neighbours of a row of the result, of which `left` are inside it; at any element's address
template <typename T> static __device__ __forceinline__ void store_row(T* to, f4 x, f4 y, int left) {
  Eight<T> o;
#pragma unroll
  for (int j = 0; j < 4; ++j) o.v[j] = from_acc<T>(x[j]), o.v[4 + j] = from_acc<T>(y[j]);
  if (left >= 8) {
    *reinterpret_cast<Eight<T>*>(to) = o;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) to[j] = o.v[j];
  }
}

// M (rows x cols) times its factor, in parts: dP x LP, zeros behind d and L, transposed where M is tall; shift: each matrix's first k
template <typename T, int STORED>
__global__ __launch_bounds__(256) void orth_parts_kernel(KfOrthArgs a, const double* part, int parts, int dP, int LP, _Float16* hi, _Float16* lo,
                                                         int* shift) {
  __shared__ float tile[64][65];
  const bool tall = a.rows > a.cols;
  const int d = tall ? a.cols : a.rows, L = tall ? a.rows : a.cols;
  const long z = blockIdx.z, at = z * dP * (long)LP * STORED;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  __shared__ double red[4];
  double norm, f = norm_factor(part + z * parts, parts, a.eps, red, &norm);
  const double size = norm * f;  // |X|_F; 2^k of it in [1/2, 1)
  const int k = size > 0. && size < 0.5 ? -1 - ilogb(size) : 0;
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) shift[z] = k;
  f = ldexp(f * SCALE_X, k);
  const T* M = (const T*)a.M + z * d * (long)L;
  if (tall) {
    for (int e = threadIdx.x; e < 4096; e += 256) {
      const int c = e >> 6, r = e & 63;  // neighbours along M's rows
      tile[r][c] = r0 + r < d && c0 + c < L ? (float)((double)to_acc(M[(c0 + c) * (long)d + r0 + r]) * f) : 0.f;
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int e = threadIdx.x + 256 * u, r = e >> 3, c = 8 * (e & 7);
    f4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
    if (tall) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = tile[r][c + j], y[j] = tile[r][c + 4 + j];
    } else if (r0 + r < d) {
      const T* m = M + (r0 + r) * (long)L + c0 + c;
      const int left = L - c0 - c;
      Eight<T> in;
      if (left >= 8) {
        in = *reinterpret_cast<const Eight<T>*>(m);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) in.v[j] = j < left ? m[j] : from_acc<T>(0.f);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = (float)((double)to_acc(in.v[j]) * f);
        y[j] = (float)((double)to_acc(in.v[4 + j]) * f);
      }
    }
    h4 xh, xl, yh, yl;
    parts_of(x, &xh, &xl);
    parts_of(y, &yh, &yl);
    const long to = at + place<STORED>(r0 + r, c0 + c, LP);
    *(h8*)(hi + to) = __builtin_shufflevector(xh, yh, 0, 1, 2, 3, 4, 5, 6, 7);
    *(h8*)(lo + to) = __builtin_shufflevector(xl, yl, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

enum { GRAM, POLY, UPDATE };

struct Product {
  int n, d, L, dP, LP;      // sizes; rows and columns are padded to dP and LP, multiples of 128
  int tiles_m, tiles_n;     // of one matrix's output
  int depth;
  long works, whole;        // tiles, of which the first `whole` are done by one workgroup each, the others (of 128) by four
  const _Float16 *P, *Q;    // left operand, rows over the depth; right: rows over the depth (GRAM, POLY), or depth x columns (UPDATE)
  const _Float16 *Dh, *Dl;  // what is added: A (POLY), X (UPDATE)
  _Float16 *Ch, *Cl;        // output in parts
  void* out;                // or in T (the last UPDATE), `tall`: transposed
  int tall;
  float unscale;            // accumulator -> the output's scale
  float add;                // factor of what is added
  const int* shift;         // each matrix's first k; in this step it is lower by k_before, in the next one by k_after (not below 0)
  int k_before, k_after;
};

// out = unscale P Q + add D, TILE x TILE of it for each workgroup of 2 x 2 waves.  Depth in steps of BK through a ring of LDS buffers
// that global_load_lds fills ahead (16 bytes a lane, no registers; each row's part of a step is one 128-byte line); the order of the
// 16-byte pieces inside a buffer is permuted by row so that the fragment reads meet different banks.  GRAM and POLY are symmetric:
// tiles on and below the diagonal, stored twice.
// PARTS 1: hi parts only, stored apart from the lo parts; 2: hi and lo parts, stored together (`place`).
constexpr int product_ring(int tile) { return tile == 128 ? 2 : 3; }  // two workgroups (three of the small tiles) fit a compute unit's 160 KB
template <typename T, int TILE, int PARTS, int MODE, bool LAST>
static __device__ __forceinline__ void product_tile(const Product& p, const long z, const int tm, const int tn, _Float16* const store) {
  constexpr int BK = PARTS == 1 ? 64 : 32;
  constexpr int WT = TILE / 32, PER = TILE * 8 / 256, GR = TILE * PARTS / 16;  // pieces of an operand for each thread; 32-byte groups of a depth's row
  constexpr bool NN = MODE == UPDATE;
  constexpr int RING = product_ring(TILE), LOADS = 2 * PER;
  _Float16 (*const lds)[2][TILE * 64] = reinterpret_cast<_Float16 (*)[2][TILE * 64]>(store);
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, i = l & 15, g = l >> 4;
  const int wm = (w & 1) * (TILE / 2), wn = (w >> 1) * (TILE / 2);
  const long ldP = MODE == GRAM ? p.LP : p.dP, ldQ = MODE == POLY ? p.dP : p.LP;
  const _Float16* P = p.P + z * PARTS * (long)p.dP * ldP;
  const _Float16* Q = p.Q + z * PARTS * (long)p.dP * ldQ;
  const int first = MODE == GRAM ? 0 : p.shift[z];

  // how the 32-byte groups of depth k's row are permuted: depths 0 .. 3 and 8 .. 11, which are read at a time, meet different banks
  auto turn = [](int k) { return GR >= 8 ? (k & 3) | ((k >> 1) & 4) : ((k >> 1) & 1) | ((k >> 2) & 2); };
  // source of each 16-byte piece this lane brings in; a step further on along the depth it is 64 entries on, or BK rows
  const _Float16 *srcP[PER], *srcQ[PER];
  const long stepQ = NN ? (long)BK * PARTS * p.LP : 64;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int s = tid + 256 * u, r = s >> 3, c = (s & 7) ^ (r & 7);
    srcP[u] = P + (tm * TILE + r) * PARTS * ldP + 8 * c;
    if (NN) {
      const int k = s / (2 * GR), pos = s % (2 * GR), gr = (pos >> 1) ^ turn(k);
      srcQ[u] = Q + k * PARTS * ldQ + tn * TILE * PARTS + 16 * gr + 8 * (pos & 1);
    } else {
      srcQ[u] = Q + (tn * TILE + r) * PARTS * ldQ + 8 * c;
    }
  }
  auto bring = [&](int buf) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)srcP[u],
                                       (__attribute__((address_space(3))) void*)&lds[buf][0][(w * 64 + 256 * u) * 8], 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)srcQ[u],
                                       (__attribute__((address_space(3))) void*)&lds[buf][1][(w * 64 + 256 * u) * 8], 16, 0, 0);
      srcP[u] += 64;
      srcQ[u] += stepQ;
    }
  };
  // row r; `half`: the second 32 depths (PARTS 1), the lo parts (PARTS 2)
  auto row = [&](const _Float16* t, int r, int half) { return *(const h8*)(t + r * 64 + 8 * ((4 * half + g) ^ (r & 7))); };
  auto col = [&](const _Float16* t, int c, int half) {  // columns c .. c + 15 of [depth][columns], depths as `row` has them
    typedef __attribute__((address_space(3))) s4* lp;
    const int k = (PARTS == 1 ? 32 * half : 0) + 8 * g + (i >> 2);  // 4 rows for 16 lanes, and the 4 behind them
    const int gr = PARTS == 1 ? c >> 4 : ((c >> 5) << 2) + 2 * half + ((c >> 4) & 1);
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(t + k * TILE * PARTS + 16 * (gr ^ turn(k)) + 4 * (i & 3)));
    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(t + (k + 4) * TILE * PARTS + 16 * (gr ^ turn(k + 4)) + 4 * (i & 3)));
    return __builtin_bit_cast(h8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  f4 acc[WT][WT];  // [m][n]: column (lane % 16) the row of the output, rows its columns
#pragma unroll
  for (int m = 0; m < WT; ++m)
#pragma unroll
    for (int n = 0; n < WT; ++n) acc[m][n] = f4{0, 0, 0, 0};
  const int steps = p.depth / BK;
#pragma unroll
  for (int s = 0; s < RING - 1; ++s)
    if (s < steps) bring(s);
  int buf = 0, next = RING - 1;
  for (int s = 0; s < steps; ++s) {
    // all but the newest RING - 2 steps' loads have arrived (at the end fewer are under way, and all are waited for), and this wave's
    // own reads of the last step have left LDS.  (__syncthreads would wait for every load.)
    if (RING > 2 && s + RING - 1 <= steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((RING - 2) * LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();  // this buffer is filled, and nobody reads the one before it any more
    asm volatile("" ::: "memory");
    if (s + RING - 1 < steps) bring(next);
    const _Float16 *tP = lds[buf][0], *tQ = lds[buf][1];
    buf = buf + 1 == RING ? 0 : buf + 1;
    next = next + 1 == RING ? 0 : next + 1;
    h8 ph[WT], pl[WT];  // PARTS 1: the step's two halves; 2: hi and lo parts
#pragma unroll
    for (int m = 0; m < WT; ++m) {
      const int r = wm + 16 * m + i;
      ph[m] = row(tP, r, 0);
      pl[m] = row(tP, r, 1);
    }
#pragma unroll
    for (int n = 0; n < WT; ++n) {
      const h8 qh = NN ? col(tQ, wn + 16 * n, 0) : row(tQ, wn + 16 * n + i, 0);
      const h8 ql = NN ? col(tQ, wn + 16 * n, 1) : row(tQ, wn + 16 * n + i, 1);
#pragma unroll
      for (int m = 0; m < WT; ++m) {
        if (PARTS == 2) {
          acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ql, ph[m], acc[m][n], 0, 0, 0);
          acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh, pl[m], acc[m][n], 0, 0, 0);
        } else {
          acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ql, pl[m], acc[m][n], 0, 0, 0);
        }
        acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh, ph[m], acc[m][n], 0, 0, 0);
      }
    }
  }
  // The tile goes through LDS, so that what is added is read and the output written by 16 bytes of neighbours a lane (straight from the
  // accumulators, 8 bytes of 16 rows at a time: a third of the time of 4 updates of 768 x 2048, 30 us where this takes 22).  Pieces of 4
  // numbers, permuted so that 16 rows written, neighbours read and 8 rows by 8 columns read all meet different banks.
  constexpr int IT = TILE * TILE / 8 / 256;
  float* tile = reinterpret_cast<float*>(store);
  static_assert(RING * 2 * 64 * 2 >= TILE * 4, "");
  float unscale = p.unscale, add = p.add;
  int k = 0;
  if (MODE != GRAM) {
    k = first > p.k_before ? first - p.k_before : 0;
    if (MODE == POLY) {
      unscale = ldexpf(unscale, -4 * k);
      add = ldexpf(add, -2 * k);
    } else if (!LAST) {
      const int down = (first > p.k_after ? first - p.k_after : 0) - k;
      unscale = ldexpf(unscale, down);
      add = ldexpf(add, down);
    }
  }
  auto spot = [](int r, int c) { return r * TILE + 4 * ((c >> 2) ^ ((r & 15) ^ ((r >> 3) & 6))) + (c & 3); };
  const int ld = MODE == UPDATE ? p.LP : p.dP;
  const long zC = z * PARTS * (long)p.dP * ld;
  h8 dh[IT], dl[IT];
  if (MODE != GRAM) {
#pragma unroll
    for (int u = 0; u < IT; ++u) {
      const int e = tid + 256 * u;
      const long at = zC + place<PARTS>(tm * TILE + e / (TILE / 8), tn * TILE + 8 * (e % (TILE / 8)), ld);
      dh[u] = *(const h8*)(p.Dh + at);
      if (MODE == UPDATE || PARTS == 2) dl[u] = *(const h8*)(p.Dl + at);
    }
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < WT; ++m)
#pragma unroll
    for (int n = 0; n < WT; ++n) *(f4*)(tile + spot(wm + 16 * m + i, wn + 16 * n + 4 * g)) = acc[m][n] * unscale;
  __syncthreads();
  const bool turned = LAST ? p.tall : MODE != UPDATE && tm != tn;
#pragma unroll
  for (int u = 0; u < IT; ++u) {
    const int e = tid + 256 * u, r = e / (TILE / 8), c = 8 * (e % (TILE / 8)), row = tm * TILE + r, col = tn * TILE + c;
    const long at = zC + place<PARTS>(row, col, ld);
    f4 *const p0 = (f4*)(tile + spot(r, c)), *const p1 = (f4*)(tile + spot(r, c + 4));
    f4 v0 = *p0, v1 = *p1;
    if (MODE != GRAM) {
      v0 += add * __builtin_convertvector(__builtin_shufflevector(dh[u], dh[u], 0, 1, 2, 3), f4);
      v1 += add * __builtin_convertvector(__builtin_shufflevector(dh[u], dh[u], 4, 5, 6, 7), f4);
      if (MODE == UPDATE || PARTS == 2) {
        v0 += add * __builtin_convertvector(__builtin_shufflevector(dl[u], dl[u], 0, 1, 2, 3), f4);
        v1 += add * __builtin_convertvector(__builtin_shufflevector(dl[u], dl[u], 4, 5, 6, 7), f4);
      }
      if (LAST) {  // (here, and not in the factors: those could leave fp32's normal numbers where the result does not)
#pragma unroll
        for (int j = 0; j < 4; ++j) v0[j] = ldexpf(v0[j], -k), v1[j] = ldexpf(v1[j], -k);
      }
      if (turned) *p0 = v0, *p1 = v1;
    }
    if (LAST) {
      if (!turned && row < p.d) store_row<T>((T*)p.out + (z * p.d + row) * (long)p.L + col, v0, v1, p.L - col);
    } else {
      h4 h0, l0, h1, l1;
      parts_of(v0, &h0, &l0);
      parts_of(v1, &h1, &l1);
      *(h8*)(p.Ch + at) = __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7);
      if (MODE == UPDATE || PARTS == 2) *(h8*)(p.Cl + at) = __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  if (turned) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < IT; ++u) {  // a wave: 8 columns of 64 rows
      const int e = w + 4 * u, c = 8 * (e % (TILE / 8)) + (l >> 3), r = 64 * (e / (TILE / 8)) + 8 * (l & 7), row = tm * TILE + r, col = tn * TILE + c;
      f4 v0, v1;
#pragma unroll
      for (int j = 0; j < 4; ++j) v0[j] = tile[spot(r + j, c)], v1[j] = tile[spot(r + 4 + j, c)];
      if (LAST) {
        if (col < p.L) store_row<T>((T*)p.out + (z * p.L + col) * (long)p.d + row, v0, v1, p.d - row);
      } else {
        const long to = zC + place<PARTS>(col, row, ld);
        h4 h0, l0, h1, l1;
        parts_of(v0, &h0, &l0);
        parts_of(v1, &h1, &l1);
        *(h8*)(p.Ch + to) = __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7);
        if (PARTS == 2) *(h8*)(p.Cl + to) = __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    }
  }
}

template <typename T, int TILE, int PARTS, int MODE, bool LAST>
__global__ __launch_bounds__(256, 2) void orth_product_kernel(Product p) {
  __shared__ __attribute__((aligned(16))) _Float16 lds[product_ring(TILE) * 2 * TILE * 64];
  const long per = (p.whole + 7) >> 3, first = 8 * per;
  const bool quarter = TILE == 128 && blockIdx.x >= first;
  const long part = blockIdx.x - first, work = quarter ? p.whole + (part >> 2) : (blockIdx.x & 7) * per + (blockIdx.x >> 3);  // neighbours on one die
  if (work >= (quarter ? p.works : p.whole)) return;
  const long tiles = p.works / p.n, z = work / tiles;
  const int x = (int)(work - z * tiles);
  int tm, tn;
  if (MODE == UPDATE) {  // bands of 8 tiles, so that what one die works on shares rows and columns
    const int width = 8 * p.tiles_n, band = x / width, in = x - band * width;
    const int rows = p.tiles_m - 8 * band < 8 ? p.tiles_m - 8 * band : 8;
    tm = 8 * band + in % rows;
    tn = in / rows;
  } else {
    tm = (int)((sqrtf(8.f * x + 1.f) - 1.f) * 0.5f);
    while ((tm + 1) * (tm + 2) / 2 <= x) ++tm;
    while (tm * (tm + 1) / 2 > x) --tm;
    tn = x - tm * (tm + 1) / 2;
  }
  if (quarter) {
    tm = 2 * tm + (int)(part >> 1 & 1);
    tn = 2 * tn + (int)(part & 1);
    if (MODE == UPDATE || tn <= tm) product_tile<T, 64, PARTS, MODE, LAST>(p, z, tm, tn, lds);
  } else {
    product_tile<T, TILE, PARTS, MODE, LAST>(p, z, tm, tn, lds);
  }
}

struct PartsPlan { int dP, LP; size_t x, aa, norm, shift; };
PartsPlan parts_plan(const KfOrthArgs& a) {
  PartsPlan p;
  const int d = a.rows < a.cols ? a.rows : a.cols, L = a.rows < a.cols ? a.cols : a.rows;
  p.dP = (d + 127) / 128 * 128;
  p.LP = (L + 127) / 128 * 128;
  p.x = kf_seq_round((size_t)a.n * p.dP * p.LP * 2);
  p.aa = kf_seq_round((size_t)a.n * p.dP * p.dP * 2);
  p.norm = norm_bytes(a);
  p.shift = kf_seq_round((size_t)a.n * 4);
  return p;
}

// one product: tiles of 128 where they fill the card, else of 64
template <typename T, int PARTS, int MODE, bool LAST>
void launch_product(const kf_handle* h, Product& p, hipStream_t stream) {
  const long cu = h->n_cu > 0 ? h->n_cu : 256;
  const int cols = MODE == UPDATE ? p.L : p.d;
  auto count = [&](int tile) {
    p.tiles_m = (p.d + tile - 1) / tile;
    p.tiles_n = (cols + tile - 1) / tile;
    p.works = p.n * (MODE == UPDATE ? (long)p.tiles_m * p.tiles_n : p.tiles_m * (p.tiles_m + 1L) / 2);
  };
  p.depth = ((MODE == GRAM ? p.L : p.d) + 63) / 64 * 64;
  count(128);
  const bool small = p.works < cu;
  if (small) count(64);
  // (A product by tiles of 64 that tiles of 128 would leave compute units without: 4 of 768 x 768, 312 tiles
  // 15 and 8 us, 84 tiles 24 and 13.  Two groups of waves
  // that share the depth of a tile of 64 gain nothing: 15 us both.)
  //
  // Two tiles of 128 at a time on each compute unit: a few that are left over would take one more round all by themselves, and are cut
  // in four (4096 x 4096, 528 tiles on 256 units: 250 us, with the last 16 cut in four 199).  Not
  // where they are many: 384 tiles of 4 x 768 x 2048 22 us, with a third of them cut 28.
  const long over = small ? 0 : p.works % (2 * cu);
  p.whole = p.works > over && 4 * over <= cu ? p.works - over : p.works;
  const dim3 grid((unsigned)(8 * ((p.whole + 7) / 8) + 4 * (p.works - p.whole)));
  if (small) hipLaunchKernelGGL((orth_product_kernel<T, 64, PARTS, MODE, LAST>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((orth_product_kernel<T, 128, PARTS, MODE, LAST>), grid, dim3(256), 0, stream, p);
}

template <typename T, int PARTS>
int launch_parts(kf_handle* h, const KfOrthArgs& a, const PartsPlan& pl, void* ws, hipStream_t stream) {
  char* w = (char*)ws;
  double* norm = (double*)w; w += pl.norm;
  int* shift = (int*)w; w += pl.shift;
  _Float16 *X[2][2], *A[2], *B[2];  // hi, lo
  // (stored together, the lo parts are 32 entries behind the hi parts)
  auto take = [&](size_t bytes, _Float16** q) {
    q[0] = (_Float16*)w;
    q[1] = PARTS == 2 ? q[0] + 32 : (_Float16*)(w + bytes);
    w += 2 * bytes;
  };
  take(pl.x, X[0]); take(pl.x, X[1]); take(pl.aa, A); take(pl.aa, B);
  const long size = (long)a.rows * a.cols;
  const int parts = norm_parts(size);
  Product p;
  p.n = (int)a.n;
  p.tall = a.rows > a.cols;
  p.d = p.tall ? a.cols : a.rows;
  p.L = p.tall ? a.rows : a.cols;
  p.dP = pl.dP; p.LP = pl.LP;
  p.out = a.X;
  p.shift = shift;
  hipLaunchKernelGGL(orth_norm_kernel<T>, dim3(parts, (unsigned)a.n), dim3(256), 0, stream, (const T*)a.M, size, norm);
  hipLaunchKernelGGL((orth_parts_kernel<T, PARTS>), dim3(pl.LP / 64, pl.dP / 64, (unsigned)a.n), dim3(256), 0, stream, a, norm, parts, pl.dP, pl.LP, X[0][0], X[0][1],
                     shift);
  double grown = 0.;  // log2 of what the steps so far can have multiplied a singular value by
  for (int s = 0; s < a.steps; ++s) {
    const double ca = a.coef[s][0], cb = a.coef[s][1], cc = a.coef[s][2];
    const int from = s & 1, to = from ^ 1;
    const double top = a.top[s];
    // |B| <= the largest |b u + c u^2|, and a singular value grows by at most the largest |a + b u + c u^2|, u = s^2 <= top^2
    double bound = fabs(top * top * (cb + cc * top * top)), most = fmax(fabs(ca), fabs(ca + top * top * (cb + cc * top * top)));
    if (cc != 0.0 && -cb / (2 * cc) > 0 && -cb / (2 * cc) < top * top) {
      bound = fmax(bound, fabs(cb * cb / (4 * cc)));
      most = fmax(most, fabs(ca - cb * cb / (4 * cc)));
    }
    p.k_before = (int)ceil(grown);
    grown += fmax(log2(most), 0.);
    p.k_after = (int)ceil(grown);
    int e = 0;
    frexp(fmax(bound, 1e-6), &e);
    const double scale_b = ldexp(1.0, 14 - e);  // |B| comes to at most 2^14: room for what A's rounding adds
    p.P = p.Q = X[from][0];
    p.Ch = A[0]; p.Cl = A[1];
    p.Dh = p.Dl = nullptr;
    p.unscale = (float)(SCALE_A / ((double)SCALE_X * SCALE_X)); p.add = 0.f;
    launch_product<T, PARTS, GRAM, false>(h, p, stream);
    p.P = p.Q = p.Dh = A[0]; p.Dl = A[1];
    p.Ch = B[0]; p.Cl = B[1];
    p.unscale = (float)(cc * scale_b / ((double)SCALE_A * SCALE_A)); p.add = (float)(cb * scale_b / SCALE_A);
    launch_product<T, PARTS, POLY, false>(h, p, stream);
    p.P = B[0];
    p.Q = p.Dh = X[from][0]; p.Dl = X[from][1];
    p.Ch = X[to][0]; p.Cl = X[to][1];
    const bool last = s + 1 == a.steps;
    p.unscale = (float)((last ? 1.0 / SCALE_X : 1.0) / scale_b); p.add = (float)(last ? ca / SCALE_X : ca);
    if (last) launch_product<T, PARTS, UPDATE, true>(h, p, stream);
    else launch_product<T, PARTS, UPDATE, false>(h, p, stream);
  }
  KF_HIP_CHECK(h, hipGetLastError());
  return KF_OK;
}

// ------------------------------------------------------------------------------------------------ fp64
__global__ __launch_bounds__(256) void orth_scale64_kernel(KfOrthArgs a, const double* part, int parts, double* X) {
  __shared__ double red[4];
  const long e = (long)blockIdx.x * 256 + threadIdx.x, size = (long)a.rows * a.cols, z = blockIdx.y, i = z * size + e;
  const double f = norm_factor(part + z * parts, parts, a.eps, red);
  if (e >= size) return;
  X[a.rows > a.cols ? z * size + (e % a.cols) * a.rows + e / a.cols : i] = ((const double*)a.M)[i] * f;
}

// out (m x n) = alpha A B + beta D: A (m x k) row-major, B (k x n) row-major or (NT) given as (n x k); `tall`: stored transposed.  64 x 64 of
// it for each workgroup of 2 x 2 waves, v_mfma_f64_16x16x4 on operands in LDS, 32 depths at a time, the 64 behind them on their way (with a
// wait for each load, 128 x 128: 318 us instead of 195).  SYM: the
// result is symmetric, tiles on and below the diagonal, stored twice.  Where there are few tiles the depth is cut into `slices`, each of
// which leaves its sum in `parts`, [slices][matrices][m n].
struct Product64 {
  int m, n, k, tiles_n, slices, tall;
  const double *A, *B, *D;
  double *out, *parts;
  double alpha, beta;
};
template <bool NT, bool SYM>
__global__ __launch_bounds__(256) void orth_product64_kernel(Product64 p) {
  typedef Tile<double> Q;
  typedef Q::type V;
  typedef V V16 __attribute__((aligned(16)));
  constexpr int BK = 32, SA = BK + 2, SB = NT ? SA : 66;  // rows an odd number of 16-byte pieces apart
  __shared__ __attribute__((aligned(16))) double sa[64 * SA], sb[NT ? 64 * SA : BK * SB];
  const long z = blockIdx.z;
  const double *A = p.A + z * p.m * (long)p.k, *B = p.B + z * p.n * (long)p.k;
  int tm, tn;
  const int x = blockIdx.x;
  if (SYM) {
    tm = (int)((sqrtf(8.f * x + 1.f) - 1.f) * 0.5f);
    while ((tm + 1) * (tm + 2) / 2 <= x) ++tm;
    while (tm * (tm + 1) / 2 > x) --tm;
    tn = x - tm * (tm + 1) / 2;
  } else {
    tm = x / p.tiles_n;
    tn = x - tm * p.tiles_n;
  }
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, i = l & 15, g = l >> 4, r0 = 64 * tm, c0 = 64 * tn;
  const int wm = 32 * (w & 1), wn = 32 * (w >> 1);
  // 4 neighbours of a row along the depth (or, NN, along B's columns), and, when they are needed (a select behind the load would wait for
  // it), zeros for what is outside
  auto four = [](const double* p, int row, int rows, int col, int cols) {
    V v;
    const double* q = p + (long)(row < rows ? row : rows - 1) * cols;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = q[col + e < cols ? col + e : cols - 1];
    return v;
  };
  auto inside = [](V v, int row, int rows, int col, int cols) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = row < rows && col + e < cols ? v[e] : 0.;
    return v;
  };
  const int ar = tid >> 3, ak = 4 * (tid & 7), bk = tid >> 4, bc = 4 * (tid & 15);
  const int blocks = (p.k + BK - 1) / BK, per = (blocks + p.slices - 1) / p.slices;
  const int first = blockIdx.y * per, last = first + per < blocks ? first + per : blocks;
  V va[2][2], vb[2][2];
  auto load = [&](int b, V (&x)[2], V (&y)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      x[u] = four(A, r0 + ar + 32 * u, p.m, BK * b + ak, p.k);
      y[u] = NT ? four(B, c0 + ar + 32 * u, p.n, BK * b + ak, p.k) : four(B, BK * b + bk + 16 * u, p.k, c0 + bc, p.n);
    }
  };
  V acc[2][2] = {};
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (first + h < last) load(first + h, va[h], vb[h]);
  for (int b0 = first; b0 < last; b0 += 2) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (b0 + h >= last) break;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k0 = BK * (b0 + h);
        *reinterpret_cast<V16*>(sa + (ar + 32 * u) * SA + ak) = inside(va[h][u], r0 + ar + 32 * u, p.m, k0 + ak, p.k);
        *reinterpret_cast<V16*>(sb + (NT ? (ar + 32 * u) * SB + ak : (bk + 16 * u) * SB + bc)) =
            NT ? inside(vb[h][u], c0 + ar + 32 * u, p.n, k0 + ak, p.k) : inside(vb[h][u], k0 + bk + 16 * u, p.k, c0 + bc, p.n);
      }
      // (not __syncthreads, which would wait for the loads under way)
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      load(b0 + h + 2 < last ? b0 + h + 2 : b0 + h, va[h], vb[h]);
#pragma unroll
      for (int kk = 0; kk < BK; kk += 16) {
        V pa[2], qb[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          pa[t] = *reinterpret_cast<const V16*>(sa + (wm + 16 * t + i) * SA + kk + 4 * g);
          if (NT) {
            qb[t] = *reinterpret_cast<const V16*>(sb + (wn + 16 * t + i) * SB + kk + 4 * g);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) qb[t][e] = sb[(kk + 4 * g + e) * SB + wn + 16 * t + i];
          }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int u = 0; u < 2; ++u) acc[t][u] = Q::mma(pa[t], qb[u], acc[t][u], 16);
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
  }
  const double* D = p.D + z * p.m * (long)p.n;
  double* out = p.slices > 1 ? p.parts + (blockIdx.y * (long)gridDim.z + z) * p.m * p.n : p.out + z * p.m * (long)p.n;
  const bool tall = p.tall && p.slices == 1;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = r0 + wm + 16 * t + Q::row(e, g), c = c0 + wn + 16 * u + i;
        if (r >= p.m || c >= p.n) continue;
        double v = acc[t][u][e];
        if (p.slices == 1) v = p.alpha * v + (p.beta != 0. ? p.beta * D[(long)r * p.n + c] : 0.);
        out[tall ? (long)c * p.m + r : (long)r * p.n + c] = v;
        if (SYM && tm != tn) out[(long)c * p.n + r] = v;
      }
}
__global__ __launch_bounds__(256) void orth_slices64_kernel(Product64 p, long size) {
  const long e = (long)blockIdx.x * 256 + threadIdx.x;
  if (e >= size) return;
  double s = 0.;
  for (int x = 0; x < p.slices; ++x) s += p.parts[x * size + e];
  const long cells = (long)p.m * p.n, z = e / cells, i = e - z * cells, r = i / p.n, c = i - r * p.n;
  p.out[p.tall ? z * cells + c * p.m + r : e] = p.alpha * s + (p.beta != 0. ? p.beta * p.D[e] : 0.);
}

// how a product's depth is cut where it has few tiles: two workgroups for each compute unit, at least 128 depths for each (one matrix of
// 100 x 4000: 1173 us uncut, 255 cut; one of 512 x 512: 498 and 295; its library products take 571 and 295)
int slices64(const kf_handle* h, long n, int d, int cols, int depth) {
  const long cu = h->n_cu > 0 ? h->n_cu : 256, td = (d + 63) / 64, tiles = n * (cols == d ? td * (td + 1) / 2 : td * ((cols + 63) / 64));
  const long most = depth / 128, want = 2 * cu / tiles;
  const long s = want < most ? want : most;
  return s < 1 ? 1 : (int)s;
}
size_t cut64(const kf_handle* h, long n, int d, int L) {  // bytes for the parts of the product that needs most
  size_t most = 0;
  auto take = [&](int cols, int depth) {
    const int s = slices64(h, n, d, cols, depth);
    const size_t bytes = s > 1 ? (size_t)s * n * d * cols * 8 : 0;
    most = bytes > most ? bytes : most;
  };
  take(d, L);
  take(d, d);
  take(L, d);
  return kf_seq_round(most);
}

int launch64(kf_handle* h, const KfOrthArgs& a, void* ws, hipStream_t stream) {
  const bool tall = a.rows > a.cols;
  const int d = tall ? a.cols : a.rows, L = tall ? a.rows : a.cols;
  const size_t big = kf_seq_round((size_t)a.n * d * L * 8), small = kf_seq_round((size_t)a.n * d * d * 8);
  char* w = (char*)ws;
  double* norm = (double*)w; w += norm_bytes(a);
  double* X = (double*)w; w += big;
  double* Y = (double*)w; w += big;
  double* A = (double*)w; w += small;
  double* B = (double*)w; w += small;
  double* cut = (double*)w;
  const long size = (long)d * L;
  const int parts = norm_parts(size);
  hipLaunchKernelGGL(orth_norm_kernel<double>, dim3(parts, (unsigned)a.n), dim3(256), 0, stream, (const double*)a.M, size, norm);
  hipLaunchKernelGGL(orth_scale64_kernel, dim3((unsigned)((size + 255) / 256), (unsigned)a.n), dim3(256), 0, stream, a, norm, parts, X);
  const unsigned td = (d + 63) / 64, tl = (L + 63) / 64, z = (unsigned)a.n;
  auto run = [&](Product64 p, bool symmetric) {
    p.tiles_n = (int)tl;
    p.parts = cut;
    p.slices = symmetric ? slices64(h, a.n, d, d, p.k) : slices64(h, a.n, d, L, p.k);
    if (symmetric) hipLaunchKernelGGL((orth_product64_kernel<true, true>), dim3(td * (td + 1) / 2, p.slices, z), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((orth_product64_kernel<false, false>), dim3(td * tl, p.slices, z), dim3(256), 0, stream, p);
    const long cells = a.n * p.m * (long)p.n;
    if (p.slices > 1) hipLaunchKernelGGL(orth_slices64_kernel, dim3((unsigned)((cells + 255) / 256)), dim3(256), 0, stream, p, cells);
  };
  for (int s = 0; s < a.steps; ++s) {
    const bool last = s + 1 == a.steps;
    run({d, d, L, 0, 1, 0, X, X, A, A, nullptr, 1., 0.}, true);
    run({d, d, d, 0, 1, 0, A, A, A, B, nullptr, a.coef[s][2], a.coef[s][1]}, true);
    run({d, L, d, 0, 1, last && tall, B, X, X, last ? (double*)a.X : Y, nullptr, 1., a.coef[s][0]}, false);
    double* t = X; X = Y; Y = t;
  }
  KF_HIP_CHECK(h, hipGetLastError());
  return KF_OK;
}

template <typename T>
int launch_t(kf_handle* h, const KfOrthArgs& a, void* ws, hipStream_t stream) {
  if (fits_wave(a)) return launch_wave<T>(h, a, stream);
  const ChipPlan c = chip_plan(a);
  if (c.fits) return launch_chip<T>(h, a, c, stream);
  return launch_parts<T, std::is_same<T, __hip_bfloat16>::value ? 1 : 2>(h, a, parts_plan(a), ws, stream);
}

}  // namespace

bool kf_orthogonalise_on_chip(const KfOrthArgs& a) { return fits_wave(a) || chip_plan(a).fits; }

size_t kf_orthogonalise_ws(const kf_handle* h, const KfOrthArgs& a) {
  if (kf_orthogonalise_on_chip(a)) return 0;
  const size_t d = a.rows < a.cols ? a.rows : a.cols, L = a.rows < a.cols ? a.cols : a.rows;
  if (a.dtype == KF_DTYPE_F64)
    return norm_bytes(a) + 2 * kf_seq_round((size_t)a.n * d * L * 8) + 2 * kf_seq_round((size_t)a.n * d * d * 8) +
           cut64(h, a.n, (int)d, (int)L);
  const PartsPlan p = parts_plan(a);
  return p.norm + p.shift + 4 * p.x + 4 * p.aa;
}

int kf_launch_orthogonalise(kf_handle* h, const KfOrthArgs& a, void* ws, hipStream_t stream) {
  switch (a.dtype) {
    case KF_DTYPE_F64: {
      if (fits_wave(a)) return launch_wave<double>(h, a, stream);
      const ChipPlan c = chip_plan(a);
      if (!c.fits) return launch64(h, a, ws, stream);
      return launch_chip<double>(h, a, c, stream);
    }
    case KF_DTYPE_F32: return launch_t<float>(h, a, ws, stream);
    case KF_DTYPE_BF16: return launch_t<__hip_bfloat16>(h, a, ws, stream);
    default: return launch_t<__half>(h, a, ws, stream);
  }
}
