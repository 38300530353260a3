// Activations kept in 8 bits for the backward pass (gfx950): packing, the root-mean-square
// norm that writes its normalised rows packed, that norm's gradients, and a linear layer's
// weight gradient from a packed input.
//
// The packed form of a row is E4M3 numbers with one power-of-two scale 2^k for every block of
// 128 consecutive features, k the smallest integer with max |x| <= 448 * 2^k in the block.
// A scale that is a power of two makes the scaling exact in both directions, the scale one
// byte, and every packed value exact in bf16 (4 significant bits, exponents -126 .. 127).
//
// A block is 16 lanes of 8 features each: one DPP row of a wavefront, so the block maximum is
// four row rotations and needs neither LDS nor a barrier.
//
// Entry points are declared and documented in include/torchft_amd.h.

#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include "errors.h"
#include "torchft_amd.h"

namespace {

using tft::fail;

constexpr int kBlock = 128;      // features that share a scale
constexpr int kMinExponent = 10;   // 2^-117: times E4M3's least step 2^-9 still a normal bf16
constexpr int kMaxExponent = 246;  // 2^119: times 448 still finite in bf16
constexpr uint32_t kInfBits = 0x7f800000u;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));  // rows start where they start: gfx950 loads
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));  // 128 bits from any address
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// 16 or 8 bytes; S: past the caches, for what is not used again soon.  One function per alignment:
// a template's type parameter would drop it.
#define TFT_ACCESS(NAME, TYPE)                                      \
  template <bool S>                                                 \
  __device__ inline TYPE load_##NAME(const void* p) {               \
    const TYPE* q = static_cast<const TYPE*>(p);                    \
    if constexpr (S) return __builtin_nontemporal_load(q);          \
    return *q;                                                      \
  }                                                                 \
  template <bool S>                                                 \
  __device__ inline void store_##NAME(void* p, TYPE v) {            \
    TYPE* q = static_cast<TYPE*>(p);                                \
    if constexpr (S) __builtin_nontemporal_store(v, q);             \
    else *q = v;                                                    \
  }
TFT_ACCESS(16_a2, u32x4_a2)
TFT_ACCESS(16_a4, u32x4_a4)
TFT_ACCESS(8, u32x2)
#undef TFT_ACCESS

// ---------------------------------------------------------------------------
// Element types: eight consecutive elements of a row as fp32
// ---------------------------------------------------------------------------
struct F32 {
  typedef float elem_t;
  typedef struct { u32x4 w[2]; } raw_t;
  template <bool S>
  __device__ static inline raw_t load(const elem_t* p) {
    raw_t r;
    r.w[0] = load_16_a4<S>(p);
    r.w[1] = load_16_a4<S>(p + 4);
    return r;
  }
  __device__ static inline void widen(const raw_t& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.w[i >> 2][i & 3]);
  }
  __device__ static inline raw_t narrow(const float (&v)[8]) {
    raw_t r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i >> 2][i & 3] = __float_as_uint(v[i]);
    return r;
  }
  template <bool S>
  __device__ static inline void store(elem_t* p, const raw_t& r) {
    store_16_a4<S>(p, r.w[0]);
    store_16_a4<S>(p + 4, r.w[1]);
  }
  __device__ static inline float widen1(elem_t x) { return x; }
  __device__ static inline elem_t narrow1(float x) { return x; }
  // a packed value as this type: every one of them is an fp32 number
  __device__ static inline float in_range(float x) { return x; }
};

struct BF16 {
  typedef uint16_t elem_t;
  typedef struct { u32x4 w[1]; } raw_t;
  template <bool S>
  __device__ static inline raw_t load(const elem_t* p) {
    raw_t r;
    r.w[0] = load_16_a2<S>(p);
    return r;
  }
  __device__ static inline void widen(const raw_t& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(r.w[0][i] << 16);
      v[2 * i + 1] = __uint_as_float(r.w[0][i] & 0xffff0000u);
    }
  }
  __device__ static inline raw_t narrow(const float (&v)[8]) {
    raw_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 pair = {v[2 * i], v[2 * i + 1]};
      r.w[0][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, bf16x2));
    }
    return r;
  }
  template <bool S>
  __device__ static inline void store(elem_t* p, const raw_t& r) {
    store_16_a2<S>(p, r.w[0]);
  }
  __device__ static inline float widen1(elem_t x) { return __uint_as_float((uint32_t)x << 16); }
  __device__ static inline elem_t narrow1(float x) {
    return __builtin_bit_cast(uint16_t, (__bf16)x);
  }
  __device__ static inline float in_range(float x) { return x; }
};

struct F16 {
  typedef uint16_t elem_t;
  typedef struct { u32x4 w[1]; } raw_t;
  template <bool S>
  __device__ static inline raw_t load(const elem_t* p) {
    raw_t r;
    r.w[0] = load_16_a2<S>(p);
    return r;
  }
  __device__ static inline float widen1(elem_t x) { return __half2float(__ushort_as_half(x)); }
  __device__ static inline elem_t narrow1(float x) {
    // keeps the compiler from folding a multiply-add into the conversion, which would round
    // once where the fp32 result rounds first
    asm volatile("" : "+v"(x));
    return __half_as_ushort(__float2half_rn(x));
  }
  __device__ static inline void widen(const raw_t& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = widen1((uint16_t)(r.w[0][i] & 0xffffu));
      v[2 * i + 1] = widen1((uint16_t)(r.w[0][i] >> 16));
    }
  }
  __device__ static inline raw_t narrow(const float (&v)[8]) {
    raw_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r.w[0][i] = (uint32_t)narrow1(v[2 * i]) | ((uint32_t)narrow1(v[2 * i + 1]) << 16);
    return r;
  }
  template <bool S>
  __device__ static inline void store(elem_t* p, const raw_t& r) {
    store_16_a2<S>(p, r.w[0]);
  }
  // a packed value may have been rounded up past fp16's largest number
  __device__ static inline float in_range(float x) {
    return fabsf(x) > 65504.0f ? copysignf(65504.0f, x) : x;  // NaN stays NaN
  }
};

// Elements n .. 7 of the eight lie behind the row's end: they are not touched and count as zero.
template <typename T, bool S = false>
__device__ inline typename T::raw_t load_row(const typename T::elem_t* p, int n) {
  if (n >= 8) return T::template load<S>(p);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? T::widen1(p[i]) : 0.0f;
  return T::narrow(v);
}

template <typename T, bool S = false>
__device__ inline void store_row(typename T::elem_t* p, const float (&v)[8], int n) {
  const typename T::raw_t r = T::narrow(v);
  if (n >= 8) {
    T::template store<S>(p, r);
    return;
  }
  constexpr int kPerWord = 4 / sizeof(typename T::elem_t);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) {
      const uint32_t word = r.w[(i / kPerWord) >> 2][(i / kPerWord) & 3];
      if constexpr (kPerWord == 1) p[i] = __uint_as_float(word);
      else p[i] = (typename T::elem_t)(word >> (16 * (i & 1)));
    }
}

// Weights are given in the activations' type or in fp32.
template <typename T>
__device__ inline void load_weight(const void* w, bool is_f32, int64_t col, int n, float (&v)[8]) {
  if (is_f32) {
    F32::widen(load_row<F32>(static_cast<const float*>(w) + col, n), v);
  } else {
    T::widen(load_row<T>(static_cast<const typename T::elem_t*>(w) + col, n), v);
  }
}

// ---------------------------------------------------------------------------
// Reductions over lanes
// ---------------------------------------------------------------------------
template <int N>
__device__ inline uint32_t row_rotate(uint32_t x) {  // within the 16 lanes of a DPP row
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + N, 0xf, 0xf, false);
}

__device__ inline uint32_t max_of_16(uint32_t x) {
  x = max(x, row_rotate<8>(x));
  x = max(x, row_rotate<4>(x));
  x = max(x, row_rotate<2>(x));
  return max(x, row_rotate<1>(x));
}

__device__ inline float sum_of_wave(float x) {
  x += __uint_as_float(row_rotate<8>(__float_as_uint(x)));
  x += __uint_as_float(row_rotate<4>(__float_as_uint(x)));
  x += __uint_as_float(row_rotate<2>(__float_as_uint(x)));
  x += __uint_as_float(row_rotate<1>(__float_as_uint(x)));
  x += __shfl_xor(x, 16, 64);
  x += __shfl_xor(x, 32, 64);
  return x;
}

// Sum over a workgroup of up to 16 wavefronts; every lane gets it.  `part` holds 16 floats of LDS
// and must not be in use from an earlier call (the caller alternates between two).
__device__ inline float sum_of_workgroup(float x, float* part) {
  x = sum_of_wave(x);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  x = part[0];
  for (uint32_t i = 1; i < blockDim.x / 64; ++i) x += part[i];
  return x;
}

// ---------------------------------------------------------------------------
// E4M3 with a power-of-two scale
// ---------------------------------------------------------------------------
__device__ inline uint32_t max_bits(const float (&v)[8]) {  // bits of max |v|; NaN counts as most
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

__device__ inline int exponent_for(uint32_t bits) {
  // (bits + 0x1fffff) >> 23 is the exponent of bits, one more where the significand is over
  // 1.75 = 448 / 2^8
  const int e = (int)((bits + 0x1fffffu) >> 23) - 8;
  return min(max(e, kMinExponent), kMaxExponent);
}

// Eight values of one lane of a block's sixteen -> 8 bytes and the block's biased exponent.
// All sixteen lanes call it together.
__device__ inline u32x2 quantise(float (&v)[8], int* exponent) {
  uint32_t top = max_of_16(max_bits(v));
  constexpr uint32_t kMost = ((uint32_t)(kMaxExponent + 8) << 23) | 0x600000u;  // 448 * 2^119
  if (top > kMost) {  // the same for all sixteen: infinities, NaN or next to fp32's largest
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
      if (b >= kInfBits) v[i] = __uint_as_float(0x7fc00000u);  // E4M3 has a NaN and no infinity
      else m = max(m, b);
    }
    top = max_of_16(m);
    const float most = __uint_as_float(kMost);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (fabsf(v[i]) > most) v[i] = copysignf(most, v[i]);
  }
  *exponent = exponent_for(top);
  const float inverse = __uint_as_float((uint32_t)(254 - *exponent) << 23);
  u32x2 q;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] * inverse, v[4 * i + 1] * inverse, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] * inverse, v[4 * i + 3] * inverse, w, true);
    q[i] = (uint32_t)w;
  }
  return q;
}

__device__ inline float scale_of(uint32_t exponent) { return __uint_as_float(exponent << 23); }

__device__ inline void dequantise(const u32x2& q, float scale, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i], false);
    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i], true);
    v[4 * i] = lo[0] * scale;
    v[4 * i + 1] = lo[1] * scale;
    v[4 * i + 2] = hi[0] * scale;
    v[4 * i + 3] = hi[1] * scale;
  }
}

// n / d for n < 2^31 by a multiplication (d >= 1): Granlund and Montgomery, "Division by invariant
// integers using multiplication", 1994
struct Divider {
  uint32_t d, magic, shift;
};

Divider make_divider(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {d, (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}

__device__ inline uint32_t divide(uint32_t n, const Divider& d) {
  return (__umulhi(n, d.magic) + n) >> d.shift;
}

// ---------------------------------------------------------------------------
// Pack and unpack
// ---------------------------------------------------------------------------
struct PackArgs {
  const void* x;
  uint8_t* values;
  uint8_t* exponents;
  int64_t features, row_stride, pitch;
  uint32_t blocks;  // of all rows
  Divider per_row;
};

constexpr int kPackThreads = 256;
constexpr int kPackUnroll = 4;
constexpr int kUnpackUnroll = 2;
constexpr int kPackBlocks = kPackThreads / 16 * kPackUnroll;  // blocks per workgroup
constexpr int kUnpackBlocks = kPackThreads / 16 * kUnpackUnroll;

// Bound by memory: an element is read once and one byte written.  8192 x 14336 bf16 (353 MB)
// takes 54-55 us, 6.4-6.5 TB/s; two or one blocks a lane instead of four 55 and 61 us.
template <typename T, bool S>
__global__ __launch_bounds__(kPackThreads) void pack_kernel(PackArgs a) {
  const int lane = threadIdx.x & 15;
  const uint32_t first = blockIdx.x * (uint32_t)kPackBlocks + (threadIdx.x >> 4);
  const typename T::elem_t* x = static_cast<const typename T::elem_t*>(a.x);
  typename T::raw_t raw[kPackUnroll];
  uint32_t row[kPackUnroll];
  int64_t col[kPackUnroll];
#pragma unroll
  for (int u = 0; u < kPackUnroll; ++u) {
    const uint32_t b = first + u * (kPackThreads / 16);
    row[u] = divide(min(b, a.blocks - 1), a.per_row);
    col[u] = (int64_t)(min(b, a.blocks - 1) - row[u] * a.per_row.d) * kBlock + lane * 8;
    const int64_t left = b < a.blocks ? a.features - col[u] : 0;
    raw[u] = load_row<T, S>(x + (int64_t)row[u] * a.row_stride + col[u], (int)min(left, (int64_t)8));
  }
#pragma unroll
  for (int u = 0; u < kPackUnroll; ++u) {
    const uint32_t b = first + u * (kPackThreads / 16);
    if (b >= a.blocks) return;  // the same for a block's sixteen lanes
    float v[8];
    T::widen(raw[u], v);
    int e;
    const u32x2 q = quantise(v, &e);
    if (col[u] < a.pitch)
      *reinterpret_cast<u32x2*>(a.values + (int64_t)row[u] * a.pitch + col[u]) = q;
    if (lane == 0) a.exponents[b] = (uint8_t)e;
  }
}

struct UnpackArgs {
  void* out;
  const uint8_t* values;
  const uint8_t* exponents;
  const void* column_scale;
  int64_t features, pitch;
  uint32_t blocks;
  Divider per_row;
};

// Bound by memory like packing: 8192 x 14336 to bf16 takes 56 us, 6.3 TB/s (four blocks a lane 58).
// W: type of the column scale
template <typename T, typename W, bool S>
__global__ __launch_bounds__(kPackThreads) void unpack_kernel(UnpackArgs a) {
  const int lane = threadIdx.x & 15;
  const uint32_t first = blockIdx.x * (uint32_t)kUnpackBlocks + (threadIdx.x >> 4);
  typename T::elem_t* out = static_cast<typename T::elem_t*>(a.out);
  u32x2 q[kUnpackUnroll];
  uint32_t e[kUnpackUnroll], row[kUnpackUnroll];
  int64_t col[kUnpackUnroll];
#pragma unroll
  for (int u = 0; u < kUnpackUnroll; ++u) {
    const uint32_t b = min(first + u * (kPackThreads / 16), a.blocks - 1);
    row[u] = divide(b, a.per_row);
    col[u] = (int64_t)(b - row[u] * a.per_row.d) * kBlock + lane * 8;
    q[u] = u32x2{0, 0};
    if (col[u] < a.pitch)
      q[u] = *reinterpret_cast<const u32x2*>(a.values + (int64_t)row[u] * a.pitch + col[u]);
    e[u] = a.exponents[b];
  }
#pragma unroll
  for (int u = 0; u < kUnpackUnroll; ++u) {
    if (first + u * (kPackThreads / 16) >= a.blocks) return;
    const int n = (int)min(a.features - col[u], (int64_t)8);
    if (n <= 0) continue;
    float v[8];
    dequantise(q[u], scale_of(e[u]), v);
    if (a.column_scale) {
      float w[8];
      load_weight<W>(a.column_scale, false, col[u], n, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= w[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = T::in_range(v[i]);
    }
    store_row<T, S>(out + (int64_t)row[u] * a.features + col[u], v, n);
  }
}

// ---------------------------------------------------------------------------
// Root-mean-square norm
// ---------------------------------------------------------------------------
struct NormArgs {
  const void* x;
  const void* residual;  // or NULL
  const void* weight;    // or NULL
  void* y;
  void* h;               // or NULL
  uint8_t* values;       // or NULL: nothing is packed
  uint8_t* exponents;
  float* rstd;           // or NULL
  uint32_t rows;
  int features;
  int64_t x_stride, residual_stride, pitch;
  int weight_is_f32;
  float eps;
};

// The row is read once and stays in registers between the sum of squares and the outputs.  Up to
// 512 features are one wavefront's, four rows to a workgroup and no barrier (Four); longer rows
// take a workgroup of as many wavefronts as it has 512 features, from 8192 on twice as many
// features a lane (C = 2).  One chunk of eight features a lane keeps the most wavefronts, and so
// the most loads, in flight: 16384 x 4096 bf16 with a residual (604 MB) takes 99 us at its least
// (median 103, 5.9 TB/s) with eight wavefronts of one chunk, 101 with four of two, 104 with two of
// four; without packing (537 MB) 90 and 94.  4096 x 14336 (C = 2, 528 MB): 94 us.  Rows much
// shorter than 512 features leave lanes idle: at 128 features 16 of 64 work, and 262144 x 128 without
// a residual (171 MB) takes 82-99 us, where its bytes alone would take 26.  A call of a few
// megabytes is 3 us and its bytes: 5001 x 1000 fp16 with a residual (45 MB) 11.7 us.
template <typename T, bool Four, int C, bool S>
__global__ __launch_bounds__(Four ? 256 : 1024) void norm_kernel(NormArgs a) {
  const int kTeam = Four ? 64 : blockDim.x;
  __shared__ float part[Four ? 1 : 16];
  typedef typename T::elem_t elem_t;
  const int lane = Four ? (threadIdx.x & 63) : threadIdx.x;
  const uint32_t row = Four ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (row >= a.rows) return;  // whole teams
  const elem_t* x = static_cast<const elem_t*>(a.x) + (int64_t)row * a.x_stride;
  float h[C][8];
  {
    typename T::raw_t rx[C], rr[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * kTeam + lane) * 8;
      rx[c] = load_row<T, S>(x + col, a.features - col);
    }
    if (a.residual) {
      const elem_t* r = static_cast<const elem_t*>(a.residual) + (int64_t)row * a.residual_stride;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int col = (c * kTeam + lane) * 8;
        rr[c] = load_row<T, S>(r + col, a.features - col);
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int col = (c * kTeam + lane) * 8;
        float s[8];
        T::widen(rx[c], h[c]);
        T::widen(rr[c], s);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[c][i] += s[i];
        // what is normed is the sum as it is stored: the layer's other readers see that one
        T::widen(T::narrow(h[c]), h[c]);
        if (col < a.features)
          store_row<T, S>(static_cast<elem_t*>(a.h) + (int64_t)row * a.features + col, h[c],
                       a.features - col);
      }
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) T::widen(rx[c], h[c]);
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(h[c][i], h[c][i], ss);
  ss = Four ? sum_of_wave(ss) : sum_of_workgroup(ss, part);
  const float rstd = 1.0f / sqrtf(ss / (float)a.features + a.eps);
  if (a.rstd && lane == 0) a.rstd[row] = rstd;
  const int blocks = (a.features + kBlock - 1) / kBlock;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * kTeam + lane) * 8;
    if (col - (lane & 15) * 8 >= a.features) return;  // whole blocks
    const int n = a.features - col;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[c][i] *= rstd;
    if (a.weight) {
      load_weight<T>(a.weight, a.weight_is_f32, col, n, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= h[c][i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = h[c][i];
    }
    if (n > 0) store_row<T, S>(static_cast<elem_t*>(a.y) + (int64_t)row * a.features + col, y, n);
    if (a.values) {
      if (n < 8) {  // 0 times an infinite rstd is no zero
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i >= n) h[c][i] = 0.0f;
      }
      int e;
      const u32x2 q = quantise(h[c], &e);
      if (col < a.pitch)
        store_8<S>(a.values + (int64_t)row * a.pitch + col, q);
      if ((lane & 15) == 0) a.exponents[(int64_t)row * blocks + col / kBlock] = (uint8_t)e;
    }
  }
}

struct NormBackArgs {
  const void* grad_y;
  const void* grad_h;  // or NULL
  const uint8_t* values;
  const uint8_t* exponents;
  const float* rstd;
  const void* weight;  // or NULL
  void* grad_x;
  float* partial;      // [gridDim.x][features], or NULL: no weight gradient
  uint32_t rows;
  int features;
  int64_t grad_y_stride, grad_h_stride, pitch;
  int weight_is_f32;
};

// Teams as in norm_kernel.  A workgroup takes rows blockIdx.x, + gridDim.x, ... and keeps the
// weight gradient of its rows in registers; column_reduce_kernel adds the workgroups' partial
// sums in a fixed order.  A row is asked for while the one before it is worked on: few rows are
// in flight, because every workgroup leaves a partial sum of a whole row behind.  8192 x 4096 bf16
// with grad_h (235 MB) takes 39-43 us, 6.0-5.5 TB/s, and 4.7 for the partial sums; without asking ahead
// 69.  4096 x 14336 (C = 2: without asking ahead, 411 MB) takes 94 and 6.7, 262144 x 128 (171 MB; idle
// lanes as in norm_kernel, and 2048 wavefronts on the whole chip) 114 and 4.8.
template <typename T, bool Four, int C>
__global__ __launch_bounds__(Four ? 256 : 1024) void norm_back_kernel(NormBackArgs a) {
  constexpr int kRows = Four ? 4 : 1;
  constexpr bool kAhead = C == 1;  // two rows of two chunks do not fit 16 wavefronts' registers
  const int kTeam = Four ? 64 : blockDim.x;
  __shared__ float part[2][16];
  __shared__ float gathered[Four ? 3 : 1][Four ? 64 * C * 8 : 1];
  typedef typename T::elem_t elem_t;
  const int lane = Four ? (threadIdx.x & 63) : threadIdx.x;
  const int team = Four ? (threadIdx.x >> 6) : 0;
  const int blocks = (a.features + kBlock - 1) / kBlock;
  const float inv_n = 1.0f / (float)a.features;
  float gw[C][8], w[C][8];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * kTeam + lane) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) gw[c][i] = 0.0f, w[c][i] = 1.0f;
    if (a.weight && col < a.features) load_weight<T>(a.weight, a.weight_is_f32, col, a.features - col, w[c]);
  }
  struct Row {
    typename T::raw_t gy[C], gh[C];
    u32x2 q[C];
    uint32_t e[C];
    float rstd;
  };
  auto ask = [&](Row& r, uint32_t row) {
    const elem_t* gy = static_cast<const elem_t*>(a.grad_y) + (int64_t)row * a.grad_y_stride;
    const elem_t* gh = static_cast<const elem_t*>(a.grad_h) + (int64_t)row * a.grad_h_stride;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * kTeam + lane) * 8;
      r.gy[c] = load_row<T>(gy + col, a.features - col);
      r.q[c] = u32x2{0, 0};
      r.e[c] = 0;
      if (col < a.features) {
        r.q[c] = *reinterpret_cast<const u32x2*>(a.values + (int64_t)row * a.pitch + col);
        r.e[c] = a.exponents[(int64_t)row * blocks + col / kBlock];
      }
      if (a.grad_h) r.gh[c] = load_row<T>(gh + col, a.features - col);
    }
    r.rstd = a.rstd[row];
  };
  int turn = 0;
  const uint32_t step = gridDim.x * kRows;
  uint32_t row = blockIdx.x * kRows + team;
  Row next;
  if (kAhead && row < a.rows) ask(next, row);
  for (; row < a.rows; turn ^= 1) {
    if (!kAhead) ask(next, row);
    const Row r = next;
    const uint32_t here = row;
    row = a.rows - row > step ? row + step : a.rows;
    if (kAhead && row < a.rows) ask(next, row);
    float n[C][8], g[C][8];
    float dot = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * kTeam + lane) * 8;
      dequantise(r.q[c], scale_of(r.e[c]), n[c]);
      if (a.features - col < 8) {  // what a caller's padding holds does not count
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i >= a.features - col) n[c][i] = 0.0f;
      }
      T::widen(r.gy[c], g[c]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        gw[c][i] = fmaf(g[c][i], n[c][i], gw[c][i]);
        g[c][i] *= w[c][i];
        dot = fmaf(g[c][i], n[c][i], dot);
      }
    }
    dot = (Four ? sum_of_wave(dot) : sum_of_workgroup(dot, part[turn])) * inv_n;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * kTeam + lane) * 8;
      if (col >= a.features) break;
      float gx[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) gx[i] = r.rstd * fmaf(-n[c][i], dot, g[c][i]);
      if (a.grad_h) {
        float gh[8];
        T::widen(r.gh[c], gh);
#pragma unroll
        for (int i = 0; i < 8; ++i) gx[i] += gh[i];
      }
      store_row<T>(static_cast<elem_t*>(a.grad_x) + (int64_t)here * a.features + col, gx,
                      a.features - col);
    }
  }
  if (!a.partial) return;
  if constexpr (Four) {  // the four wavefronts' sums, in their order
    if (team) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) gathered[team - 1][(c * 8 + i) * 64 + lane] = gw[c][i];
    }
    __syncthreads();
    if (team) return;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int t = 0; t < 3; ++t) gw[c][i] += gathered[t][(c * 8 + i) * 64 + lane];
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * kTeam + lane) * 8;
    if (col >= a.features) break;
    store_row<F32>(a.partial + (int64_t)blockIdx.x * a.features + col, gw[c], a.features - col);
  }
}

// out[c] = sum over g of partial[g][c], g in fixed order: 32 columns and 32 row lanes per
// workgroup, the row lanes joined through LDS.  `pitch` floats from one g to the next.
template <typename T>
__global__ __launch_bounds__(1024) void column_reduce_kernel(const float* partial, void* out, uint32_t groups,
                                                             int64_t columns, int64_t pitch) {
  __shared__ float part[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.x * 32 + x;
  float s = 0.0f;
  if (col < columns)
#pragma unroll 8
    for (uint32_t g = y; g < groups; g += 32) s += partial[(int64_t)g * pitch + col];
  part[y][x] = s;
  __syncthreads();
  if (y || col >= columns) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) s += part[i][x];
  static_cast<typename T::elem_t*>(out)[col] = T::narrow1(s);
}

// Partial column sums of a [rows, columns] matrix: 256 lanes of eight columns, rows
// blockIdx.y, + gridDim.y, ..., four of them in flight.  Bound by memory, with few loads in flight as
// for the norm's gradients: 8192 x 14336 bf16 (235 MB) takes 49 us, 4.8 TB/s, and 4.8 for the partial
// sums; 8192 x 4096 13.3 and 4.0.
template <typename T>
__global__ __launch_bounds__(256) void column_sum_kernel(const void* x, float* partial, uint32_t rows,
                                                         int64_t columns, int64_t stride) {
  const int64_t col = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (col >= columns) return;
  const int n = (int)min(columns - col, (int64_t)8);
  const typename T::elem_t* p = static_cast<const typename T::elem_t*>(x) + col;
  float s[8] = {};
  for (uint64_t r = blockIdx.y; r < rows; r += 4ull * gridDim.y) {
    typename T::raw_t raw[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t at = r + (uint64_t)k * gridDim.y;
      raw[k] = load_row<T>(p + (int64_t)min(at, (uint64_t)rows - 1) * stride, at < rows ? n : 0);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float v[8];
      T::widen(raw[k], v);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += v[i];
    }
  }
  store_row<F32>(partial + (int64_t)blockIdx.y * columns + col, s, n);
}

// ---------------------------------------------------------------------------
// Weight gradient of a linear layer:  G[o][f] = w[f] * sum_t D[t][o] X[t][f]
// ---------------------------------------------------------------------------
// The products run on the bf16 matrix cores.  X is exact in bf16, and D is split into bf16 parts
// that add up to it exactly while it goes into LDS: one part for bf16, two for fp16 (11 bits),
// three for fp32 (24 bits; the matrix cores take bf16's subnormal numbers, so that only bits under
// 2^-133 are lost).  Every part is multiplied with the same X.
template <typename T>
struct Parts;
template <>
struct Parts<BF16> {
  static constexpr int kParts = 1, kTokens = 64;  // tokens of one step: with all parts of D and X
};                                                // twice, a step's tiles fill the LDS
template <>
struct Parts<F16> {
  static constexpr int kParts = 2, kTokens = 32;
};
template <>
struct Parts<F32> {
  static constexpr int kParts = 3, kTokens = 32;
};

// Eight elements -> their parts, eight bf16 each
template <typename T>
__device__ inline void split(const typename T::raw_t& raw, u32x4 (&part)[Parts<T>::kParts]) {
  if constexpr (Parts<T>::kParts == 1) {
    part[0] = raw.w[0];
  } else {
    float v[8];
    T::widen(raw, v);
#pragma unroll
    for (int p = 0; p < Parts<T>::kParts; ++p) {
      uint32_t b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // cut, not rounded: what is left over is exact, and nothing is rounded to infinity
        b[i] = __float_as_uint(v[i]);
        const float cut = __uint_as_float(b[i] & 0xffff0000u);
        v[i] = (b[i] & 0x7fffffffu) == kInfBits ? 0.0f : v[i] - cut;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) part[p][i] = (b[2 * i] >> 16) | (b[2 * i + 1] & 0xffff0000u);
    }
  }
}

// D with rows that start at multiples of 16 bytes and are whole chunks of eight, where the
// caller's are not
struct AlignArgs {
  const void* d;
  void* aligned;  // [rows][padded]
  int64_t columns, stride, padded;
  uint64_t chunks;  // rows * padded / 8
};

template <typename T>
__global__ __launch_bounds__(256) void align_kernel(AlignArgs a) {
  typedef typename T::elem_t elem_t;
  const uint64_t per_row = (uint64_t)a.padded / 8;
  for (uint64_t c = blockIdx.x * 256ull + threadIdx.x; c < a.chunks; c += gridDim.x * 256ull) {
    const uint64_t row = c / per_row;
    const int64_t col = (int64_t)(c - row * per_row) * 8;
    T::template store<false>(
        static_cast<elem_t*>(a.aligned) + c * 8,
        load_row<T>(static_cast<const elem_t*>(a.d) + (int64_t)row * a.stride + col,
                    (int)min(a.columns - col, (int64_t)8)));
  }
}

struct WgradArgs {
  const void* d;  // [rows][d_stride]
  const uint8_t* values;
  const uint8_t* exponents;
  const void* column_scale;  // or NULL
  void* out;                 // [out_features][features]
  float* partial;            // [splits][cut tiles][tile], or NULL
  int64_t rows, d_stride, pitch;
  uint32_t out_features, features, blocks;
  uint32_t tiles_o, tiles_f;
  uint32_t whole, cut, splits;  // tiles of one workgroup each, tiles of `splits` workgroups each
  uint32_t steps;
  int scale_type, out_type;  // TFT_F32 ...
  int partial_past_caches;
};

// Workgroup ids go round the 8 XCDs in turn; this gives each of them a run of neighbouring
// numbers out of n, so that what its workgroups share stays in its own L2.
__device__ inline uint32_t neighbours_on_an_xcd(uint32_t id, uint32_t n) {
  const uint32_t xcd = id % 8, each = n / 8, more = n % 8;
  return xcd * each + min(xcd, more) + id / 8;
}

// Tiles are numbered down bands of four rows of tiles: 32 in a row, one XCD's worth, are 4 x 8.
__device__ inline void tile_at(const WgradArgs& a, uint32_t n, uint32_t* o, uint32_t* f) {
  const uint32_t band = n / (4 * a.tiles_f), in_band = n - band * 4 * a.tiles_f;
  const uint32_t high = min(4u, a.tiles_o - band * 4);
  *o = band * 4 + in_band % high;
  *f = in_band / high;
}

__device__ inline __amdgpu_buffer_rsrc_t buffer(const void* base, int64_t bytes) {
  // reads behind the end give zero
  const int n = (int)max((int64_t)0, min(bytes, (int64_t)0x7fffffff));
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, n, 0x00020000);
}

__device__ inline float load_scale(const void* p, int type, int64_t at) {
  if (type == TFT_F32) return static_cast<const float*>(p)[at];
  if (type == TFT_BF16) return BF16::widen1(static_cast<const uint16_t*>(p)[at]);
  return F16::widen1(static_cast<const uint16_t*>(p)[at]);
}

// Up to four neighbouring features f .. of an output row, scaled and rounded: the slow form, for
// rows that are no whole number of fours
__device__ inline void store_out(const WgradArgs& a, int64_t o, int64_t f, const f32x4& v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (f + i >= a.features) return;
    const float x = a.column_scale ? v[i] * load_scale(a.column_scale, a.scale_type, f + i) : v[i];
    const int64_t at = o * a.features + f + i;
    if (a.out_type == TFT_F32) static_cast<float*>(a.out)[at] = x;
    else static_cast<uint16_t*>(a.out)[at] = a.out_type == TFT_BF16 ? BF16::narrow1(x) : F16::narrow1(x);
  }
}

template <typename T>
__device__ inline void store_four(typename T::elem_t* p, const f32x4& v) {
  if constexpr (sizeof(typename T::elem_t) == 4) {
    *reinterpret_cast<f32x4*>(p) = v;
  } else {
    uint16_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = T::narrow1(v[i]);
    *reinterpret_cast<u32x2*>(p) = u32x2{b[0] | ((uint32_t)b[1] << 16), b[2] | ((uint32_t)b[3] << 16)};
  }
}

// Tile of O output rows x F features, wavefronts in a WO x WF grid.
//
// Both operands lie with the summed axis (tokens) outermost, so LDS holds a step's tiles as they
// lie in memory, [token][column], and the transposing LDS reads (ds_read_b64_tr_b16: 16 lanes
// fetch 4 tokens x 16 columns, lane i gets column i's four tokens) turn them into matrix
// operands: lanes 0 .. 31 hold a product's first eight tokens of 32 columns, lanes 32 .. 63 the
// other eight.  Rows of a tile are units of 16 columns (32 bytes); unit u of token t lies at
// u ^ spread(t), so that the four rows of a transposing read, and the two units that lanes 0 .. 31
// read together, lie on different banks (248 of LDS's 256 bytes a cycle; 64 with every unit u at u).
//
// What bounds it.  A step of a large tile is 2048 cycles of matrix instructions on every SIMD.
// Next to them LDS gives out 192 KiB and takes in 64 (about 770 and 830 cycles), and the vector
// memory path brings 48 KiB (about 770), all from the same two wavefronts per SIMD.  8192 tokens,
// 14336 x 4096 bf16 take 775 to 830 us from box to box (1160 to 1240 TFLOP/s): the matrix
// units are busy about 55 % of the time at the 2.0 GHz that the power limit leaves (zeros in place
// of the data: 2.4 GHz, 630 us).  On the same box torch's product of these operands as they lie,
// already unpacked, takes 997 us, and with both operands turned beforehand 650 to 710.
// Tried and no faster: two groups of wavefronts that take turns at the matrix units (807 to
// 860 us), four wavefronts of 128 x 128 with every instruction's place laid down by hand (875),
// D through registers (850), half the loads of exponents (822).
__device__ inline int spread(int t) { return (t & 3) | ((t & 1) << 2); }

template <typename T, int O, int F, int WO, int WF>
__global__ __launch_bounds__(64 * WO * WF, 1) void wgrad_kernel(WgradArgs a) {
  typedef typename T::elem_t elem_t;
  constexpr int kThreads = 64 * WO * WF, kParts = Parts<T>::kParts, kTokens = Parts<T>::kTokens;
  constexpr int kDChunks = kTokens * O / 8 / kThreads;   // chunks of eight elements of D per thread and step
  constexpr int kXChunks = kTokens * F / 16 / kThreads;  // 16-byte chunks of X
  constexpr int kDTile = kParts * kTokens * O, kXTile = kTokens * F;
  constexpr int kFragO = O / WO / 32, kFragF = F / WF / 32;
  // bf16 goes from memory into LDS by itself, past the registers (kDirect), into one of three buffers
  // because a tile is asked for while two are in use; what has to be split goes through registers
  constexpr bool kDirect = kParts == 1;
  constexpr int kDBuffers = kDirect ? 3 : 2;
  __shared__ __attribute__((aligned(128))) uint16_t lds[kDBuffers * kDTile + 2 * kXTile];
  uint16_t* const lds_d = lds;                       // tiles [part][token][O]
  uint16_t* const lds_x = lds + kDBuffers * kDTile;  // two tiles [token][F]

  const bool is_cut = blockIdx.x >= a.whole;
  uint32_t tile_o, tile_f, slot = 0, step_begin = 0, step_end = a.steps;
  if (is_cut) {
    slot = neighbours_on_an_xcd(blockIdx.x - a.whole, a.cut * a.splits);  // split-major
    const uint32_t split = slot / a.cut;
    const uint32_t each = a.steps / a.splits, more = a.steps - each * a.splits;
    step_begin = split * each + min(split, more);
    step_end = step_begin + each + (split < more ? 1 : 0);
    tile_at(a, a.whole + slot - split * a.cut, &tile_o, &tile_f);
  } else {
    tile_at(a, neighbours_on_an_xcd(blockIdx.x, a.whole), &tile_o, &tile_f);
  }
  const int64_t o0 = (int64_t)tile_o * O, f0 = (int64_t)tile_f * F;

  // what this thread stages, the same in every step but for the token offset
  uint32_t d_off[kDChunks], d_lds[kDChunks], x_off[kXChunks], x_lds[kXChunks], e_off[kXChunks];
#pragma unroll
  for (int i = 0; i < kDChunks; ++i) {
    const int c = i * kThreads + threadIdx.x, t = c / (O / 8), j = c % (O / 8);
    const int spread_j = (((j >> 1) ^ spread(t)) << 1) + (j & 1);
    // direct loads lie in LDS in the order of the lanes, so a lane asks for the chunk whose place is its own
    const int from = kDirect ? spread_j : j;
    d_off[i] = o0 + from * 8 < a.out_features ? (uint32_t)((t * a.d_stride + from * 8) * sizeof(elem_t)) : 0x80000000u;
    d_lds[i] = t * O + spread_j * 8;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int swap = (lane >> 2) & 1;  // lanes 4 .. 7 of eight write a unit's halves the other way round
#pragma unroll
  for (int i = 0; i < kXChunks; ++i) {
    const int c = i * kThreads + threadIdx.x, t = c / (F / 16), u = c % (F / 16);
    x_off[i] = f0 + u * 16 < a.pitch ? (uint32_t)(t * a.pitch + u * 16) : 0x80000000u;
    e_off[i] = f0 + u * 16 < a.pitch ? (uint32_t)(t * a.blocks + (u * 16) / kBlock) : 0x80000000u;
    x_lds[i] = t * F + ((u ^ spread(t)) << 4) + swap * 8;
  }
  // what this lane reads: token 8 (lane / 32) + i / 4 of a product's 16 (+ 4), columns 4 (i % 4) ..
  // of unit 2f + (lane / 16) % 2, for lane i of 16
  const int t_lane = ((lane >> 5) << 3) + ((lane & 15) >> 2);
  const int wave_o = (wave / WF) * (O / WO), wave_f = (wave % WF) * (F / WF);
  uint32_t d_read[kFragO], x_read[kFragF];
#pragma unroll
  for (int f = 0; f < kFragO; ++f)
    d_read[f] = t_lane * O + (((wave_o / 16 + 2 * f + ((lane >> 4) & 1)) ^ spread(t_lane)) << 4) + ((lane & 3) << 2);
#pragma unroll
  for (int f = 0; f < kFragF; ++f)
    x_read[f] = t_lane * F + (((wave_f / 16 + 2 * f + ((lane >> 4) & 1)) ^ spread(t_lane)) << 4) + ((lane & 3) << 2);

  // the tile of the next step to ask for: d, x and e point at its first token and column
  const int64_t t0 = (int64_t)step_begin * kTokens;
  const elem_t* d_at = static_cast<const elem_t*>(a.d) + t0 * a.d_stride + o0;
  const uint8_t* x_at = a.values + t0 * a.pitch + f0;
  const uint8_t* e_at = a.exponents + t0 * a.blocks + f0 / kBlock;
  int64_t left = min(a.rows, (int64_t)step_end * kTokens) - t0;  // tokens from there on; may pass below 0
  typename T::raw_t d_reg[kDChunks];
  u32x4 x_reg[kXChunks];
  uint32_t e_reg[kXChunks];
  // D and X are asked for at different times, each as soon as its registers are free
  auto fetch_d_into = [&](typename T::raw_t (&d_reg)[kDChunks]) {
    const auto d = buffer(d_at, (left * a.d_stride - o0) * (int64_t)sizeof(elem_t));
#pragma unroll
    for (int i = 0; i < kDChunks; ++i)
#pragma unroll
      for (int w = 0; w < (int)sizeof(elem_t) / 2; ++w)
        d_reg[i].w[w] = __builtin_amdgcn_raw_buffer_load_b128(d, d_off[i] + 16 * w, 0, 0);
  };
  auto fetch_x_into = [&](u32x4 (&x_reg)[kXChunks], uint32_t (&e_reg)[kXChunks]) {
    const auto x = buffer(x_at, left * a.pitch - f0);
    const auto e = buffer(e_at, left * a.blocks - f0 / kBlock);
#pragma unroll
    for (int i = 0; i < kXChunks; ++i) {
      x_reg[i] = __builtin_amdgcn_raw_buffer_load_b128(x, x_off[i], 0, 0);
      e_reg[i] = __builtin_amdgcn_raw_buffer_load_b8(e, e_off[i], 0, 0);
    }
  };
  // D past the registers, into buffer `to`.  The compiler does not know of these loads: who reads
  // the buffer has waited for them by hand.  (With the compiler's own form of this load every
  // barrier waits for all of them.)  Nothing else here uses M0, which gfx950's LDS accesses ignore.
  auto fetch_d_direct = [&](int to) {
    const uint64_t base = (uint64_t)d_at;
    const int64_t bytes = (left * a.d_stride - o0) * (int64_t)sizeof(elem_t);
    const u32x4 d = {(uint32_t)base, (uint32_t)(base >> 32) & 0xffffu,
                     (uint32_t)max((int64_t)0, min(bytes, (int64_t)0x7fffffff)), 0x00020000u};
    const uint32_t at =
        (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint16_t*)(lds_d + to * kDTile + wave * 512);
#pragma unroll
    for (int i = 0; i < kDChunks; ++i)  // 64 lanes of 16 bytes, one behind the other, from M0 on
      asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                   :
                   : "v"(d_off[i]), "s"(d), "s"(at + i * kThreads * 16)
                   : "memory");
  };
  auto advance = [&]() {
    left -= kTokens;
    d_at += kTokens * a.d_stride;
    x_at += kTokens * a.pitch;
    e_at += (int64_t)kTokens * a.blocks;
  };
  auto fetch_d = [&]() { fetch_d_into(d_reg); };
  auto fetch_x = [&]() { fetch_x_into(x_reg, e_reg); };
  auto stage_d = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kDChunks; ++i) {
      u32x4 part[kParts];
      split<T>(d_reg[i], part);
#pragma unroll
      for (int p = 0; p < kParts; ++p)
        *reinterpret_cast<u32x4*>(&lds_d[buf * kDTile + p * kTokens * O + d_lds[i]]) = part[p];
    }
  };
  auto stage_x = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kXChunks; ++i) {
      const float scale = scale_of(e_reg[i]);
      u32x4 half[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t from = (h ^ swap) ? x_reg[i][2 + w] : x_reg[i][w];
          half[h][2 * w] = __builtin_bit_cast(
              uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(from, scale, false));
          half[h][2 * w + 1] = __builtin_bit_cast(
              uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(from, scale, true));
        }
      *reinterpret_cast<u32x4*>(&lds_x[buf * kXTile + x_lds[i]]) = half[0];
      *reinterpret_cast<u32x4*>(&lds_x[buf * kXTile + (x_lds[i] ^ 8)]) = half[1];
    }
  };

  f32x16 acc[kFragF][kFragO];
#pragma unroll
  for (int i = 0; i < kFragF; ++i)
#pragma unroll
    for (int j = 0; j < kFragO; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  typedef __attribute__((address_space(3))) s16x4* lds_ptr;
  auto read_tr = [&](const uint16_t* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(const_cast<uint16_t*>(p)));
  };
  auto operand = [&](const uint16_t* base, int columns) {  // 16 tokens of two units
    const s16x4 lo = read_tr(base), hi = read_tr(base + 4 * columns);
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  // A step's products: kTokens / 16 groups of tokens, every part of D with the same X
  constexpr int kProducts = kTokens / 16 * kParts;
  bf16x8 d[2][kFragO], x[2][kFragF];
  auto load = [&](int product, int d_buf, int x_buf) {
    const int group = product / kParts, part = product % kParts;
    if (part == 0)
#pragma unroll
      for (int i = 0; i < kFragF; ++i)
        x[group & 1][i] = operand(&lds_x[x_buf * kXTile + x_read[i] + group * 16 * F], F);
#pragma unroll
    for (int j = 0; j < kFragO; ++j)
      d[product & 1][j] = operand(&lds_d[d_buf * kDTile + d_read[j] + (part * kTokens + group * 16) * O], O);
  };
  auto multiply = [&](int product) {
#pragma unroll
    for (int i = 0; i < kFragF; ++i)
#pragma unroll
      for (int j = 0; j < kFragO; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[product / kParts & 1][i], d[product & 1][j],
                                                            acc[i][j], 0, 0, 0);
  };

  // While one product runs, the next one's operands come out of LDS; meanwhile the next step's
  // tile goes into another buffer, and the tile after that is asked for.  One barrier a step:
  // behind it the next tile is whole, and nobody reads the present one any more.
  static_assert(kProducts % 2 == 0 && kTokens / 16 % 2 == 0, "the operands' turns close with a step");
  if (step_begin < step_end) {
    int d_now = 0, d_next = 1, d_after = kDirect ? 2 : 0, x_now = 0;
    // the first two tiles are asked for together: one memory latency before the first product
    typename T::raw_t d_second[kDChunks];
    u32x4 x_second[kXChunks];
    uint32_t e_second[kXChunks];
    if constexpr (kDirect) fetch_d_direct(0);
    else fetch_d();
    fetch_x();
    advance();
    if constexpr (kDirect) fetch_d_direct(1);
    else fetch_d_into(d_second);
    fetch_x_into(x_second, e_second);
    advance();
    if constexpr (!kDirect) stage_d(0);
    stage_x(0);
    if constexpr (kDirect) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < kDChunks; ++i)
      if (!kDirect) d_reg[i] = d_second[i];
#pragma unroll
    for (int i = 0; i < kXChunks; ++i) x_reg[i] = x_second[i], e_reg[i] = e_second[i];
    __syncthreads();
    load(0, 0, 0);
    for (uint32_t s = step_begin; s < step_end; ++s) {
#pragma unroll
      for (int k = 0; k + 1 < kProducts; ++k) {
        load(k + 1, d_now, x_now);
        if (kDirect && k == 1) {
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the next step's D and X, asked for a step ago
          fetch_d_direct(d_after);
          stage_x(x_now ^ 1);
          fetch_x();
          advance();
        }
        if (!kDirect && k == 1) {
          stage_d(d_next);
          fetch_d();
        }
        if (!kDirect && k == 2) {
          stage_x(x_now ^ 1);
          fetch_x();
          advance();
        }
        multiply(k);
      }
      // waits for this wavefront's LDS accesses, not for the loads under way
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      load(0, d_next, x_now ^ 1);
      multiply(kProducts - 1);
      x_now ^= 1;
      const int before = d_now;
      d_now = d_next;
      d_next = d_after;
      d_after = before;
      if (!kDirect) d_next = before, d_after = d_now;
    }
    if constexpr (kDirect) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing lands in LDS any more
  }

  // Of 32 features x 32 output rows a lane holds output row lane % 32, features 8q + 4 (lane / 32)
  // .. + 3 for q = 0 .. 3.  Every wavefront turns its 32 rows around in LDS of its own, so that it
  // stores whole rows; four floats of padding keep the rows on different banks.
  constexpr int kWide = F / WF, kPitch = kWide + 4;
  static_assert(WO * WF * 32 * kPitch * 4 <= (int)sizeof(lds), "the turned rows fit the tiles");
  __syncthreads();
  float* const turn = reinterpret_cast<float*>(lds) + wave * 32 * kPitch;
  constexpr int kLanes = kWide / 4;  // lanes per row
  const int64_t f = f0 + wave_f + (lane % kLanes) * 4;
  const int64_t o_lane = wave_o + lane / kLanes;  // this lane's first row; the next one is 64 / kLanes on
  constexpr int kRows = kLanes / 2;               // of 32 that it stores
  auto fence = [&]() {  // between lanes of the wavefront, through LDS
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  // store(row of the tile, four features); all rows of a turn are read before the first is stored
  auto store_all = [&](auto store) {
#pragma unroll
    for (int j = 0; j < kFragO; ++j) {
#pragma unroll
      for (int i = 0; i < kFragF; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4*>(&turn[(lane & 31) * kPitch + i * 32 + q * 8 + (lane >> 5) * 4]) =
              f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
      fence();
      f32x4 v[kRows];
#pragma unroll
      for (int k = 0; k < kRows; ++k)
        v[k] = *reinterpret_cast<const f32x4*>(&turn[(k * (64 / kLanes) + lane / kLanes) * kPitch + (lane % kLanes) * 4]);
      fence();
#pragma unroll
      for (int k = 0; k < kRows; ++k) store(o_lane + j * 32 + k * (64 / kLanes), v[k]);
    }
  };
  auto store_as = [&](auto type, const f32x4& scale) {
    typedef decltype(type) Out;
    typename Out::elem_t* const to = static_cast<typename Out::elem_t*>(a.out) + o0 * a.features + f;
    const int64_t rows = f < a.features ? (int64_t)a.out_features - o0 : 0;
    store_all([&](int64_t row, const f32x4& v) {
      if (row < rows) store_four<Out>(to + row * a.features, v * scale);
    });
  };
  if (is_cut) {
    float* const to = a.partial + (int64_t)slot * O * F + wave_f + (lane % kLanes) * 4;
    if (a.partial_past_caches)
      store_all([&](int64_t row, const f32x4& v) {
        __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(to + row * F));
      });
    else
      store_all([&](int64_t row, const f32x4& v) { *reinterpret_cast<f32x4*>(to + row * F) = v; });
  } else if (a.features % 4 == 0) {
    f32x4 scale = {1.0f, 1.0f, 1.0f, 1.0f};
    if (a.column_scale) {
      const int64_t at = min(f, (int64_t)a.features - 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) scale[i] = load_scale(a.column_scale, a.scale_type, at + i);
    }
    if (a.out_type == TFT_BF16) store_as(BF16(), scale);
    else if (a.out_type == TFT_F16) store_as(F16(), scale);
    else store_as(F32(), scale);
  } else {
#pragma unroll
    for (int j = 0; j < kFragO; ++j) {
#pragma unroll
      for (int i = 0; i < kFragF; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4*>(&turn[(lane & 31) * kPitch + i * 32 + q * 8 + (lane >> 5) * 4]) =
              f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
      fence();
#pragma unroll 1
      for (int k = 0; k < kRows; ++k) {
        const int r = k * (64 / kLanes) + lane / kLanes;
        const int64_t o = o0 + wave_o + j * 32 + r;
        if (o < a.out_features)
          store_out(a, o, f, *reinterpret_cast<const f32x4*>(&turn[r * kPitch + (lane % kLanes) * 4]));
      }
      fence();
    }
  }
}

// Joins the partial products of the cut tiles, in the order of the sum.  Bound by memory: 128 large
// tiles in two pieces (67 MB in, 17 out) take 18 us.
template <int O, int F>
__global__ __launch_bounds__(256) void wgrad_join_kernel(WgradArgs a) {
  constexpr uint32_t kPerTile = O * F / 4;
  const uint32_t at = blockIdx.x * 256 + threadIdx.x, tile = at / kPerTile, in = at % kPerTile;
  uint32_t tile_o, tile_f;
  tile_at(a, a.whole + tile, &tile_o, &tile_f);
  const int64_t o = (int64_t)tile_o * O + in / (F / 4), f = (int64_t)tile_f * F + in % (F / 4) * 4;
  if (o >= a.out_features || f >= a.features) return;
  const float* p = a.partial + ((int64_t)tile * kPerTile + in) * 4;
  const int64_t next = (int64_t)a.cut * O * F;
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t s = 0; s < a.splits; s += 4) {  // four loads in flight
    f32x4 part[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      part[i] = s + i < a.splits ? *reinterpret_cast<const f32x4*>(p + (s + i) * next) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) v += part[i];
  }
  if (a.features % 4 != 0) {
    store_out(a, o, f, v);
    return;
  }
  if (a.column_scale)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= load_scale(a.column_scale, a.scale_type, f + i);
  const int64_t to = o * a.features + f;
  if (a.out_type == TFT_BF16) store_four<BF16>(static_cast<uint16_t*>(a.out) + to, v);
  else if (a.out_type == TFT_F16) store_four<F16>(static_cast<uint16_t*>(a.out) + to, v);
  else store_four<F32>(static_cast<float*>(a.out) + to, v);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// A call that moves more than the last-level cache holds reads and writes past the caches: packing
// 224 MiB of bf16 takes 54 us so and 62 through them, unpacking 56 and 60, the norm of two times
// 128 MiB 99 and 107.  Below, what a call leaves in the cache is worth more to the next one:
// unpacking 128 MiB and summing it takes 62 us past the caches and 57 through them.
constexpr int64_t kLastLevelCache = 256ll << 20;
constexpr int64_t kMostRows = 1ll << 31;
constexpr int kMostNormFeatures = 16384;

bool known_type(int t) { return t == TFT_F32 || t == TFT_BF16 || t == TFT_F16; }

int check_types(const char* what, int dtype, int weight_dtype, bool has_weight) {
  if (!known_type(dtype))
    return fail(TFT_ERR_UNSUPPORTED, "%s: dtype %d is not fp32, bf16 or fp16", what, dtype);
  if (has_weight && !known_type(weight_dtype))
    return fail(TFT_ERR_UNSUPPORTED, "%s: weight dtype %d is not fp32, bf16 or fp16", what, weight_dtype);
  return TFT_OK;
}

// Common checks of a packed matrix; `rows` and `features` at least 1 behind this.
int check_packed(const char* what, const void* values, const void* exponents, int64_t rows,
                 int64_t features, int64_t pitch) {
  if (rows >= kMostRows) return fail(TFT_ERR_UNSUPPORTED, "%s: %lld rows, at most 2^31 - 1", what, (long long)rows);
  if (features >= kMostRows)
    return fail(TFT_ERR_UNSUPPORTED, "%s: %lld features, at most 2^31 - 1", what, (long long)features);
  if (pitch < features || pitch % 16 || pitch >= features + kBlock)
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: pitch %lld does not fit %lld features (a multiple of 16, less than 128 more)",
                what, (long long)pitch, (long long)features);
  const int64_t blocks = (features + kBlock - 1) / kBlock;
  if (pitch > blocks * kBlock)
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: pitch %lld lies behind the last block of %lld features", what,
                (long long)pitch, (long long)features);
  if (rows * blocks >= (1ll << 31))
    return fail(TFT_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 blocks of 128 features", what);
  if (!values || !exponents) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: packed buffers are NULL", what);
  if (reinterpret_cast<uintptr_t>(values) & 15u)
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: packed values must start at a multiple of 16 bytes", what);
  return TFT_OK;
}

int esize(int dtype) { return dtype == TFT_F32 ? 4 : 2; }

bool misaligned(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(esize(dtype) - 1)) != 0; }

int launch(const char* what, const void* kernel, dim3 grid, int threads, void** params, hipStream_t s) {
  const hipError_t e = hipLaunchKernel(kernel, grid, dim3(threads), params, 0, s);
  if (e != hipSuccess) return fail(TFT_ERR_LAUNCH, "%s: launch failed: %s", what, hipGetErrorString(e));
  return TFT_OK;
}

// A dispatch counts its threads with 32 bits.  Calls of more rows than fit into one are launched in
// slices: rows are independent of each other, so a slice is the same call of fewer rows.
int64_t most_groups(int threads) { return 0xffffffffll / threads; }

// launch_slice(first row, rows) for slices of at most `most` rows
template <typename F>
int in_slices(int64_t rows, int64_t most, F launch_slice) {
  for (int64_t first = 0; first < rows; first += most)
    if (int rc = launch_slice(first, rows - first < most ? rows - first : most)) return rc;
  return TFT_OK;
}

const void* row_at(const void* p, int64_t row, int64_t stride, int dtype) {
  return p ? static_cast<const char*>(p) + row * stride * esize(dtype) : nullptr;
}

void* row_at(void* p, int64_t row, int64_t stride, int dtype) {
  return p ? static_cast<char*>(p) + row * stride * esize(dtype) : nullptr;
}

#define TFT_KERNEL(...) reinterpret_cast<const void*>(&__VA_ARGS__)

// Threads of a workgroup for rows of so many features, `chunks` of eight a lane
int norm_threads(int features, int chunks) { return (features + 512 * chunks - 1) / (512 * chunks) * 64; }

template <typename T, bool S>
int launch_norm(const char* what, const NormArgs& a, int dtype, hipStream_t s) {
  const bool four = a.features <= 512;  // rows to a workgroup
  const int chunks = a.features <= 8192 ? 1 : 2, threads = four ? 256 : norm_threads(a.features, chunks);
  const int64_t blocks = (a.features + kBlock - 1) / kBlock;
  return in_slices(a.rows, most_groups(threads) * (four ? 4 : 1), [&](int64_t first, int64_t rows) {
    NormArgs args = a;
    args.rows = (uint32_t)rows;
    args.x = row_at(a.x, first, a.x_stride, dtype);
    args.residual = row_at(a.residual, first, a.residual_stride, dtype);
    args.y = row_at(a.y, first, a.features, dtype);
    args.h = row_at(a.h, first, a.features, dtype);
    args.values = a.values ? a.values + first * a.pitch : nullptr;
    args.exponents = a.exponents ? a.exponents + first * blocks : nullptr;
    args.rstd = a.rstd ? a.rstd + first : nullptr;
    void* params[] = {&args};
    if (four) return launch(what, TFT_KERNEL(norm_kernel<T, true, 1, S>), dim3((args.rows + 3) / 4), threads, params, s);
    return launch(what, chunks == 1 ? TFT_KERNEL(norm_kernel<T, false, 1, S>) : TFT_KERNEL(norm_kernel<T, false, 2, S>),
                  dim3(args.rows), threads, params, s);
  });
}

// Two workgroups a CU: more of them hide more of a row's latency and leave more partial sums
// behind.  8192 x 4096 bf16: 512 take 43.7 us, 256 45.3, 768 50, 1024 48.
constexpr uint32_t kNormBackGroups = 512;

uint32_t norm_back_groups(int64_t rows, int64_t features) {
  const int64_t teams = features <= 512 ? (rows + 3) / 4 : rows;
  return (uint32_t)(teams < (int64_t)kNormBackGroups ? teams : (int64_t)kNormBackGroups);
}

template <typename T>
int launch_norm_back(const char* what, const NormBackArgs& a, hipStream_t s) {
  NormBackArgs args = a;
  void* params[] = {&args};
  const dim3 grid(norm_back_groups(a.rows, a.features));
  if (a.features <= 512) return launch(what, TFT_KERNEL(norm_back_kernel<T, true, 1>), grid, 256, params, s);
  if (a.features <= 8192)
    return launch(what, TFT_KERNEL(norm_back_kernel<T, false, 1>), grid, norm_threads(a.features, 1), params, s);
  return launch(what, TFT_KERNEL(norm_back_kernel<T, false, 2>), grid, norm_threads(a.features, 2), params, s);
}

int launch_column_reduce(const char* what, const float* partial, void* out, uint32_t groups,
                         int64_t columns, int dtype, hipStream_t s) {
  const void* k = dtype == TFT_F32 ? TFT_KERNEL(column_reduce_kernel<F32>)
                  : dtype == TFT_BF16 ? TFT_KERNEL(column_reduce_kernel<BF16>)
                                      : TFT_KERNEL(column_reduce_kernel<F16>);
  return in_slices(columns, most_groups(1024) * 32, [&](int64_t first, int64_t n) {  // of columns
    const float* from = groups ? partial + first : nullptr;
    void* to = row_at(out, first, 1, dtype);
    int64_t pitch = columns;
    void* params[] = {&from, &to, &groups, &n, &pitch};
    return launch(what, k, dim3((uint32_t)((n + 31) / 32)), 1024, params, s);
  });
}

uint32_t column_sum_groups(int64_t rows, int64_t columns) {
  const int64_t across = (columns + 2047) / 2048;
  int64_t g = (512 + across - 1) / across;
  if (g > (rows + 7) / 8) g = (rows + 7) / 8;
  return (uint32_t)(g < 1 ? 1 : g);
}

// Partial tiles that fit the XCDs' L2 together are written past it: the kernel's end would wait for
// their write-back (1000 tokens, 1001 x 768 fp32, 16 MB: 27.5 us so, 29.4 through L2; 1024, 768 x 768
// bf16, 9 MB: 15.5 and 16.6).  More of them are written back while the kernel runs, and the join
// finds the rest in the cache (8192, 1024 x 4096, 67 MB: 80.7 and 77.3).
constexpr int64_t kL2Bytes = 32ll << 20;

// How a weight gradient is cut.
struct WgradPlan {
  bool align_first;  // the gradient is copied to aligned rows of the workspace
  int64_t padded;    // their length
  bool large;
  uint32_t tiles_o, tiles_f, steps, whole, cut, splits;
  int64_t aligned_bytes, partial_bytes;
};

constexpr int64_t kLarge = 256, kSmall = 128;  // tiles; one large or two small ones fill a CU's LDS
constexpr int64_t kCUs = 256;

// Microseconds that the tiles of one size take with those left over from whole rounds of the chip
// cut into `splits` pieces along the tokens.  A step of 16 x kProducts tokens takes 0.8 us of a
// small tile alone on its CU, 1.15 of two beside each other and 1.8 of a large one; a round of
// workgroups starts and ends in 5; partial tiles are written and read at 7 TB/s and joined by a
// launch of 2.
double wgrad_time(bool large, int64_t tiles, int64_t steps, int products, int64_t splits) {
  const int64_t at_once = large ? kCUs : 2 * kCUs, size = large ? kLarge : kSmall, pieces = tiles % at_once * splits;
  const double step = products / 4.0;
  const double whole = (double)(tiles / at_once) * (3.0 + steps * step * (large ? 1.8 : 1.15));
  if (!pieces) return whole;
  const double each = step * (large ? 1.8 : pieces > kCUs ? 1.15 : 0.8);
  const int64_t rounds = (pieces + at_once - 1) / at_once, longest = (steps + splits - 1) / splits;
  return whole + rounds * (5.0 + longest * each) + (splits > 1 ? 2.0 + pieces * size * size * 8 / 7e6 : 0.0);
}

// Large tiles read LDS less per product and small ones fill the chip with less; which of them, and
// how many pieces, is the least of the times above.  Measured, us, large tiles in their best number
// of pieces / small ones in theirs: 8192 tokens, 4096 x 4096 bf16 219 (1) / 290 (1); 8192,
// 1024 x 4096 77 (4) / 85 (2); 4096, 2048 x 2048 fp16 78 (4) / 87 (2); 16384, 1000 x 1000 fp32 103 (16) /
// 117 (8); 4096, 1024 x 4096 bf16 51 (3) / 49 (1), where small ones in 2 are taken (51); 1024, 768 x 768
// bf16 18 (6) / 14.3 (3), where 4 are taken (15.1); 1000, 1001 x 768 fp32 31 (7) / 26 (4), where 5 are
// taken (27.7): the estimate is up to 6 % off the best.
WgradPlan plan_wgrad(int64_t rows, int64_t out_features, int64_t features, int64_t grad_stride,
                     int dtype, bool aligned) {
  WgradPlan p{};
  p.align_first = !aligned || out_features % 8 || grad_stride % 8 ||
                  grad_stride < out_features;  // a row that stands for several (an expanded gradient)
  p.padded = p.align_first ? (out_features + 7) / 8 * 8 : grad_stride;
  p.aligned_bytes = p.align_first ? (rows * p.padded * esize(dtype) + 255) / 256 * 256 : 0;
  const int tokens = dtype == TFT_F32 ? Parts<F32>::kTokens : dtype == TFT_F16 ? Parts<F16>::kTokens : Parts<BF16>::kTokens;
  const int parts = dtype == TFT_F32 ? Parts<F32>::kParts : dtype == TFT_F16 ? Parts<F16>::kParts : Parts<BF16>::kParts;
  p.steps = (uint32_t)((rows + tokens - 1) / tokens);
  double best = 0.0;
  for (int large = 1; large >= 0; --large) {
    const int64_t size = large ? kLarge : kSmall, at_once = large ? kCUs : 2 * kCUs;
    const int64_t across = (out_features + size - 1) / size, along = (features + size - 1) / size;
    const int64_t tiles = across * along, over = tiles % at_once;
    const int64_t most = over == 0 ? 1 : at_once / over < p.steps ? at_once / over : p.steps > 1 ? p.steps : 1;
    for (int64_t splits = 1; splits <= most; splits += 1 + splits / 8) {
      const double time = wgrad_time(large, tiles, p.steps, tokens / 16 * parts, splits);
      if (best != 0.0 && time >= best) continue;
      best = time;
      p.large = large;
      p.tiles_o = (uint32_t)across;
      p.tiles_f = (uint32_t)along;
      p.splits = (uint32_t)splits;
      p.cut = (uint32_t)(splits > 1 ? over : 0);
      p.whole = (uint32_t)(tiles - p.cut);
      p.partial_bytes = p.cut * splits * size * size * 4;
    }
  }
  return p;
}

template <typename T>
int launch_wgrad(const char* what, const WgradArgs& a, const WgradPlan& p, const AlignArgs& align, hipStream_t s) {
  if (p.align_first && a.rows > 0) {
    AlignArgs args = align;
    void* params[] = {&args};
    const uint64_t groups = (align.chunks + 255) / 256;
    if (int rc = launch(what, TFT_KERNEL(align_kernel<T>), dim3((uint32_t)(groups < 16384 ? groups : 16384)), 256,
                        params, s))
      return rc;
  }
  WgradArgs args = a;
  void* params[] = {&args};
  const dim3 grid(p.whole + p.cut * p.splits);
  if (int rc = p.large ? launch(what, TFT_KERNEL(wgrad_kernel<T, kLarge, kLarge, 2, 4>), grid, 512, params, s)
                       : launch(what, TFT_KERNEL(wgrad_kernel<T, kSmall, kSmall, 2, 2>), grid, 256, params, s))
    return rc;
  if (!p.cut) return TFT_OK;
  const int64_t size = p.large ? kLarge : kSmall;
  const dim3 join((uint32_t)(p.cut * (size * size / 1024)));
  return p.large ? launch(what, TFT_KERNEL(wgrad_join_kernel<kLarge, kLarge>), join, 256, params, s)
                 : launch(what, TFT_KERNEL(wgrad_join_kernel<kSmall, kSmall>), join, 256, params, s);
}

}  // namespace

extern "C" {

uint64_t tft_capture_id(void* stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &status, &id) != hipSuccess) {
    (void)hipGetLastError();  // not for the next caller who asks
    return ~0ull;
  }
  return status == hipStreamCaptureStatusNone ? 0 : status == hipStreamCaptureStatusActive ? id + 1 : ~0ull;
}

int tft_pack_e4m3(void* values, void* exponents, const void* x, int64_t rows, int64_t features,
                  int64_t x_row_stride, int64_t pitch, int dtype, void* stream) {
  static const char* what = "tft_pack_e4m3";
  if (int rc = check_types(what, dtype, 0, false)) return rc;
  if (rows < 0 || features < 0) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  if (rows == 0 || features == 0) return TFT_OK;
  if (int rc = check_packed(what, values, exponents, rows, features, pitch)) return rc;
  if (!x || misaligned(x, dtype)) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: x is NULL or misaligned", what);
  if (x_row_stride < 0) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: negative row stride", what);
  const uint32_t per_row = (uint32_t)((features + kBlock - 1) / kBlock);
  const bool far = rows * features * (esize(dtype) + 1) >= kLastLevelCache;
#define TFT_PACK(T) (far ? TFT_KERNEL(pack_kernel<T, true>) : TFT_KERNEL(pack_kernel<T, false>))
  const void* k = dtype == TFT_F32 ? TFT_PACK(F32) : dtype == TFT_BF16 ? TFT_PACK(BF16) : TFT_PACK(F16);
#undef TFT_PACK
  // a row has at most 2^24 blocks, far less than one launch
  return in_slices(rows, most_groups(kPackThreads) * kPackBlocks / per_row, [&](int64_t first, int64_t n) {
    PackArgs a{row_at(x, first, x_row_stride, dtype), static_cast<uint8_t*>(values) + first * pitch,
               static_cast<uint8_t*>(exponents) + first * per_row, features, x_row_stride, pitch,
               (uint32_t)(n * per_row), make_divider(per_row)};
    void* params[] = {&a};
    return launch(what, k, dim3((a.blocks + kPackBlocks - 1) / kPackBlocks), kPackThreads, params,
                  static_cast<hipStream_t>(stream));
  });
}

int tft_unpack_e4m3(void* out, const void* values, const void* exponents, const void* column_scale,
                    int64_t rows, int64_t features, int64_t pitch, int scale_dtype, int dtype,
                    void* stream) {
  static const char* what = "tft_unpack_e4m3";
  if (int rc = check_types(what, dtype, scale_dtype, column_scale != nullptr)) return rc;
  if (rows < 0 || features < 0) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  if (rows == 0 || features == 0) return TFT_OK;
  if (int rc = check_packed(what, values, exponents, rows, features, pitch)) return rc;
  if (!out || misaligned(out, dtype)) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: out is NULL or misaligned", what);
  if (column_scale && misaligned(column_scale, scale_dtype))
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: column_scale is misaligned", what);
  const uint32_t per_row = (uint32_t)((features + kBlock - 1) / kBlock);
  const int st = column_scale ? scale_dtype : TFT_F32;
  const bool far = rows * features * (esize(dtype) + 1) >= kLastLevelCache;
#define TFT_UNPACK2(T, W) (far ? TFT_KERNEL(unpack_kernel<T, W, true>) : TFT_KERNEL(unpack_kernel<T, W, false>))
#define TFT_UNPACK(T)                                   \
  (st == TFT_F32 ? TFT_UNPACK2(T, F32)                  \
   : st == TFT_BF16 ? TFT_UNPACK2(T, BF16)              \
                    : TFT_UNPACK2(T, F16))
  const void* k = dtype == TFT_F32 ? TFT_UNPACK(F32) : dtype == TFT_BF16 ? TFT_UNPACK(BF16) : TFT_UNPACK(F16);
#undef TFT_UNPACK
#undef TFT_UNPACK2
  return in_slices(rows, most_groups(kPackThreads) * kUnpackBlocks / per_row, [&](int64_t first, int64_t n) {
    UnpackArgs a{row_at(out, first, features, dtype), static_cast<const uint8_t*>(values) + first * pitch,
                 static_cast<const uint8_t*>(exponents) + first * per_row, column_scale, features, pitch,
                 (uint32_t)(n * per_row), make_divider(per_row)};
    void* params[] = {&a};
    return launch(what, k, dim3((a.blocks + kUnpackBlocks - 1) / kUnpackBlocks), kPackThreads, params,
                  static_cast<hipStream_t>(stream));
  });
}

int tft_rms_norm(void* y, void* h, void* values, void* exponents, float* rstd, const void* x,
                 const void* residual, const void* weight, int64_t rows, int64_t features,
                 int64_t x_row_stride, int64_t residual_row_stride, int64_t pitch, float eps,
                 int weight_dtype, int dtype, void* stream) {
  static const char* what = "tft_rms_norm";
  if (int rc = check_types(what, dtype, weight_dtype, weight != nullptr)) return rc;
  if (weight && weight_dtype != dtype && weight_dtype != TFT_F32)
    return fail(TFT_ERR_UNSUPPORTED, "%s: the weight is of the activations' dtype or fp32", what);
  if (rows < 0 || features < 0) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  if (features > kMostNormFeatures)
    return fail(TFT_ERR_UNSUPPORTED, "%s: %lld features, at most %d", what, (long long)features, kMostNormFeatures);
  if (rows == 0 || features == 0) return TFT_OK;
  if (rows >= kMostRows) return fail(TFT_ERR_UNSUPPORTED, "%s: %lld rows, at most 2^31 - 1", what, (long long)rows);
  if (values || exponents)
    if (int rc = check_packed(what, values, exponents, rows, features, pitch)) return rc;
  if (!x || !y || misaligned(x, dtype) || misaligned(y, dtype))
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: x or y is NULL or misaligned", what);
  if ((residual != nullptr) != (h != nullptr))
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: residual and h come together", what);
  if (residual && (misaligned(residual, dtype) || misaligned(h, dtype)))
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: residual or h is misaligned", what);
  if (weight && misaligned(weight, weight_dtype))
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: weight is misaligned", what);
  if (x_row_stride < 0 || residual_row_stride < 0)
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: negative row stride", what);
  if (!(eps >= 0.0f)) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: eps must be at least 0", what);
  NormArgs a{x, residual, weight, y, h, static_cast<uint8_t*>(values), static_cast<uint8_t*>(exponents), rstd,
             (uint32_t)rows, (int)features, x_row_stride, residual_row_stride, pitch,
             weight_dtype == TFT_F32 ? 1 : 0, eps};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool far = rows * features * (esize(dtype) * (residual ? 4 : 2) + (values ? 1 : 0)) >= kLastLevelCache;
#define TFT_NORM(T) (far ? launch_norm<T, true>(what, a, dtype, s) : launch_norm<T, false>(what, a, dtype, s))
  return dtype == TFT_F32 ? TFT_NORM(F32) : dtype == TFT_BF16 ? TFT_NORM(BF16) : TFT_NORM(F16);
#undef TFT_NORM
}

int64_t tft_rms_norm_backward_workspace(int64_t rows, int64_t features) {
  if (rows <= 0 || features <= 0 || rows >= kMostRows || features > kMostNormFeatures) return 0;
  return (int64_t)norm_back_groups(rows, features) * features * 4;
}

int tft_rms_norm_backward(void* grad_x, void* grad_weight, void* workspace, int64_t workspace_bytes,
                          const void* grad_y, const void* grad_h, const void* values,
                          const void* exponents, const float* rstd, const void* weight, int64_t rows,
                          int64_t features, int64_t grad_y_row_stride, int64_t grad_h_row_stride,
                          int64_t pitch, int weight_dtype, int dtype, void* stream) {
  static const char* what = "tft_rms_norm_backward";
  if (int rc = check_types(what, dtype, weight_dtype, weight != nullptr || grad_weight != nullptr)) return rc;
  if ((weight || grad_weight) && weight_dtype != dtype && weight_dtype != TFT_F32)
    return fail(TFT_ERR_UNSUPPORTED, "%s: the weight is of the activations' dtype or fp32", what);
  if (rows < 0 || features < 0) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  if (features > kMostNormFeatures)
    return fail(TFT_ERR_UNSUPPORTED, "%s: %lld features, at most %d", what, (long long)features, kMostNormFeatures);
  if (features == 0) return TFT_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (grad_weight && misaligned(grad_weight, weight_dtype))
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: grad_weight is misaligned", what);
  if (rows == 0)  // the empty sum
    return grad_weight ? launch_column_reduce(what, nullptr, grad_weight, 0, features, weight_dtype, s) : TFT_OK;
  if (int rc = check_packed(what, values, exponents, rows, features, pitch)) return rc;
  if (!grad_x || !grad_y || !rstd || misaligned(grad_x, dtype) || misaligned(grad_y, dtype) ||
      misaligned(rstd, TFT_F32))
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: grad_x, grad_y or rstd is NULL or misaligned", what);
  if (grad_h && misaligned(grad_h, dtype)) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: grad_h is misaligned", what);
  if (weight && misaligned(weight, weight_dtype))
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: weight is misaligned", what);
  if (grad_y_row_stride < 0 || grad_h_row_stride < 0)
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: negative row stride", what);
  if (grad_weight && (!workspace || misaligned(workspace, TFT_F32) ||
                      workspace_bytes < tft_rms_norm_backward_workspace(rows, features)))
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: workspace of %lld bytes, %lld are needed", what,
                (long long)workspace_bytes, (long long)tft_rms_norm_backward_workspace(rows, features));
  float* partial = grad_weight ? static_cast<float*>(workspace) : nullptr;
  NormBackArgs a{grad_y, grad_h, static_cast<const uint8_t*>(values), static_cast<const uint8_t*>(exponents), rstd,
                 weight, grad_x, partial, (uint32_t)rows, (int)features, grad_y_row_stride, grad_h_row_stride,
                 pitch, weight_dtype == TFT_F32 ? 1 : 0};
  const int rc = dtype == TFT_F32    ? launch_norm_back<F32>(what, a, s)
                 : dtype == TFT_BF16 ? launch_norm_back<BF16>(what, a, s)
                                     : launch_norm_back<F16>(what, a, s);
  if (rc || !grad_weight) return rc;
  return launch_column_reduce(what, partial, grad_weight, norm_back_groups(rows, features), features,
                              weight_dtype, s);
}

int64_t tft_column_sum_workspace(int64_t rows, int64_t columns) {
  if (rows <= 0 || columns <= 0 || rows >= kMostRows || columns >= kMostRows) return 0;
  return (int64_t)column_sum_groups(rows, columns) * columns * 4;
}

int tft_column_sum(void* out, void* workspace, int64_t workspace_bytes, const void* x, int64_t rows,
                   int64_t columns, int64_t x_row_stride, int out_dtype, int dtype, void* stream) {
  static const char* what = "tft_column_sum";
  if (int rc = check_types(what, dtype, out_dtype, true)) return rc;
  if (rows < 0 || columns < 0) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  if (columns == 0) return TFT_OK;
  if (rows >= kMostRows || columns >= kMostRows)
    return fail(TFT_ERR_UNSUPPORTED, "%s: at most 2^31 - 1 rows and columns", what);
  if (!out || misaligned(out, out_dtype)) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: out is NULL or misaligned", what);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows == 0) return launch_column_reduce(what, nullptr, out, 0, columns, out_dtype, s);
  if (!x || misaligned(x, dtype)) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: x is NULL or misaligned", what);
  if (x_row_stride < 0) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: negative row stride", what);
  if (!workspace || misaligned(workspace, TFT_F32) || workspace_bytes < tft_column_sum_workspace(rows, columns))
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: workspace of %lld bytes, %lld are needed", what,
                (long long)workspace_bytes, (long long)tft_column_sum_workspace(rows, columns));
  float* partial = static_cast<float*>(workspace);
  uint32_t r = (uint32_t)rows;
  void* params[] = {&x, &partial, &r, &columns, &x_row_stride};
  const dim3 grid((uint32_t)((columns + 2047) / 2048), column_sum_groups(rows, columns));
  const void* k = dtype == TFT_F32 ? TFT_KERNEL(column_sum_kernel<F32>)
                  : dtype == TFT_BF16 ? TFT_KERNEL(column_sum_kernel<BF16>)
                                      : TFT_KERNEL(column_sum_kernel<F16>);
  if (int rc = launch(what, k, grid, 256, params, s)) return rc;
  return launch_column_reduce(what, partial, out, grid.y, columns, out_dtype, s);
}

int64_t tft_linear_weight_grad_workspace(const void* grad_out, int64_t rows, int64_t out_features,
                                         int64_t features, int64_t grad_row_stride, int64_t pitch,
                                         int dtype) {
  if (rows <= 0 || out_features <= 0 || features <= 0) return 0;
  const WgradPlan p = plan_wgrad(rows, out_features, features, grad_row_stride, dtype,
                                 (reinterpret_cast<uintptr_t>(grad_out) & 15u) == 0);
  return p.aligned_bytes + p.partial_bytes;
}

int tft_linear_weight_grad(void* grad_weight, void* workspace, int64_t workspace_bytes,
                           const void* grad_out, const void* values, const void* exponents,
                           const void* column_scale, int64_t rows, int64_t out_features,
                           int64_t features, int64_t grad_row_stride, int64_t pitch, int out_dtype,
                           int scale_dtype, int dtype, void* stream) {
  static const char* what = "tft_linear_weight_grad";
  if (int rc = check_types(what, dtype, scale_dtype, column_scale != nullptr)) return rc;
  if (int rc = check_types(what, out_dtype, 0, false)) return rc;
  if (rows < 0 || out_features < 0 || features < 0)
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: negative size", what);
  if (out_features == 0 || features == 0) return TFT_OK;
  if (out_features >= kMostRows) return fail(TFT_ERR_UNSUPPORTED, "%s: at most 2^31 - 1 output features", what);
  if (!grad_weight || (reinterpret_cast<uintptr_t>(grad_weight) & 15u))
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: grad_weight is NULL or not at a multiple of 16 bytes", what);
  if (rows > 0) {
    if (int rc = check_packed(what, values, exponents, rows, features, pitch)) return rc;
    if (!grad_out || misaligned(grad_out, dtype))
      return fail(TFT_ERR_INVALID_ARGUMENT, "%s: grad_out is NULL or misaligned", what);
    if (grad_row_stride < 0) return fail(TFT_ERR_INVALID_ARGUMENT, "%s: negative row stride", what);
  }
  if (column_scale && misaligned(column_scale, scale_dtype))
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: column_scale is misaligned", what);
  const WgradPlan p = plan_wgrad(rows, out_features, features, grad_row_stride, dtype,
                                 (reinterpret_cast<uintptr_t>(grad_out) & 15u) == 0);
  // offsets within a step's rows are 31 bits
  if (p.padded * esize(dtype) * 64 >= (1ll << 31) || pitch * 64 >= (1ll << 31))
    return fail(TFT_ERR_UNSUPPORTED, "%s: rows of %lld gradients or %lld packed values are too long", what,
                (long long)p.padded, (long long)pitch);
  if ((int64_t)p.tiles_o * p.tiles_f * 4 >= (1ll << 31) ||
      p.whole + (int64_t)p.cut * p.splits > most_groups(p.large ? 512 : 256))
    return fail(TFT_ERR_UNSUPPORTED, "%s: too many tiles for one grid", what);
  const int64_t needed = p.aligned_bytes + p.partial_bytes;
  if (needed && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) || workspace_bytes < needed))
    return fail(TFT_ERR_INVALID_ARGUMENT, "%s: workspace of %lld bytes, %lld are needed", what,
                (long long)workspace_bytes, (long long)needed);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const AlignArgs align{grad_out, workspace, out_features, grad_row_stride, p.padded,
                        (uint64_t)rows * (uint64_t)(p.padded / 8)};
  const WgradArgs a{p.align_first ? workspace : grad_out, static_cast<const uint8_t*>(values),
                    static_cast<const uint8_t*>(exponents), column_scale, grad_weight,
                    reinterpret_cast<float*>(static_cast<char*>(workspace) + p.aligned_bytes), rows, p.padded, pitch,
                    (uint32_t)out_features, (uint32_t)features, (uint32_t)((features + kBlock - 1) / kBlock),
                    p.tiles_o, p.tiles_f, p.whole, p.cut, p.splits, p.steps, scale_dtype, out_dtype,
                    p.partial_bytes <= kL2Bytes ? 1 : 0};
  if (dtype == TFT_F32) return launch_wgrad<F32>(what, a, p, align, s);
  if (dtype == TFT_BF16) return launch_wgrad<BF16>(what, a, p, align, s);
  return launch_wgrad<F16>(what, a, p, align, s);
}

}  // extern "C"
