// AdamW over many tensors in a few launches, both moments in 32 or in 8 bits, with the gradients' joint 2-norm for
// clipping.  The reference builds one torch.optim.Adam per network (render_surface.py:213-231); with weight_decay = 0
// this is the same step:
//   g' = g min(1, max_norm / (|g| + 1e-6))                                       (only with max_norm)
//   m  = beta1 m + (1 - beta1) g'          v = beta2 v + (1 - beta2) g'^2
//   p  = p - lr weight_decay p - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)
//
// 8-bit moments: 256 consecutive elements of a tensor share one scale per moment,
//   m = a (q / 127) |q / 127|, q in [-127, 127]          v = b (c / 255)^4, c in [0, 255]
// with a, b the block's largest |m| and v in fp32.  The power laws make a code's step relative to the value small near
// the largest (2/127 and 4/255) and still reach 6e-5 a and 2e-10 b; what all elements of a block have in common -- the
// decay by beta -- is carried by the fp32 scale, so that no code can get stuck on it.
#include "pir_common.h"
#include <cmath>

namespace pir {

constexpr int kOptThreads = 256;
constexpr int kOptBlock = 256;                // elements that share a scale
constexpr int kOptChunk = 1024;               // elements one workgroup updates, with 32-bit moments
constexpr int kOptChunk8 = 2048;              // and with 8-bit ones
constexpr int kPrepRows = 104;                // tensors and hyper-parameter sets per prologue launch: what 4 KB of kernel
constexpr int kPrepGroups = 8;                // arguments hold
constexpr int kPrepThreads = 1024;
constexpr long kNormChunk = 4096;             // the smallest number of elements a workgroup sums
constexpr int kNormTable = 312;               // tensors per launch of the norm's first pass
constexpr int kFinishWaves = 4;              // tensors per workgroup of the second pass (16: 3.6 us, 4: 2.8 for 126 tensors)
constexpr int kFirstTable = 1000;             // tensors per launch of that

// what one tensor's update needs, computed once per step by the prologue
struct OptCoef {
  float b1, c1, b2, c2;                       // beta, 1 - beta
  float size, root, eps, decay;               // lr / (1 - beta1^t), (1 - beta2^t)^-1/2, eps, lr weight_decay
  float gscale, run, pad0, pad1;              // clip factor; run = 0: leave the tensor as it is
};

// One tensor as the update kernels read it from the workspace.  The descriptors reach the device as arguments of the
// prologue, never by a copy from host memory that a captured graph would read again at its replays.
struct OptRow {
  void* param;
  const void* grad;
  void* m;
  void* v;
  float* scales;
  long numel;
};

// A row on its way, in 32 bytes: addresses as differences from those of the launch's first row, parameters and gradients
// in units of 2 bytes, the others of 4.  A tensor that is too far away starts another launch.
struct PrepRow {
  int param, grad, m, v, scales, step;
  unsigned numel;                             // lower 32 bits
  unsigned first;                             // first workgroup of the tensor within its launch (24 bits), group (3), numel (5)
};

struct PrepGroup {
  double lr, log1, log2, wd;
  const float* lr_device;
  float b1, c1, b2, c2, eps, pad;
};

struct PrepTable {
  int n, row0, n_partial, finalize, clip, skip, n_groups, pad;
  double max_norm;
  const double* partial;
  float* norm;                                // [total, clip factor]; NULL: no norm wanted
  float* total;                               // the caller's copy of the norm, or NULL
  OptRow* rows;
  OptCoef* coef;
  unsigned* first;
  OptRow base;
  float* step_base;
  PrepGroup g[kPrepGroups];
  PrepRow row[kPrepRows];
};

struct NormTable {
  int n;
  unsigned chunk;                             // elements one workgroup sums
  double* partial;
  const void* base;                           // the first tensor; the others by their differences, in units of 2 bytes
  int grad[kNormTable];
  unsigned numel[kNormTable];                 // lower 32 bits
  unsigned first[kNormTable];                 // first workgroup
  unsigned char more[kNormTable];             // type (2 bits), upper bits of numel
};

struct FinishTable {
  int n, n_partial;
  const double* partial;
  float* total;                               // NULL: another launch writes it
  float* each;
  unsigned first[kFirstTable + 1];            // first partial sum of each tensor, and the end
};

static_assert(sizeof(PrepTable) <= 4096 && sizeof(NormTable) <= 4096 && sizeof(FinishTable) <= 4096, "kernel arguments");

template <typename T> __device__ inline float to_float(T x) { return (float)x; }
template <typename T> __device__ inline T from_float(float x) { return (T)x; }   // round to nearest even

// N values of type T at any address that is a multiple of sizeof(T): one wide access all the same
template <typename T, int N> struct Vec { typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T)))); };

// kStream: accesses that leave the caches to others, where the call's data exceeds the last-level one.  284 M fp32 elements
// take 1.41 ms with them, 1.51 without; 7.3 M with 8-bit moments (117 MB, which the next call finds in the cache) 55.5 us
// with them, 51.5 without.
template <bool kStream, typename T, int N>
__device__ inline void load(float (&x)[N], const T* __restrict__ p) {
  const typename Vec<T, N>::type* q = (const typename Vec<T, N>::type*)p;
  const typename Vec<T, N>::type r = kStream ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
  for (int j = 0; j < N; ++j) x[j] = to_float(r[j]);
}

template <bool kStream, typename T, int N>
__device__ inline void store(T* __restrict__ p, const float (&x)[N]) {
  typename Vec<T, N>::type* q = (typename Vec<T, N>::type*)p;
  typename Vec<T, N>::type r;
#pragma unroll
  for (int j = 0; j < N; ++j) r[j] = from_float<T>(x[j]);
  if (kStream) __builtin_nontemporal_store(r, q); else *q = r;
}

// The last i with first[i] <= block, by a whole wave, 64 candidates at a time (first[0] = 0, ascending): two dependent
// reads for up to 4096 tensors.
__device__ inline int find_tensor(const unsigned* first, int n, unsigned block) {
  const int lane = threadIdx.x & 63;
  int lo = 0, len = n;
  while (len > 1) {
    const int stride = (len + 63) >> 6;
    const bool below = lane * stride < len && first[lo + lane * stride] <= block;
    const int part = __popcll(__ballot(below)) - 1;
    lo += part * stride;
    len = len - part * stride < stride ? len - part * stride : stride;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

struct UpdateArgs {
  const OptRow* rows;
  const OptCoef* coef;
  const unsigned* first;
  int n;
};

// 32-bit moments, 4 consecutive elements a thread and no loop: 28 bytes an element in fp32, 22 in 16 bits, bound by memory.
// 284 M fp32 elements: 1.31 ms, 6.1 TB/s; 88 M bf16: 0.29 ms, 6.6 TB/s.  What a workgroup covers decides how near to each
// other the card's accesses lie: with 32768, 8192 and 2048 elements a workgroup the fp32 step took 1.60, 1.54 and 1.51 ms,
// with streaming accesses 1.47 (8192), 1.41 (2048) and 1.34 (1024, as here; 512: 1.35).
template <typename T, bool kStream>
__global__ void __launch_bounds__(kOptThreads)
adamw32_kernel(const UpdateArgs args) {
  static_assert(kOptChunk == 4 * kOptThreads, "4 elements a thread");
  const int k = find_tensor(args.first, args.n, blockIdx.x);
  const OptCoef c = args.coef[k];
  if (c.run == 0.0f) return;
  const OptRow t = args.rows[k];
  const long end = t.numel, i = (long)(blockIdx.x - args.first[k]) * kOptChunk + 4 * threadIdx.x;
  T* __restrict__ P = (T*)t.param;
  const T* __restrict__ G = (const T*)t.grad;
  float* __restrict__ M = (float*)t.m;
  float* __restrict__ V = (float*)t.v;
  const bool whole = i + 4 <= end;
  float p[4], g[4], m[4], v[4];
  if (whole) {
    load<kStream>(p, P + i);
    load<kStream>(g, G + i);
    load<kStream>(m, M + i);
    load<kStream>(v, V + i);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = i + j < end;
      p[j] = in ? to_float(P[i + j]) : 0.0f;
      g[j] = in ? to_float(G[i + j]) : 0.0f;
      m[j] = in ? M[i + j] : 0.0f;
      v[j] = in ? V[i + j] : 0.0f;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float gj = g[j] * c.gscale;
    m[j] = fmaf(c.b1, m[j], c.c1 * gj);
    v[j] = fmaf(c.b2, v[j], c.c2 * gj * gj);
    const float u = m[j] / fmaf(sqrtf(v[j]), c.root, c.eps);
    p[j] -= fmaf(c.decay, p[j], c.size * u);  // the decay is added to the step: 1 - lr wd in fp32 would lose a small one
  }
  if (whole) {
    store<kStream>(P + i, p);
    store<kStream>(M + i, m);
    store<kStream>(V + i, v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < end) {
        P[i + j] = from_float<T>(p[j]);
        M[i + j] = m[j];
        V[i + j] = v[j];
      }
  }
}

// The scale of a block from the largest bit pattern of its magnitudes: integers order like the floats they stand for,
// with infinities and NaN on top.  Below 2^-126 the block is zero; a value that is not finite makes the scale NaN.
__device__ inline float block_scale(unsigned top) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return top < 0x00800000u ? 0.0f : __uint_as_float(top);
}

__device__ inline unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }
__device__ inline unsigned umin(unsigned a, unsigned b) { return a < b ? a : b; }
__device__ inline unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <int kCtrl>
__device__ inline unsigned dpp_max(unsigned x) {
  return umax(x, (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, kCtrl, 0xf, 0xf, false));
}

// the largest of the 32 lanes that share a block, in all of them: lanes 1 and 2 apart, the mirrors of 8 and of 16, then
// the two rows of 16
__device__ inline unsigned half_max(unsigned x) {
  x = dpp_max<0xB1>(x);
  x = dpp_max<0x4E>(x);
  x = dpp_max<0x141>(x);
  x = dpp_max<0x140>(x);
  const auto rows = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return umax(rows[0], rows[1]);
}

__device__ inline float decode_m(int q, float a) { const float x = (float)q * (1.0f / 127.0f); return a * (x * fabsf(x)); }
__device__ inline float decode_v(int c, float b) { const float x = (float)c * (1.0f / 255.0f), y = x * x; return b * (y * y); }

__device__ inline int encode_m(float m, float a) {
  if (!(a > 0.0f)) return 0;
  const int q = (int)rintf(127.0f * sqrtf(fabsf(m) / a));
  return m < 0.0f ? -q : q;
}

__device__ inline int encode_v(float v, float b) {
  if (!(b > 0.0f) || !(v > 0.0f)) return 0;   // else at least 1: a denominator never loses its moment
  const int c = (int)rintf(255.0f * sqrtf(sqrtf(v / b)));
  return c < 1 ? 1 : c;
}

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef signed char s8x8 __attribute__((ext_vector_type(8)));
typedef unsigned char u8x8 __attribute__((ext_vector_type(8)));

// 1.5 2^23: adding it to a number below 2^22 rounds that to the nearest integer, ties to even, and leaves the integer in
// the low bits, negative ones in two's complement
constexpr float kRoundBits = 12582912.0f;

__device__ inline unsigned pack_low_bytes(float a, float b, float c, float d) {
  const unsigned lo = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x0c0c0400);
  const unsigned hi = __builtin_amdgcn_perm(__float_as_uint(d), __float_as_uint(c), 0x04000c0c);
  return lo | hi;
}

// 8-bit moments: half a wave per block of 256 elements, 8 consecutive ones per lane.  10 bytes an element (16-bit
// parameters) leave the vector unit about 60 operations each, so the arithmetic is counted (it takes 49): square roots and
// reciprocals are the hardware's (one ulp; about 5e-6 of the codes differ by one from those of correctly rounded ones), the
// root of v serves the step and the new code, codes are rounded and packed as bits, and maxima cross lanes without shared
// memory.  435 M bf16 elements: 0.69 ms, 6.4 TB/s, bound by memory; with IEEE roots and divisions and shuffles through
// shared memory 1.51 ms.
template <typename T, bool kStream>
__global__ void __launch_bounds__(kOptThreads)
adamw8_kernel(const UpdateArgs args) {
  static_assert(kOptChunk8 == 8 * kOptThreads, "8 elements a thread");
  const int k = find_tensor(args.first, args.n, blockIdx.x);
  const OptCoef c = args.coef[k];
  if (c.run == 0.0f) return;
  const OptRow t = args.rows[k];
  const long end = t.numel, i = (long)(blockIdx.x - args.first[k]) * kOptChunk8 + 8 * threadIdx.x;
  T* __restrict__ P = (T*)t.param;
  const T* __restrict__ G = (const T*)t.grad;
  if (i - (i & (kOptBlock - 1)) >= end) return;       // no such block
  u32x2* mq = (u32x2*)((signed char*)t.m + i);
  u32x2* vq = (u32x2*)((unsigned char*)t.v + i);
  float2* sc = (float2*)t.scales + i / kOptBlock;
  u32x2 q = kStream ? __builtin_nontemporal_load(mq) : *mq, w = kStream ? __builtin_nontemporal_load(vq) : *vq;
  const float2 ab = *sc;
  const bool whole = i + 8 <= end;
  float p[8], g[8], m[8], r[8];
  if (whole) {
    load<kStream>(p, P + i);
    load<kStream>(g, G + i);
  } else {                                  // what fills up the last block is zero, and stays so
    unsigned long keep = i < end ? (1ul << (8 * (end - i))) - 1 : 0;
    q.x &= (unsigned)keep;
    q.y &= (unsigned)(keep >> 32);
    w.x &= (unsigned)keep;
    w.y &= (unsigned)(keep >> 32);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = i + j < end ? to_float(P[i + j]) : 0.0f;
      g[j] = i + j < end ? to_float(G[i + j]) : 0.0f;
    }
  }
  const float a1 = c.b1 * ab.x, b2 = c.b2 * ab.y;
  float ma = 0.0f;
  unsigned mb = 0, low = ~0u;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int qj = (int)((j < 4 ? q.x : q.y) << (24 - 8 * (j & 3))) >> 24;
    const unsigned wj = ((j < 4 ? w.x : w.y) >> (8 * (j & 3))) & 255u;
    const float x = (float)qj * (1.0f / 127.0f), y = (float)wj * (1.0f / 255.0f), y2 = y * y;
    const float gj = g[j] * c.gscale;
    m[j] = fmaf(a1, x * fabsf(x), c.c1 * gj);
    r[j] = fmaf(b2, y2 * y2, c.c2 * gj * gj);
    ma = fmaxf(ma, fabsf(m[j]));
    mb = umax(mb, __float_as_uint(r[j]));   // v is not below zero: its bits order as it does, NaN on top
    low = umin(low, __float_as_uint(r[j]));
  }
  if (low < 0x00800000u) {                  // the hardware's root takes what is below 2^-126 for zero: 2^64 v, 2^-32 its root
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool tiny = r[j] < 0x1p-126f;
      r[j] = __builtin_amdgcn_sqrtf(r[j] * (tiny ? 0x1p64f : 1.0f)) * (tiny ? 0x1p-32f : 1.0f);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = __builtin_amdgcn_sqrtf(r[j]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float u = m[j] * __builtin_amdgcn_rcpf(fmaf(r[j], c.root, c.eps));
    p[j] -= fmaf(c.decay, p[j], c.size * u);
  }
  if (whole) {
    store<kStream>(P + i, p);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < end) P[i + j] = from_float<T>(p[j]);
  }
  const float nb = block_scale(half_max(mb));
  float na = block_scale(half_max(__float_as_uint(ma)));
  // the maximum of floats passes over a NaN: one of g is in v too, one of a scale is in the whole block
  na = nb != nb ? nb : ab.x != ab.x ? ab.x : na;
  const float ra = na > 0.0f ? 1.0f / na : 0.0f, rb = nb > 0.0f ? __builtin_amdgcn_rsqf(nb) : 0.0f;
  const float live = nb > 0.0f ? 0x1p127f : 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = copysignf(__builtin_amdgcn_sqrtf(fabsf(m[j]) * ra), m[j]);
    const float y = __builtin_amdgcn_sqrtf(r[j] * rb);
    const float least = __builtin_amdgcn_fmed3f(r[j] * live, 0.0f, 1.0f / 255.0f);   // c >= 1 if v > 0: no
    m[j] = fmaf(x, 127.0f, kRoundBits);                                              // denominator is lost
    r[j] = fmaf(fmaxf(y, least), 255.0f, kRoundBits);
  }
  q = u32x2{pack_low_bytes(m[0], m[1], m[2], m[3]), pack_low_bytes(m[4], m[5], m[6], m[7])};
  w = u32x2{pack_low_bytes(r[0], r[1], r[2], r[3]), pack_low_bytes(r[4], r[5], r[6], r[7])};
  if (kStream) {
    __builtin_nontemporal_store(q, mq);
    __builtin_nontemporal_store(w, vq);
  } else {
    *mq = q;
    *vq = w;
  }
  if ((threadIdx.x & 31) == 0) *sc = make_float2(na, nb);
}

// 435 M elements to bf16 (2.6 GB): 0.42 ms, 6.2 TB/s; to fp32 (4.4 GB) 1.64 ms, 2.7 TB/s
template <typename T>
__global__ void __launch_bounds__(kOptThreads)
moments8_decode_kernel(long n_blocks, const signed char* __restrict__ mq, const unsigned char* __restrict__ vq,
                       const float* __restrict__ scales, T* __restrict__ m, T* __restrict__ v) {
  const long i = 8 * ((long)blockIdx.x * kOptThreads + threadIdx.x);
  if (i >= n_blocks * kOptBlock) return;
  const s8x8 q = __builtin_nontemporal_load((const s8x8*)(mq + i));
  const u8x8 w = __builtin_nontemporal_load((const u8x8*)(vq + i));
  const float2 ab = ((const float2*)scales)[i / kOptBlock];
  float x[8], y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = decode_m(q[j], ab.x);
    y[j] = decode_v(w[j], ab.y);
  }
  store<true>(m + i, x);
  store<true>(v + i, y);
}

// Guarded loads of one element each, not tuned: a program encodes when it loads or converts a state.  435 M elements of
// bf16 (2.6 GB): 1.3 ms, 2.0 TB/s; of fp32 (4.4 GB) 1.56 ms, 2.8 TB/s.
template <typename T>
__global__ void __launch_bounds__(kOptThreads)
moments8_encode_kernel(long numel, const T* __restrict__ m, const T* __restrict__ v, signed char* __restrict__ mq,
                       unsigned char* __restrict__ vq, float* __restrict__ scales) {
  const long i = 8 * ((long)blockIdx.x * kOptThreads + threadIdx.x);
  if (i - (i & (kOptBlock - 1)) >= numel) return;
  float x[8], y[8];
  unsigned ma = 0, mb = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = i + j < numel ? to_float(m[i + j]) : 0.0f;
    y[j] = i + j < numel ? to_float(v[i + j]) : 0.0f;
    ma = umax(ma, magnitude(x[j]));
    mb = umax(mb, magnitude(y[j]));
  }
  const float a = block_scale(half_max(ma)), b = block_scale(half_max(mb));
  s8x8 q;
  u8x8 w;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    q[j] = (signed char)encode_m(x[j], a);
    w[j] = (unsigned char)encode_v(y[j], b);
  }
  *(s8x8*)(mq + i) = q;
  *(u8x8*)(vq + i) = w;
  if ((threadIdx.x & 31) == 0) ((float2*)scales)[i / kOptBlock] = make_float2(a, b);
}

// ---- norms: squares and sums in 64 bits (no overflow for any fp32 gradient), one partial sum per workgroup, added up
// in a fixed order: the same bits on every run.  Bound by memory (6.9 TB/s at 284 M fp32 elements).  Gradients that fit the
// last-level cache are left there: the step reads them again (88 M bf16, clipped: 330 us, 352 with streaming reads).

__device__ inline double wave_sum(double x) {
  for (int d = 32; d >= 1; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

// 16 bytes a thread and load, four of them in flight
template <int kThreads, bool kStream, typename T>
__device__ inline double sum_squares(const T* __restrict__ g, long base, long end) {
  constexpr int N = 16 / sizeof(T);
  constexpr long kRow = (long)N * kThreads;
  double s0 = 0.0, s1 = 0.0;
  long i = base + N * threadIdx.x;
  for (; i + 3 * kRow + N <= end; i += 4 * kRow) {
    float x[4][N];
#pragma unroll
    for (int h = 0; h < 4; ++h) load<kStream>(x[h], g + i + h * kRow);
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        s0 = fma((double)x[h][j], (double)x[h][j], s0);
        s1 = fma((double)x[h][j + 1], (double)x[h][j + 1], s1);
      }
  }
  for (; i < end; i += kRow) {
    float x[N];
    if (i + N <= end) {
      load<kStream>(x, g + i);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = i + j < end ? to_float(g[i + j]) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      s0 = fma((double)x[j], (double)x[j], s0);
      s1 = fma((double)x[j + 1], (double)x[j + 1], s1);
    }
  }
  return s0 + s1;
}

template <int kThreads, bool kStream>
__global__ void __launch_bounds__(kThreads)
norm_partial_kernel(const NormTable tab) {
  __shared__ double part[kThreads / 64];
  const int k = find_tensor(tab.first, tab.n, blockIdx.x);
  const int dtype = tab.more[k] & 3;
  const void* grad = (const short*)tab.base + tab.grad[k];
  const long base = (long)(blockIdx.x - tab.first[k]) * tab.chunk, numel = (long)(tab.more[k] >> 2) << 32 | tab.numel[k];
  const long end = base + tab.chunk < numel ? base + tab.chunk : numel;
  double s;
  if (dtype == PIR_F32) s = sum_squares<kThreads, kStream>((const float*)grad, base, end);
  else if (dtype == PIR_BF16) s = sum_squares<kThreads, kStream>((const __bf16*)grad, base, end);
  else s = sum_squares<kThreads, kStream>((const _Float16*)grad, base, end);
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < kThreads / 64; ++w) s += part[w];
  tab.partial[blockIdx.x] = s;
}

// sum of the partials by a workgroup of kPrepThreads
__device__ inline double sum_partials(const double* __restrict__ partial, int n, double* part) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kPrepThreads) s += partial[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  double all = 0.0;
  for (int i = 0; i < kPrepThreads / 64; ++i) all += part[i];
  return all;
}

// One workgroup: the joint norm and clip factor from the partial sums, then the step counts and coefficients of its
// tensors (in 64 bits: 1 - beta2^t at t = 1 loses three digits in 32), and their descriptors for the update kernels.  2.4 to
// 4 us, nearly all of it the launch and one chain of dependent reads; it spares every workgroup of the update the 64-bit
// exponentials, and a step of many tensors all but one update launch (301 tensors, clipped: 155 us with 64 tensors a launch, 48 so).
__global__ void __launch_bounds__(kPrepThreads)
adamw_prologue_kernel(const PrepTable tab) {
  __shared__ double part[kPrepThreads / 64];
  float norm = 0.0f, clip = 1.0f;
  if (tab.norm) {
    if (tab.finalize) {
      const double all = sqrt(sum_partials(tab.partial, tab.n_partial, part));
      norm = (float)all;
      if (tab.clip) {
        const double f = tab.max_norm / (all + 1e-6);
        clip = f < 1.0 ? (float)f : (f >= 1.0 ? 1.0f : (float)f);      // NaN stays NaN
      }
      if (threadIdx.x == 0) {
        tab.norm[0] = norm;
        tab.norm[1] = clip;
        if (tab.total) *tab.total = norm;
      }
    } else {
      norm = tab.norm[0];
      clip = tab.norm[1];
    }
  }
  const bool run = !tab.skip || (norm - norm == 0.0f);
  const int i = threadIdx.x;
  if (i >= tab.n) return;
  const PrepRow& r = tab.row[i];
  const PrepGroup& g = tab.g[r.first >> 24 & 7];
  float* step = tab.step_base + r.step;
  const float t = *step + 1.0f;
  const double lr = g.lr_device ? (double)*g.lr_device : g.lr;
  OptCoef c;
  c.b1 = g.b1;
  c.c1 = g.c1;
  c.b2 = g.b2;
  c.c2 = g.c2;
  c.size = (float)(lr / -expm1((double)t * g.log1));
  c.root = (float)(1.0 / sqrt(-expm1((double)t * g.log2)));
  c.eps = g.eps;
  c.decay = (float)(lr * g.wd);
  c.gscale = clip;
  c.run = run ? 1.0f : 0.0f;
  c.pad0 = c.pad1 = 0.0f;
  tab.coef[tab.row0 + i] = c;
  OptRow row;
  row.param = (short*)tab.base.param + r.param;
  row.grad = (const short*)tab.base.grad + r.grad;
  row.m = (int*)tab.base.m + r.m;
  row.v = (int*)tab.base.v + r.v;
  row.scales = tab.base.scales + r.scales;
  row.numel = (long)(r.first >> 27) << 32 | r.numel;
  tab.rows[tab.row0 + i] = row;
  tab.first[tab.row0 + i] = r.first & 0xffffffu;
  if (run) *step = t;
}

// norms of all tensors together (workgroup 0 of the first launch) and of each (a wave each, in the others), from the
// partial sums
__global__ void __launch_bounds__(kPrepThreads)
norm_finish_kernel(const FinishTable tab) {
  __shared__ double part[kPrepThreads / 64];
  int group = blockIdx.x;
  if (tab.total) {
    if (group == 0) {
      const double all = sum_partials(tab.partial, tab.n_partial, part);
      if (threadIdx.x == 0) *tab.total = (float)sqrt(all);
      return;
    }
    --group;
  }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, k = group * kFinishWaves + wave;
  if (wave >= kFinishWaves || k >= tab.n) return;
  double x = 0.0;
  for (unsigned i = tab.first[k] + lane; i < tab.first[k + 1]; i += 64) x += tab.partial[i];
  x = wave_sum(x);
  if (lane == 0) tab.each[k] = (float)sqrt(x);
}

static inline long ceil_div(long a, long b) { return (a + b - 1) / b; }

static const long kMaxGroups = (1L << 24) - 1;     // workgroups: a grid has fewer than 2^32 threads
static const long kCacheBytes = 256L << 20;        // last-level cache

static inline long element_bytes(int dtype) { return dtype == PIR_F32 ? 4 : 2; }

// scales[i]: whether tensor i has 8-bit moments (scales NULL: none has)
static int check_tensors(int n, const long* numels, const int* dtypes, const void* const* grads, float* const* scales) {
  if (n < 0 || (n > 0 && (!numels || !dtypes || !grads))) return PIR_ERR_ARG;
  long groups = 0;
  for (int i = 0; i < n; ++i) {
    if (numels[i] < 0 || dtypes[i] < PIR_F32 || dtypes[i] > PIR_F16) return PIR_ERR_ARG;
    if ((numels[i] > 0 && !grads[i]) || ((size_t)grads[i] & (element_bytes(dtypes[i]) - 1))) return PIR_ERR_ARG;
    if (numels[i] > kMaxGroups * kOptChunk8) return PIR_ERR_TOO_LARGE;
    groups += ceil_div(numels[i], scales && scales[i] ? kOptChunk8 : kOptChunk);
    if (groups > kMaxGroups) return PIR_ERR_TOO_LARGE;
  }
  return PIR_OK;
}

// Elements a workgroup takes: as few as fill the card when there is little to do (4096 for 256 threads: 4.5 us for 2.4 M
// fp32 elements, 6.9 with 1024 threads), more of them when there is much, so that the search for its tensor and the second
// pass over the partial sums stay small beside it (65536 for 1024 threads: 164 us for 284 M, 6.9 TB/s; with 256 threads 190).
static unsigned norm_chunk(int n, const long* numels) {
  long total = 0;
  for (int i = 0; i < n; ++i) total += numels[i];
  long chunk = kNormChunk;
  while (chunk < 65536 && total / chunk > 4096) chunk *= 2;
  return (unsigned)chunk;
}

static long norm_partials(int n, const long* numels) {
  const unsigned chunk = norm_chunk(n, numels);
  long c = 0;
  for (int i = 0; i < n; ++i) c += ceil_div(numels[i], chunk);
  return c;
}

// to - from in units of 1 << shift bytes; whether it fits
static inline bool difference(const void* to, const void* from, int shift, int& d) {
  const long x = ((long)to - (long)from) >> shift;
  d = (int)x;
  return x == d;
}

static int launch_partials(int n, const void* const* grads, const long* numels, const int* dtypes, double* partial,
                           hipStream_t stream) {
  NormTable tab;
  tab.n = 0;
  tab.chunk = norm_chunk(n, numels);
  tab.partial = partial;
  long at = 0, bytes = 0;                       // workgroups of this launch so far
  for (int i = 0; i < n; ++i) bytes += numels[i] * element_bytes(dtypes[i]);
  for (int i = 0; i <= n; ++i) {
    const long blocks = i < n ? ceil_div(numels[i], tab.chunk) : 0;
    if (i < n && blocks == 0) continue;
    int away = 0;
    if (tab.n > 0 && (i == n || tab.n == kNormTable || !difference(grads[i], tab.base, 1, away))) {
      const dim3 grid((unsigned)at);
      if (bytes > kCacheBytes) hipLaunchKernelGGL((norm_partial_kernel<1024, true>), grid, dim3(1024), 0, stream, tab);
      else if (tab.chunk > kNormChunk) hipLaunchKernelGGL((norm_partial_kernel<1024, false>), grid, dim3(1024), 0, stream, tab);
      else hipLaunchKernelGGL((norm_partial_kernel<256, false>), grid, dim3(256), 0, stream, tab);
      tab.partial += at;
      tab.n = 0;
      at = away = 0;
    }
    if (i == n) break;
    if (tab.n == 0) tab.base = grads[i];
    tab.grad[tab.n] = away;
    tab.numel[tab.n] = (unsigned)numels[i];
    tab.more[tab.n] = (unsigned char)(numels[i] >> 32 << 2 | dtypes[i]);
    tab.first[tab.n] = (unsigned)at;
    at += blocks;
    ++tab.n;
  }
  return pir_check_launch();
}

template <bool kStream>
static void launch_update(int kind, const UpdateArgs& args, long groups, hipStream_t stream) {
  const dim3 grid((unsigned)groups), block(kOptThreads);
  switch (kind) {
    case PIR_F32: hipLaunchKernelGGL((adamw32_kernel<float, kStream>), grid, block, 0, stream, args); break;
    case PIR_BF16: hipLaunchKernelGGL((adamw32_kernel<__bf16, kStream>), grid, block, 0, stream, args); break;
    case PIR_F16: hipLaunchKernelGGL((adamw32_kernel<_Float16, kStream>), grid, block, 0, stream, args); break;
    case 3 + PIR_F32: hipLaunchKernelGGL((adamw8_kernel<float, kStream>), grid, block, 0, stream, args); break;
    case 3 + PIR_BF16: hipLaunchKernelGGL((adamw8_kernel<__bf16, kStream>), grid, block, 0, stream, args); break;
    default: hipLaunchKernelGGL((adamw8_kernel<_Float16, kStream>), grid, block, 0, stream, args);
  }
}

static PrepGroup prologue_group(const PirAdamwGroup& g) {
  PrepGroup d;
  d.lr = g.lr;
  d.lr_device = g.lr_device;
  d.log1 = std::log(g.beta1);
  d.log2 = std::log(g.beta2);
  d.wd = g.weight_decay;
  d.b1 = (float)g.beta1;
  d.c1 = (float)(1.0 - g.beta1);
  d.b2 = (float)g.beta2;
  d.c2 = (float)(1.0 - g.beta2);
  d.eps = (float)g.eps;
  d.pad = 0.0f;
  return d;
}

// the row's addresses as differences from the launch's; false: some do not fit.  An empty tensor has none that count, and
// a launch whose first tensor is empty takes no others but such.
static bool relative(const OptRow& row, const float* step, const PrepTable& tab, PrepRow& r) {
  r.param = r.grad = r.m = r.v = r.scales = 0;
  if (!difference(step, tab.step_base, 2, r.step)) return false;
  if (row.numel == 0) return true;
  if (tab.base.numel == 0) return false;
  if (!difference(row.param, tab.base.param, 1, r.param) || !difference(row.grad, tab.base.grad, 1, r.grad) ||
      !difference(row.m, tab.base.m, 2, r.m) || !difference(row.v, tab.base.v, 2, r.v))
    return false;
  return !row.scales || difference(row.scales, tab.base.scales, 2, r.scales);
}

static long align16(long x) { return (x + 15) & ~15L; }

// the parts of a step's workspace, by their offsets
struct StepSpace {
  long rows, coef, first, partial, bytes;
  StepSpace(int n, const long* numels, bool with_norm) {
    rows = 16;                                  // [norm, clip factor, -, -] in front
    coef = rows + (long)n * (long)sizeof(OptRow);
    first = coef + (long)n * (long)sizeof(OptCoef);
    partial = align16(first + 4L * n);
    bytes = partial + (with_norm ? 8 * norm_partials(n, numels) : 0);
  }
};

}  // namespace pir

using namespace pir;

extern "C" {

size_t pir_adamw_workspace_bytes(int n, const long* numels, int with_norm) {
  if (n < 0 || (n > 0 && !numels)) return 0;
  return (size_t)StepSpace(n, numels, with_norm != 0).bytes;
}

int pir_adamw_step(int n, void* const* params, const void* const* grads, void* const* exp_avgs, void* const* exp_avg_sqs,
                   float* const* scales, float* const* steps, const long* numels, const int* dtypes, const int* groups,
                   const PirAdamwGroup* group, int n_groups, double max_norm, int skip_nonfinite, float* total_norm,
                   void* workspace, size_t workspace_bytes, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  const int rc = check_tensors(n, numels, dtypes, grads, scales);
  if (rc != PIR_OK) return rc;
  if (n > 0 && (!params || !exp_avgs || !exp_avg_sqs || !steps || !groups || !group || n_groups < 1)) return PIR_ERR_ARG;
  for (int k = 0; k < n_groups && n > 0; ++k) {
    const PirAdamwGroup& g = group[k];
    if (!(g.beta1 >= 0 && g.beta1 < 1 && g.beta2 >= 0 && g.beta2 < 1 && g.eps >= 0 && g.lr >= 0 && g.weight_decay >= 0) ||
        ((size_t)g.lr_device & 3))
      return PIR_ERR_ARG;
  }
  for (int i = 0; i < n; ++i) {
    if (!steps[i] || groups[i] < 0 || groups[i] >= n_groups) return PIR_ERR_ARG;
    if (numels[i] > 0 && (!params[i] || !exp_avgs[i] || !exp_avg_sqs[i])) return PIR_ERR_ARG;
    if (((size_t)params[i] & (element_bytes(dtypes[i]) - 1)) || (((size_t)exp_avgs[i] | (size_t)exp_avg_sqs[i] | (size_t)steps[i]) & 3))
      return PIR_ERR_ARG;
    if (scales && scales[i] && ((((size_t)exp_avgs[i] | (size_t)exp_avg_sqs[i]) & 15) || ((size_t)scales[i] & 7) ||
                                group[groups[i]].eps < 1e-30))
      return PIR_ERR_ARG;
  }
  const bool clip = max_norm > 0.0, with_norm = clip || skip_nonfinite || total_norm;
  if ((size_t)total_norm & 3) return PIR_ERR_ARG;
  if (n == 0 && !total_norm) return PIR_OK;
  const StepSpace space(n, numels, with_norm);
  if (!workspace || ((size_t)workspace & 15) || workspace_bytes < (size_t)space.bytes) return PIR_ERR_SCRATCH;
  char* ws = (char*)workspace;
  OptRow* rows = (OptRow*)(ws + space.rows);
  OptCoef* coef = (OptCoef*)(ws + space.coef);
  unsigned* first = (unsigned*)(ws + space.first);
  double* partial = (double*)(ws + space.partial);
  long bytes = 0;                               // what the update touches: parameter, gradient, two moments
  for (int i = 0; i < n; ++i) bytes += numels[i] * (2 * element_bytes(dtypes[i]) + (scales && scales[i] ? 2 : 8));
  if (with_norm && launch_partials(n, grads, numels, dtypes, partial, stream) != PIR_OK) return PIR_ERR_LAUNCH;

  PrepTable tab;
  tab.n = tab.row0 = tab.n_groups = tab.pad = 0;
  tab.n_partial = with_norm ? (int)norm_partials(n, numels) : 0;
  tab.finalize = 1;
  tab.clip = clip;
  tab.skip = skip_nonfinite != 0;
  tab.max_norm = max_norm;
  tab.partial = partial;
  tab.norm = with_norm ? (float*)ws : nullptr;
  tab.total = total_norm;
  tab.rows = rows;
  tab.coef = coef;
  tab.first = first;
  tab.base.scales = nullptr;
  int ids[kPrepGroups];
  auto prologue = [&]() {
    hipLaunchKernelGGL(adamw_prologue_kernel, dim3(1), dim3(tab.norm && tab.finalize ? kPrepThreads : 128), 0, stream, tab);
    tab.row0 += tab.n;
    tab.n = tab.n_groups = tab.finalize = 0;
  };
  // tensors in the order of their kind (moments in 32 or 8 bits, then type): one update launch for each kind that occurs
  struct { int n; long groups; } kinds[6];
  for (int kind = 0; kind < 6; ++kind) {
    kinds[kind].n = 0;
    kinds[kind].groups = 0;
    for (int i = 0; i < n; ++i) {
      if (dtypes[i] + (scales && scales[i] ? 3 : 0) != kind) continue;
      const OptRow row = {params[i], grads[i], exp_avgs[i], exp_avg_sqs[i], kind >= 3 ? scales[i] : nullptr, numels[i]};
      int j = 0;
      while (j < tab.n_groups && ids[j] != groups[i]) ++j;
      PrepRow r;
      if (!tab.base.scales) tab.base.scales = row.scales;
      if (tab.n == kPrepRows || j == kPrepGroups || (tab.n > 0 && !relative(row, steps[i], tab, r))) {
        prologue();
        j = 0;
      }
      if (tab.n == 0) {
        tab.base = row;
        tab.step_base = steps[i];
        relative(row, steps[i], tab, r);
      }
      if (j == tab.n_groups) {
        ids[tab.n_groups++] = groups[i];
        tab.g[j] = prologue_group(group[groups[i]]);
      }
      r.numel = (unsigned)numels[i];
      r.first = (unsigned)kinds[kind].groups | (unsigned)j << 24 | (unsigned)(numels[i] >> 32) << 27;
      tab.row[tab.n++] = r;
      kinds[kind].groups += ceil_div(numels[i], kind >= 3 ? kOptChunk8 : kOptChunk);
      ++kinds[kind].n;
    }
  }
  if (tab.n > 0 || tab.finalize) prologue();
  int row = 0;
  for (int kind = 0; kind < 6; ++kind) {
    const UpdateArgs args = {rows + row, coef + row, first + row, kinds[kind].n};
    if (kinds[kind].groups > 0 && bytes > kCacheBytes) launch_update<true>(kind, args, kinds[kind].groups, stream);
    else if (kinds[kind].groups > 0) launch_update<false>(kind, args, kinds[kind].groups, stream);
    row += kinds[kind].n;
  }
  return pir_check_launch();
}

size_t pir_grad_norm_workspace_bytes(int n, const long* numels) {
  if (n < 0 || (n > 0 && !numels)) return 0;
  return 8 * (size_t)norm_partials(n, numels) + 8;
}

int pir_grad_norm(int n, const void* const* grads, const long* numels, const int* dtypes, float* total, float* each,
                  void* workspace, size_t workspace_bytes, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  const int rc = check_tensors(n, numels, dtypes, grads, nullptr);
  if (rc != PIR_OK) return rc;
  if (!total || (((size_t)total | (size_t)each) & 3)) return PIR_ERR_ARG;
  if (!workspace || ((size_t)workspace & 7) || workspace_bytes < pir_grad_norm_workspace_bytes(n, numels)) return PIR_ERR_SCRATCH;
  const long n_partial = norm_partials(n, numels);
  double* partial = (double*)workspace;
  if (launch_partials(n, grads, numels, dtypes, partial, stream) != PIR_OK) return PIR_ERR_LAUNCH;
  const unsigned chunk = norm_chunk(n, numels);
  FinishTable tab;
  tab.n_partial = (int)n_partial;
  tab.partial = partial;
  tab.total = total;
  long at = 0;
  int i = 0;
  do {
    tab.n = 0;
    tab.each = each ? each + i : nullptr;
    tab.first[0] = (unsigned)at;
    for (; each && i < n && tab.n < kFirstTable; ++i) {
      at += ceil_div(numels[i], chunk);
      tab.first[++tab.n] = (unsigned)at;
    }
    const unsigned waves = (unsigned)ceil_div(tab.n, kFinishWaves);
    hipLaunchKernelGGL(norm_finish_kernel, dim3((tab.total ? 1 : 0) + waves), dim3(kPrepThreads), 0, stream, tab);
    tab.total = nullptr;
  } while (each && i < n);
  return pir_check_launch();
}

int pir_moments8_decode(long n_blocks, const signed char* exp_avg, const unsigned char* exp_avg_sq, const float* scales,
                        int dtype, void* m, void* v, void* stream) {
  if (n_blocks < 0 || dtype < PIR_F32 || dtype > PIR_F16) return PIR_ERR_ARG;
  if (n_blocks > kMaxGroups * (kOptChunk8 / kOptBlock)) return PIR_ERR_TOO_LARGE;
  if (n_blocks == 0) return PIR_OK;
  if (!exp_avg || !exp_avg_sq || !scales || !m || !v || ((((size_t)exp_avg | (size_t)exp_avg_sq) & 15) || ((size_t)scales & 7)) ||
      (((size_t)m | (size_t)v) & (element_bytes(dtype) - 1)))
    return PIR_ERR_ARG;
  const dim3 grid((unsigned)ceil_div(n_blocks * kOptBlock, kOptChunk8)), block(kOptThreads);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PIR_F32)
    hipLaunchKernelGGL(moments8_decode_kernel<float>, grid, block, 0, s, n_blocks, exp_avg, exp_avg_sq, scales, (float*)m, (float*)v);
  else if (dtype == PIR_BF16)
    hipLaunchKernelGGL(moments8_decode_kernel<__bf16>, grid, block, 0, s, n_blocks, exp_avg, exp_avg_sq, scales, (__bf16*)m, (__bf16*)v);
  else
    hipLaunchKernelGGL(moments8_decode_kernel<_Float16>, grid, block, 0, s, n_blocks, exp_avg, exp_avg_sq, scales, (_Float16*)m, (_Float16*)v);
  return pir_check_launch();
}

int pir_moments8_encode(long numel, int dtype, const void* m, const void* v, signed char* exp_avg,
                        unsigned char* exp_avg_sq, float* scales, void* stream) {
  if (numel < 0 || dtype < PIR_F32 || dtype > PIR_F16) return PIR_ERR_ARG;
  if (numel > kMaxGroups * kOptChunk8) return PIR_ERR_TOO_LARGE;
  if (numel == 0) return PIR_OK;
  if (!exp_avg || !exp_avg_sq || !scales || !m || !v || ((((size_t)exp_avg | (size_t)exp_avg_sq) & 15) || ((size_t)scales & 7)) ||
      (((size_t)m | (size_t)v) & (element_bytes(dtype) - 1)))
    return PIR_ERR_ARG;
  const dim3 grid((unsigned)ceil_div(numel, kOptChunk8)), block(kOptThreads);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PIR_F32)
    hipLaunchKernelGGL(moments8_encode_kernel<float>, grid, block, 0, s, numel, (const float*)m, (const float*)v, exp_avg, exp_avg_sq, scales);
  else if (dtype == PIR_BF16)
    hipLaunchKernelGGL(moments8_encode_kernel<__bf16>, grid, block, 0, s, numel, (const __bf16*)m, (const __bf16*)v, exp_avg, exp_avg_sq, scales);
  else
    hipLaunchKernelGGL(moments8_encode_kernel<_Float16>, grid, block, 0, s, numel, (const _Float16*)m, (const _Float16*)v, exp_avg, exp_avg_sq, scales);
  return pir_check_launch();
}

}  // extern "C"
