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
constexpr int kOptTable = 64;                 // tensors per launch: their descriptors travel as kernel arguments
constexpr int kOptBlock = 256;                // elements that share a scale
constexpr long kOptChunk = 4096;              // elements one workgroup updates
constexpr long kNormChunk = 16384;            // elements one workgroup sums
constexpr int kPrepThreads = 1024;
constexpr int kPrepTensors = 192;             // step counters per prologue launch
constexpr int kPrepGroups = 16;               // hyper-parameter sets per prologue launch

// what one tensor's update needs, computed once per step by the prologue
struct OptCoef {
  float b1, c1, b2, c2;                       // beta, 1 - beta
  float size, root, eps, decay;               // lr / (1 - beta1^t), (1 - beta2^t)^-1/2, eps, lr weight_decay
  float gscale, run, pad0, pad1;              // clip factor; run = 0: leave the tensor as it is
};

struct OptTensor {
  void* param;
  const void* grad;
  void* m;
  void* v;
  float* scales;
  long numel;
};

struct OptTable {
  int n;
  const OptCoef* coef;                        // of tensor i: coef[index[i]]
  OptTensor t[kOptTable];
  int index[kOptTable];
  int first[kOptTable + 1];                   // first workgroup of each tensor
};

struct NormTable {
  int n;
  double* partial;
  const void* grad[kOptTable];
  long numel[kOptTable];
  int dtype[kOptTable];
  int first[kOptTable + 1];
};

struct PrepGroup {
  double lr, log1, log2, c1, c2, wd;
  const float* lr_device;
  float b1, b2, eps;
};

struct PrepTable {
  int n, n_partial, finalize, clip, skip;
  double max_norm;
  const double* partial;
  float* norm;                                // [total, clip factor]
  OptCoef* coef;
  float* total;                               // the caller's copy of the norm, or NULL
  float* step[kPrepTensors];
  unsigned char group[kPrepTensors];
  PrepGroup g[kPrepGroups];
};

static_assert(sizeof(OptTable) <= 4096 && sizeof(NormTable) <= 4096 && sizeof(PrepTable) <= 4096, "kernel arguments");

template <typename T> __device__ inline float to_float(T x) { return (float)x; }
template <typename T> __device__ inline T from_float(float x) { return (T)x; }   // round to nearest even

__device__ inline int find_tensor(const int* first, int n, int block) {
  int lo = 0, hi = n;                         // first[lo] <= block < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= block) lo = mid; else hi = mid;
  }
  return lo;
}

struct Updated { float p, m, v; };

__device__ inline Updated adamw_element(const OptCoef& c, float p, float g, float m, float v) {
  g *= c.gscale;
  Updated r;
  r.m = fmaf(c.b1, m, c.c1 * g);
  r.v = fmaf(c.b2, v, c.c2 * g * g);
  const float u = r.m / fmaf(sqrtf(r.v), c.root, c.eps);
  r.p = p - fmaf(c.decay, p, c.size * u);
  return r;
}

template <typename T>
__global__ void __launch_bounds__(kOptThreads)
adamw32_kernel(const OptTable tab) {
  const int k = find_tensor(tab.first, tab.n, blockIdx.x);
  const OptCoef c = tab.coef[tab.index[k]];
  if (c.run == 0.0f) return;
  const OptTensor t = tab.t[k];
  const long base = (long)(blockIdx.x - tab.first[k]) * kOptChunk;
  const long end = base + kOptChunk < t.numel ? base + kOptChunk : t.numel;
  T* __restrict__ P = (T*)t.param;
  const T* __restrict__ G = (const T*)t.grad;
  float* __restrict__ M = (float*)t.m;
  float* __restrict__ V = (float*)t.v;
  for (long i = base + threadIdx.x; i < end; i += kOptThreads) {
    const Updated r = adamw_element(c, to_float(P[i]), to_float(G[i]), M[i], V[i]);
    P[i] = from_float<T>(r.p);
    M[i] = r.m;
    V[i] = r.v;
  }
}

__device__ inline unsigned wave_max(unsigned x) {
  for (int d = 32; d >= 1; d >>= 1) {
    const unsigned y = __shfl_xor(x, d);
    x = x > y ? x : y;
  }
  return x;
}

// The scale of a block from the largest bit pattern of its magnitudes: integers order like the floats they stand for,
// with infinities and NaN on top.  Below 2^-126 the block is zero; a value that is not finite makes the scale NaN.
__device__ inline float block_scale(unsigned top) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return top < 0x00800000u ? 0.0f : __uint_as_float(top);
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

// one wave per block of 256 elements, 4 consecutive ones per lane
template <typename T>
__global__ void __launch_bounds__(kOptThreads)
adamw8_kernel(const OptTable tab) {
  const int k = find_tensor(tab.first, tab.n, blockIdx.x);
  const OptCoef c = tab.coef[tab.index[k]];
  if (c.run == 0.0f) return;
  const OptTensor t = tab.t[k];
  const long base = (long)(blockIdx.x - tab.first[k]) * kOptChunk;
  const long end = base + kOptChunk < t.numel ? base + kOptChunk : t.numel;
  const int lane = threadIdx.x & 63;
  T* __restrict__ P = (T*)t.param;
  const T* __restrict__ G = (const T*)t.grad;
  for (long b0 = base + (threadIdx.x >> 6) * kOptBlock; b0 < end; b0 += 4 * kOptBlock) {
    const long i0 = b0 + 4 * lane, blk = b0 / kOptBlock;
    char4* mq = (char4*)((signed char*)t.m + i0);
    uchar4* vq = (uchar4*)((unsigned char*)t.v + i0);
    const float a = t.scales[2 * blk], b = t.scales[2 * blk + 1];
    const char4 q = *mq;
    const uchar4 w = *vq;
    const int qs[4] = {q.x, q.y, q.z, q.w}, ws[4] = {w.x, w.y, w.z, w.w};
    float m[4], v[4];
    unsigned ma = 0, mb = 0;
    for (int j = 0; j < 4; ++j) {
      m[j] = v[j] = 0.0f;                     // what fills up the last block stays zero
      if (i0 + j >= t.numel) continue;
      const Updated r = adamw_element(c, to_float(P[i0 + j]), to_float(G[i0 + j]), decode_m(qs[j], a), decode_v(ws[j], b));
      P[i0 + j] = from_float<T>(r.p);
      m[j] = r.m;
      v[j] = r.v;
      const unsigned x = __float_as_uint(r.m) & 0x7fffffffu, y = __float_as_uint(r.v) & 0x7fffffffu;
      ma = ma > x ? ma : x;
      mb = mb > y ? mb : y;
    }
    const float na = block_scale(wave_max(ma)), nb = block_scale(wave_max(mb));
    *mq = make_char4(encode_m(m[0], na), encode_m(m[1], na), encode_m(m[2], na), encode_m(m[3], na));
    *vq = make_uchar4(encode_v(v[0], nb), encode_v(v[1], nb), encode_v(v[2], nb), encode_v(v[3], nb));
    if (lane == 0) {
      t.scales[2 * blk] = na;
      t.scales[2 * blk + 1] = nb;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kOptThreads)
moments8_decode_kernel(long n_blocks, const signed char* __restrict__ mq, const unsigned char* __restrict__ vq,
                       const float* __restrict__ scales, T* __restrict__ m, T* __restrict__ v) {
  const int lane = threadIdx.x & 63;
  for (long blk = (long)blockIdx.x * 4 + (threadIdx.x >> 6); blk < n_blocks; blk += (long)gridDim.x * 4) {
    const long i0 = blk * kOptBlock + 4 * lane;
    const float a = scales[2 * blk], b = scales[2 * blk + 1];
    for (int j = 0; j < 4; ++j) {
      m[i0 + j] = from_float<T>(decode_m(mq[i0 + j], a));
      v[i0 + j] = from_float<T>(decode_v(vq[i0 + j], b));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kOptThreads)
moments8_encode_kernel(long n_blocks, long numel, const T* __restrict__ m, const T* __restrict__ v,
                       signed char* __restrict__ mq, unsigned char* __restrict__ vq, float* __restrict__ scales) {
  const int lane = threadIdx.x & 63;
  for (long blk = (long)blockIdx.x * 4 + (threadIdx.x >> 6); blk < n_blocks; blk += (long)gridDim.x * 4) {
    const long i0 = blk * kOptBlock + 4 * lane;
    float x[4], y[4];
    unsigned ma = 0, mb = 0;
    for (int j = 0; j < 4; ++j) {
      x[j] = i0 + j < numel ? to_float(m[i0 + j]) : 0.0f;
      y[j] = i0 + j < numel ? to_float(v[i0 + j]) : 0.0f;
      const unsigned p = __float_as_uint(x[j]) & 0x7fffffffu, q = __float_as_uint(y[j]) & 0x7fffffffu;
      ma = ma > p ? ma : p;
      mb = mb > q ? mb : q;
    }
    const float a = block_scale(wave_max(ma)), b = block_scale(wave_max(mb));
    for (int j = 0; j < 4; ++j) {
      mq[i0 + j] = (signed char)encode_m(x[j], a);
      vq[i0 + j] = (unsigned char)encode_v(y[j], b);
    }
    if (lane == 0) {
      scales[2 * blk] = a;
      scales[2 * blk + 1] = b;
    }
  }
}

// ---- norms: squares and sums in 64 bits (no overflow for any fp32 gradient), one partial sum per workgroup, added up
// in a fixed order: the same bits on every run

__device__ inline double wave_sum(double x) {
  for (int d = 32; d >= 1; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

template <typename T>
__device__ inline double sum_squares(const T* __restrict__ g, long i, long end) {
  double s = 0.0;
  for (; i < end; i += kOptThreads) {
    const double x = (double)to_float(g[i]);
    s = fma(x, x, s);
  }
  return s;
}

__global__ void __launch_bounds__(kOptThreads)
norm_partial_kernel(const NormTable tab) {
  __shared__ double part[kOptThreads / 64];
  const int k = find_tensor(tab.first, tab.n, blockIdx.x);
  const long base = (long)(blockIdx.x - tab.first[k]) * kNormChunk, numel = tab.numel[k];
  const long end = base + kNormChunk < numel ? base + kNormChunk : numel;
  const long i = base + threadIdx.x;
  double s;
  if (tab.dtype[k] == PIR_F32) s = sum_squares((const float*)tab.grad[k], i, end);
  else if (tab.dtype[k] == PIR_BF16) s = sum_squares((const __bf16*)tab.grad[k], i, end);
  else s = sum_squares((const _Float16*)tab.grad[k], i, end);
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) tab.partial[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

__device__ inline double block_sum(double s, double* part) {
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  double all = 0.0;
  for (int i = 0; i < kPrepThreads / 64; ++i) all += part[i];
  __syncthreads();
  return all;
}

// one workgroup: the joint norm and clip factor from the partial sums, then every tensor's step count and coefficients
__global__ void __launch_bounds__(kPrepThreads)
adamw_prologue_kernel(const PrepTable tab) {
  __shared__ double part[kPrepThreads / 64];
  float norm = 0.0f, clip = 1.0f;
  if (tab.norm) {
    if (tab.finalize) {
      double s = 0.0;
      for (int i = threadIdx.x; i < tab.n_partial; i += kPrepThreads) s += tab.partial[i];
      const double all = sqrt(block_sum(s, part));
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
  for (int i = threadIdx.x; i < tab.n; i += kPrepThreads) {
    const PrepGroup& g = tab.g[tab.group[i]];
    const float t = *tab.step[i] + 1.0f;
    const double lr = g.lr_device ? (double)*g.lr_device : g.lr;
    OptCoef c;
    c.b1 = g.b1;
    c.c1 = (float)g.c1;
    c.b2 = g.b2;
    c.c2 = (float)g.c2;
    c.size = (float)(lr / -expm1((double)t * g.log1));
    c.root = (float)(1.0 / sqrt(-expm1((double)t * g.log2)));
    c.eps = g.eps;
    c.decay = (float)(lr * g.wd);
    c.gscale = clip;
    c.run = run ? 1.0f : 0.0f;
    c.pad0 = c.pad1 = 0.0f;
    tab.coef[i] = c;
    if (run) *tab.step[i] = t;
  }
}

// one workgroup: per-tensor norms from the partial sums of each, and the joint one
__global__ void __launch_bounds__(kPrepThreads)
norm_finish_kernel(int n, const int* __restrict__ first, int n_partial, const double* __restrict__ partial,
                   float* __restrict__ total, float* __restrict__ each) {
  __shared__ double part[kPrepThreads / 64];
  double s = 0.0;
  for (int i = threadIdx.x; i < n_partial; i += kPrepThreads) s += partial[i];
  const double all = block_sum(s, part);
  if (threadIdx.x == 0) *total = (float)sqrt(all);
  if (each == nullptr) return;
  for (int k = threadIdx.x >> 6; k < n; k += kPrepThreads / 64) {
    double x = 0.0;
    for (int i = first[k] + (threadIdx.x & 63); i < first[k + 1]; i += 64) x += partial[i];
    x = wave_sum(x);
    if ((threadIdx.x & 63) == 0) each[k] = (float)sqrt(x);
  }
}

// the prefix table of norm_finish_kernel: 256 entries at a time as kernel arguments
struct IntTable { int n; int v[512]; };
__global__ void write_ints_kernel(const IntTable tab, int* out) {
  for (int i = threadIdx.x; i < tab.n; i += blockDim.x) out[i] = tab.v[i];
}

static inline long ceil_div(long a, long b) { return (a + b - 1) / b; }

static const long kMaxGroups = (1L << 24) - 1;     // workgroups of 256 threads: a grid has fewer than 2^32 threads

static int check_tensors(int n, const long* numels, const int* dtypes, const void* const* grads) {
  if (n < 0 || (n > 0 && (!numels || !dtypes || !grads))) return PIR_ERR_ARG;
  for (int i = 0; i < n; ++i) {
    if (numels[i] < 0 || dtypes[i] < PIR_F32 || dtypes[i] > PIR_F16) return PIR_ERR_ARG;
    if (numels[i] > 0 && !grads[i]) return PIR_ERR_ARG;
    if (ceil_div(numels[i], kOptChunk) > kMaxGroups) return PIR_ERR_TOO_LARGE;
  }
  return PIR_OK;
}

static long norm_partials(int n, const long* numels) {
  long c = 0;
  for (int i = 0; i < n; ++i) c += ceil_div(numels[i], kNormChunk);
  return c;
}

static int launch_partials(int n, const void* const* grads, const long* numels, const int* dtypes, double* partial,
                           hipStream_t stream) {
  NormTable tab;
  tab.n = 0;
  tab.first[0] = 0;
  tab.partial = partial;
  for (int i = 0; i <= n; ++i) {
    const long blocks = i < n ? ceil_div(numels[i], kNormChunk) : 0;
    if (tab.n > 0 && (i == n || tab.n == kOptTable || tab.first[tab.n] + blocks > kMaxGroups)) {
      hipLaunchKernelGGL(norm_partial_kernel, dim3(tab.first[tab.n]), dim3(kOptThreads), 0, stream, tab);
      tab.partial += tab.first[tab.n];
      tab.n = 0;
    }
    if (blocks == 0) continue;
    tab.grad[tab.n] = grads[i];
    tab.numel[tab.n] = numels[i];
    tab.dtype[tab.n] = dtypes[i];
    tab.first[tab.n + 1] = tab.first[tab.n] + (int)blocks;
    ++tab.n;
  }
  return pir_check_launch();
}

template <int kBits>
static void launch_update(int dtype, const OptTable& tab, hipStream_t stream) {
  const dim3 grid(tab.first[tab.n]), block(kOptThreads);
  if (kBits == 32) {
    if (dtype == PIR_F32) hipLaunchKernelGGL(adamw32_kernel<float>, grid, block, 0, stream, tab);
    else if (dtype == PIR_BF16) hipLaunchKernelGGL(adamw32_kernel<__bf16>, grid, block, 0, stream, tab);
    else hipLaunchKernelGGL(adamw32_kernel<_Float16>, grid, block, 0, stream, tab);
  } else {
    if (dtype == PIR_F32) hipLaunchKernelGGL(adamw8_kernel<float>, grid, block, 0, stream, tab);
    else if (dtype == PIR_BF16) hipLaunchKernelGGL(adamw8_kernel<__bf16>, grid, block, 0, stream, tab);
    else hipLaunchKernelGGL(adamw8_kernel<_Float16>, grid, block, 0, stream, tab);
  }
}

}  // namespace pir

using namespace pir;

extern "C" {

size_t pir_adamw_workspace_bytes(int n, const long* numels, int with_norm) {
  if (n < 0 || (n > 0 && !numels)) return 0;
  return 16 + (size_t)n * sizeof(OptCoef) + (with_norm ? 8 * (size_t)norm_partials(n, numels) : 0);
}

int pir_adamw_step(int n, void* const* params, const void* const* grads, void* const* exp_avgs, void* const* exp_avg_sqs,
                   float* const* scales, float* const* steps, const long* numels, const int* dtypes, const int* groups,
                   const PirAdamwGroup* group, int n_groups, double max_norm, int skip_nonfinite, float* total_norm,
                   void* workspace, size_t workspace_bytes, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  const int rc = check_tensors(n, numels, dtypes, grads);
  if (rc != PIR_OK) return rc;
  if (n > 0 && (!params || !exp_avgs || !exp_avg_sqs || !steps || !groups || !group || n_groups < 1)) return PIR_ERR_ARG;
  for (int k = 0; k < n_groups && n > 0; ++k) {
    const PirAdamwGroup& g = group[k];
    if (!(g.beta1 >= 0 && g.beta1 < 1 && g.beta2 >= 0 && g.beta2 < 1 && g.eps >= 0 && g.lr >= 0 && g.weight_decay >= 0))
      return PIR_ERR_ARG;
  }
  for (int i = 0; i < n; ++i) {
    if (!steps[i] || groups[i] < 0 || groups[i] >= n_groups) return PIR_ERR_ARG;
    if (numels[i] > 0 && (!params[i] || !exp_avgs[i] || !exp_avg_sqs[i])) return PIR_ERR_ARG;
    if (scales && scales[i] && ((((size_t)exp_avgs[i] | (size_t)exp_avg_sqs[i]) & 15) || ((size_t)scales[i] & 7)))
      return PIR_ERR_ARG;
  }
  const int clip = max_norm > 0.0 ? 1 : 0, with_norm = clip || skip_nonfinite || total_norm;
  if (n == 0 && !total_norm) return PIR_OK;
  if (!workspace || workspace_bytes < pir_adamw_workspace_bytes(n, numels, with_norm)) return PIR_ERR_SCRATCH;
  float* norm = (float*)workspace;                                    // [total, clip factor, -, -]
  OptCoef* coef = (OptCoef*)((char*)workspace + 16);
  double* partial = (double*)(coef + n);
  long n_partial = 0;
  if (with_norm) {
    n_partial = norm_partials(n, numels);
    if (n_partial > 0x7fffffffL) return PIR_ERR_TOO_LARGE;
    if (launch_partials(n, grads, numels, dtypes, partial, stream) != PIR_OK) return PIR_ERR_LAUNCH;
  }
  for (int i0 = 0, first = 1; first || i0 < n; first = 0) {
    PrepTable tab;
    tab.n = 0;
    tab.n_partial = (int)n_partial;
    tab.finalize = first;
    tab.clip = clip;
    tab.skip = skip_nonfinite != 0;
    tab.max_norm = max_norm;
    tab.partial = partial;
    tab.norm = with_norm ? norm : nullptr;
    tab.total = total_norm;
    tab.coef = coef + i0;
    int ids[kPrepGroups], n_ids = 0;
    for (; i0 < n && tab.n < kPrepTensors; ++i0) {
      int j = 0;
      while (j < n_ids && ids[j] != groups[i0]) ++j;
      if (j == n_ids) {
        if (n_ids == kPrepGroups) break;
        const PirAdamwGroup& g = group[groups[i0]];
        PrepGroup& d = tab.g[n_ids];
        ids[n_ids++] = groups[i0];
        d.lr = g.lr;
        d.lr_device = g.lr_device;
        d.log1 = std::log(g.beta1);
        d.log2 = std::log(g.beta2);
        d.c1 = 1.0 - g.beta1;
        d.c2 = 1.0 - g.beta2;
        d.wd = g.weight_decay;
        d.b1 = (float)g.beta1;
        d.b2 = (float)g.beta2;
        d.eps = (float)g.eps;
      }
      tab.step[tab.n] = steps[i0];
      tab.group[tab.n++] = (unsigned char)j;
    }
    hipLaunchKernelGGL(adamw_prologue_kernel, dim3(1), dim3(kPrepThreads), 0, stream, tab);
  }
  for (int kind = 0; kind < 6; ++kind) {                              // (8-bit moments or not) x dtype
    const int bits8 = kind / 3, dtype = kind % 3;
    OptTable tab;
    tab.n = 0;
    tab.coef = coef;
    tab.first[0] = 0;
    for (int i = 0; i <= n; ++i) {
      const bool mine = i < n && dtypes[i] == dtype && (scales && scales[i] ? 1 : 0) == bits8;
      const long blocks = mine ? ceil_div(numels[i], kOptChunk) : 0;
      if (tab.n > 0 && (i == n || (mine && (tab.n == kOptTable || tab.first[tab.n] + blocks > kMaxGroups)))) {
        if (bits8) launch_update<8>(dtype, tab, stream); else launch_update<32>(dtype, tab, stream);
        tab.n = 0;
      }
      if (blocks == 0) continue;
      OptTensor& t = tab.t[tab.n];
      t.param = params[i];
      t.grad = grads[i];
      t.m = exp_avgs[i];
      t.v = exp_avg_sqs[i];
      t.scales = bits8 ? scales[i] : nullptr;
      t.numel = numels[i];
      tab.index[tab.n] = i;
      tab.first[tab.n + 1] = tab.first[tab.n] + (int)blocks;
      ++tab.n;
    }
  }
  return pir_check_launch();
}

size_t pir_grad_norm_workspace_bytes(int n, const long* numels) {
  if (n < 0 || (n > 0 && !numels)) return 0;
  return 8 * (size_t)norm_partials(n, numels) + 4 * ((size_t)n + 1);
}

int pir_grad_norm(int n, const void* const* grads, const long* numels, const int* dtypes, float* total, float* each,
                  void* workspace, size_t workspace_bytes, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  const int rc = check_tensors(n, numels, dtypes, grads);
  if (rc != PIR_OK) return rc;
  if (!total) return PIR_ERR_ARG;
  if (!workspace || workspace_bytes < pir_grad_norm_workspace_bytes(n, numels)) return PIR_ERR_SCRATCH;
  const long n_partial = norm_partials(n, numels);
  if (n_partial > 0x7fffffffL) return PIR_ERR_TOO_LARGE;
  double* partial = (double*)workspace;
  int* first = (int*)(partial + n_partial);
  if (launch_partials(n, grads, numels, dtypes, partial, stream) != PIR_OK) return PIR_ERR_LAUNCH;
  if (each) {
    IntTable tab;
    long at = 0;
    tab.n = 0;
    int done = 0;
    for (int i = 0; i <= n; ++i) {
      tab.v[tab.n++] = (int)at;
      if (i < n) at += ceil_div(numels[i], kNormChunk);
      if (tab.n == 512 || i == n) {
        hipLaunchKernelGGL(write_ints_kernel, dim3(1), dim3(256), 0, stream, tab, first + done);
        done += tab.n;
        tab.n = 0;
      }
    }
  }
  hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(kPrepThreads), 0, stream, n, (const int*)first, (int)n_partial,
                     (const double*)partial, total, each);
  return pir_check_launch();
}

static unsigned moments8_grid(long n_blocks) {
  const long g = (n_blocks + 3) / 4, cap = 32L * pir_num_cus();
  return (unsigned)(g < cap ? g : cap);
}

int pir_moments8_decode(long n_blocks, const signed char* exp_avg, const unsigned char* exp_avg_sq, const float* scales,
                        int dtype, void* m, void* v, void* stream) {
  if (n_blocks < 0 || dtype < PIR_F32 || dtype > PIR_F16) return PIR_ERR_ARG;
  if (n_blocks == 0) return PIR_OK;
  if (!exp_avg || !exp_avg_sq || !scales || !m || !v) return PIR_ERR_ARG;
  const dim3 grid(moments8_grid(n_blocks)), block(kOptThreads);
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
  if (numel == 0) return PIR_OK;
  if (!exp_avg || !exp_avg_sq || !scales || !m || !v) return PIR_ERR_ARG;
  const long n_blocks = ceil_div(numel, kOptBlock);
  const dim3 grid(moments8_grid(n_blocks)), block(kOptThreads);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PIR_F32)
    hipLaunchKernelGGL(moments8_encode_kernel<float>, grid, block, 0, s, n_blocks, numel, (const float*)m, (const float*)v, exp_avg, exp_avg_sq, scales);
  else if (dtype == PIR_BF16)
    hipLaunchKernelGGL(moments8_encode_kernel<__bf16>, grid, block, 0, s, n_blocks, numel, (const __bf16*)m, (const __bf16*)v, exp_avg, exp_avg_sq, scales);
  else
    hipLaunchKernelGGL(moments8_encode_kernel<_Float16>, grid, block, 0, s, n_blocks, numel, (const _Float16*)m, (const _Float16*)v, exp_avg, exp_avg_sq, scales);
  return pir_check_launch();
}

}  // extern "C"
