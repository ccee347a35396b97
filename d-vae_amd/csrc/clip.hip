// Global norm of many gradient tensors, and the gradients scaled down to a largest norm:
//   norm = sqrt(sum over all tensors of g^2);  coef = min(1, max_norm / (norm + 1e-6));  out = coef g
// Two streaming passes and a tiny launch between them that adds the partial sums in a fixed order (the same bits every
// time) and leaves {norm, coef} on the device: nothing waits on the host.  Squares are formed and added in double: fp32
// gradients of 1e-30 or 1e30 neither vanish nor overflow, and no order of summation shows in the fp32 result.
// Tensors are described in the kernel's arguments (no table in device memory to keep or upload): a launch covers up to
// CLIP_BATCH of them, cut into chunks of CHUNK elements.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "common.h"

namespace {

constexpr int CLIP_BATCH = 96;          // 96 descriptors of 32 bytes and their chunk starts: under the 4 KB of arguments
constexpr int CHUNK = 8192;             // elements of a workgroup's step: 256 threads x 4 loads of 8
constexpr int MAX_GRID = 2048;

struct Batch {
  const void* in[CLIP_BATCH];
  void* out[CLIP_BATCH];
  long long n[CLIP_BATCH];
  int start[CLIP_BATCH + 1];            // first chunk of each tensor
  unsigned char in_type[CLIP_BATCH], out_type[CLIP_BATCH];
  int count;
};
static_assert(sizeof(Batch) <= 3584, "kernel arguments");

typedef uint32_t u32x4_u2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float load1(const void* p, int type, long long i) {
  if (type == DVAE_F32) return static_cast<const float*>(p)[i];
  if (type == DVAE_BF16) return __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
  return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void store1(void* p, int type, long long i, float v) {
  if (type == DVAE_F32) static_cast<float*>(p)[i] = v;
  else if (type == DVAE_BF16) static_cast<__bf16*>(p)[i] = (__bf16)v;
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

// tensor of a chunk (uniform over the workgroup)
__device__ __forceinline__ int tensor_of(const Batch& b, int chunk) {
  int lo = 0, hi = b.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (b.start[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ __launch_bounds__(256) void norm_kernel(Batch b, double* __restrict__ part) {
  __shared__ double sh[4];
  double s = 0.0;
  const int chunks = b.start[b.count];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = tensor_of(b, c);
    const long long base = (long long)(c - b.start[t]) * CHUNK;
    const long long end = min(base + CHUNK, b.n[t]);
    for (long long i = base + threadIdx.x; i < end; i += 256) {
      const double v = load1(b.in[t], b.in_type[t], i);
      s = fma(v, v, s);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

__global__ __launch_bounds__(256) void norm_join_kernel(const double* __restrict__ part, int n, double max_norm,
                                                        float* __restrict__ out2) {
  __shared__ double sh[4];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) s += part[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  const double norm = sqrt((sh[0] + sh[1]) + (sh[2] + sh[3]));
  const double coef = max_norm / (norm + 1e-6);
  out2[0] = (float)norm;
  out2[1] = coef > 1.0 ? 1.f : (float)coef;       // a NaN norm stays NaN
}

__global__ __launch_bounds__(256) void scale_kernel(Batch b, const float* __restrict__ out2) {
  const float k = out2[1];
  const int chunks = b.start[b.count];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = tensor_of(b, c);
    if (k == 1.f && b.in[t] == b.out[t]) continue;              // in place, nothing to clip
    const long long base = (long long)(c - b.start[t]) * CHUNK;
    const long long end = min(base + CHUNK, b.n[t]);
    for (long long i = base + threadIdx.x; i < end; i += 256)
      store1(b.out[t], b.out_type[t], i, load1(b.in[t], b.in_type[t], i) * k);
  }
}

int type_bytes(int t) { return t == DVAE_F32 ? 4 : 2; }

struct Span { uintptr_t lo, hi; int tensor; bool write; };

// no output may overlap another tensor; an input may be its own output
int check_tensors(const dvae_tensor* t, int n, bool write, const char* who) {
  DVAE_REQUIRE(n >= 0 && (t || n == 0), "%s: null pointer", who);
  for (int i = 0; i < n; ++i) {
    DVAE_REQUIRE(t[i].n >= 0, "%s: tensor %d has %lld elements", who, i, t[i].n);
    DVAE_REQUIRE(t[i].in_type >= DVAE_F32 && t[i].in_type <= DVAE_F16, "%s: tensor %d has type %d", who, i, t[i].in_type);
    DVAE_REQUIRE(t[i].in || t[i].n == 0, "%s: tensor %d is null", who, i);
    DVAE_REQUIRE((uintptr_t)t[i].in % type_bytes(t[i].in_type) == 0, "%s: tensor %d is not aligned to its type", who, i);
    if (!write) continue;
    DVAE_REQUIRE(t[i].out_type >= DVAE_F32 && t[i].out_type <= DVAE_F16, "%s: output %d has type %d", who, i, t[i].out_type);
    DVAE_REQUIRE(t[i].out || t[i].n == 0, "%s: output %d is null", who, i);
    DVAE_REQUIRE((uintptr_t)t[i].out % type_bytes(t[i].out_type) == 0, "%s: output %d is not aligned to its type", who, i);
    DVAE_REQUIRE(t[i].n == 0 || t[i].in != t[i].out || t[i].in_type == t[i].out_type, "%s: tensor %d is its own output in another type", who, i);
  }
  if (!write) return DVAE_OK;
  try {
    std::vector<Span> v;
    v.reserve((size_t)n * 2);
    for (int i = 0; i < n; ++i) {
      if (t[i].n == 0) continue;
      const uintptr_t o = (uintptr_t)t[i].out, p = (uintptr_t)t[i].in;
      v.push_back({o, o + (uintptr_t)t[i].n * type_bytes(t[i].out_type), i, true});
      if (p != o) v.push_back({p, p + (uintptr_t)t[i].n * type_bytes(t[i].in_type), i, false});
    }
    std::sort(v.begin(), v.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
    // the farthest end seen so far, of any span and of the written ones
    uintptr_t any = 0, written = 0;
    for (const Span& s : v) {
      if (s.lo < (s.write ? any : written)) {
        dvae_set_error("%s: tensor %d overlaps another one that is written", who, s.tensor);
        return DVAE_ERR_ARG;
      }
      any = std::max(any, s.hi);
      if (s.write) written = std::max(written, s.hi);
    }
  } catch (const std::bad_alloc&) {
    dvae_set_error("%s: out of host memory", who);
    return DVAE_ERR_ARG;
  }
  return DVAE_OK;
}

// calls f(batch, grid) for batches of tensors in order; grid: the batch's workgroups
template <typename F>
int for_batches(const dvae_tensor* t, int n, F f) {
  int i = 0;
  while (i < n) {
    Batch b;
    b.count = 0;
    long long chunks = 0;
    while (i < n && b.count < CLIP_BATCH) {
      const long long c = (t[i].n + CHUNK - 1) / CHUNK;
      if (chunks + c > INT32_MAX / 2) {
        if (b.count) break;
        dvae_set_error("clip: tensor of %lld elements is too large", t[i].n);
        return DVAE_ERR_ARG;
      }
      if (c) {
        b.in[b.count] = t[i].in; b.out[b.count] = t[i].out; b.n[b.count] = t[i].n;
        b.in_type[b.count] = (unsigned char)t[i].in_type; b.out_type[b.count] = (unsigned char)t[i].out_type;
        b.start[b.count] = (int)chunks;
        ++b.count;
        chunks += c;
      }
      ++i;
    }
    if (!b.count) continue;
    b.start[b.count] = (int)chunks;
    DVAE_TRY(f(b, (int)std::min<long long>(chunks, MAX_GRID)));
  }
  return DVAE_OK;
}

}  // namespace

extern "C" size_t dvae_clip_ws_bytes(int n) {
  return n < 0 ? 0 : ((size_t)n / CLIP_BATCH + 1) * 2 * MAX_GRID * sizeof(double);
}

extern "C" int dvae_grad_norm(const dvae_tensor* tensors, int n, double max_norm, float* norm_coef, void* ws, void* stream) {
  DVAE_TRY(check_tensors(tensors, n, false, "grad_norm"));
  DVAE_REQUIRE(norm_coef && ws, "grad_norm: null pointer");
  DVAE_REQUIRE(max_norm >= 0.0, "grad_norm: max_norm must not be negative");
  hipStream_t st = (hipStream_t)stream;
  double* part = (double*)ws;
  const size_t room = dvae_clip_ws_bytes(n) / sizeof(double);
  size_t used = 0;
  DVAE_TRY(for_batches(tensors, n, [&](const Batch& b, int grid) -> int {
    DVAE_REQUIRE(used + grid <= room, "grad_norm: too many batches");
    hipLaunchKernelGGL(norm_kernel, dim3(grid), dim3(256), 0, st, b, part + used);
    DVAE_LAUNCH_CHECK();
    used += grid;
    return DVAE_OK;
  }));
  hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(256), 0, st, part, (int)used, max_norm, norm_coef);
  DVAE_LAUNCH_CHECK();
  return DVAE_OK;
}

extern "C" int dvae_clip_grads(const dvae_tensor* tensors, int n, double max_norm, float* norm_coef, void* ws, void* stream) {
  DVAE_TRY(check_tensors(tensors, n, true, "clip_grads"));
  DVAE_TRY(dvae_grad_norm(tensors, n, max_norm, norm_coef, ws, stream));
  return for_batches(tensors, n, [&](const Batch& b, int grid) -> int {
    hipLaunchKernelGGL(scale_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, b, norm_coef);
    DVAE_LAUNCH_CHECK();
    return DVAE_OK;
  });
}
