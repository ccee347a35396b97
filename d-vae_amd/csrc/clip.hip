// Global norm of many gradient tensors, and the gradients scaled down to a largest norm:
//   norm = sqrt(sum over all tensors of g^2);  coef = min(1, max_norm / (norm + 1e-6));  out = coef g
// Two streaming passes; every workgroup of the second adds the first one's partial sums in the same fixed order (the same bits
// every time) and scales by the coefficient: nothing waits on the host.  Beyond one batch of tensors a launch of its own adds
// them, once for all batches.  Squares are formed and added in double: fp32 gradients of 1e-30 or 1e30 neither vanish nor
// overflow, and no order of summation shows in the fp32 result.
// Tensors are described in the kernel's arguments (no table in device memory to keep or upload): a launch covers up to
// CLIP_BATCH of them, cut into chunks of CHUNK elements, each loaded whole before its first value is used.
// Bound by memory: 400 M bf16 / fp32 gradients into fp32 191 + 524 us (4.2 and 4.6 TB/s; element by element it took 1285); the
// 40 tensors of a model with 6.9 M parameters 10 + 15 us, most of it the way to the memory and back.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "elem.h"

namespace {

constexpr int CLIP_BATCH = 96;          // 96 descriptors of 32 bytes and their chunk starts: under the 4 KB of arguments
// elements of a workgroup's step: 256 threads x 2 loads of 8, or 4 of 4.  Twice as many per step leave fewer workgroups: 13 + 17 us
// for a model's 28 MB instead of 10 + 15, and 212 + 524 for 2.4 GB instead of 194 + 535.
constexpr int CHUNK = 4096;
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

// The tensor of a chunk: every lane of a wave holds two chunk starts, the wave counts those at or before the chunk -- no
// search through memory between two chunks.
struct Lookup {
  int s0, s1;
  __device__ __forceinline__ explicit Lookup(const Batch& b) {
    const int lane = threadIdx.x & 63;
    s0 = lane < b.count ? b.start[lane] : INT32_MAX;
    s1 = lane + 64 < b.count ? b.start[lane + 64] : INT32_MAX;
  }
  __device__ __forceinline__ int operator()(int chunk) const {
    return __popcll(__ballot(s0 <= chunk)) + __popcll(__ballot(s1 <= chunk)) - 1;
  }
};
static_assert(CLIP_BATCH <= 128, "two chunk starts a lane");

// squares of one chunk, in four sums
template <int T>
__device__ __forceinline__ void norm_chunk(const void* in, long long base, int n, double (&s)[4]) {
  typedef Elem<T> E;
  constexpr int EV = E::EV, NV = CHUNK / (256 * EV);
  const typename E::type* p = static_cast<const typename E::type*>(in) + base;
  if (n == CHUNK) {
    u32x4 r[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) r[j] = *reinterpret_cast<const u32x4_u*>(p + (j * 256 + threadIdx.x) * EV);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const double v = E::at(r[j], e);
        s[e & 3] = fma(v, v, s[e & 3]);
      }
  } else {
    for (int i = threadIdx.x; i < n; i += 256) {
      const double v = E::one(p, i);
      s[0] = fma(v, v, s[0]);
    }
  }
}

__global__ __launch_bounds__(256) void norm_kernel(Batch b, double* __restrict__ part) {
  __shared__ double sh[4];
  double s4[4] = {0.0, 0.0, 0.0, 0.0};
  const int chunks = b.start[b.count];
  const Lookup tensor_of(b);
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = tensor_of(c);
    const long long base = (long long)(c - b.start[t]) * CHUNK;
    const int n = (int)min((long long)CHUNK, b.n[t] - base);
    if (b.in_type[t] == DVAE_F32) norm_chunk<DVAE_F32>(b.in[t], base, n, s4);
    else if (b.in_type[t] == DVAE_BF16) norm_chunk<DVAE_BF16>(b.in[t], base, n, s4);
    else norm_chunk<DVAE_F16>(b.in[t], base, n, s4);
  }
  double s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// {norm, coef} from the partial sums, the same in every workgroup that forms them
struct Sum { double norm, coef; };
__device__ __forceinline__ Sum join(const double* __restrict__ part, int n, double max_norm) {
  __shared__ double sh[4];
  double s = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 256) s += part[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  Sum r;
  r.norm = sqrt((sh[0] + sh[1]) + (sh[2] + sh[3]));
  const double coef = max_norm / (r.norm + 1e-6);
  r.coef = coef > 1.0 ? 1.0 : coef;               // a NaN norm stays NaN
  return r;
}

__global__ __launch_bounds__(256) void norm_join_kernel(const double* __restrict__ part, int n, double max_norm,
                                                        float* __restrict__ out2) {
  const Sum s = join(part, n, max_norm);
  if (threadIdx.x) return;
  out2[0] = (float)s.norm;
  out2[1] = (float)s.coef;
}

template <int TI, int TO>
__device__ __forceinline__ void scale_chunk(const void* in, void* out, long long base, int n, float k) {
  typedef Elem<TI> I;
  typedef Elem<TO> O;
  constexpr int EV = I::EV, NV = CHUNK / (256 * EV);
  const typename I::type* p = static_cast<const typename I::type*>(in) + base;
  typename O::type* q = static_cast<typename O::type*>(out) + base;
  if (n == CHUNK) {
    u32x4 r[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) r[j] = *reinterpret_cast<const u32x4_u*>(p + (j * 256 + threadIdx.x) * EV);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      typename O::type o[EV];
#pragma unroll
      for (int e = 0; e < EV; ++e) o[e] = O::cast(I::at(r[j], e) * k);
      typename O::type* w = q + (j * 256 + threadIdx.x) * EV;
      constexpr int BYTES = EV * (int)sizeof(o[0]);          // 8 (fp32 to half), 16 or 32 (half to fp32)
      if (BYTES == 8) {
        u32x2 v;
        __builtin_memcpy(&v, o, 8);
        *reinterpret_cast<u32x2_u*>(w) = v;
      } else {
#pragma unroll
        for (int h = 0; h < BYTES / 16; ++h) {
          u32x4 v;
          __builtin_memcpy(&v, reinterpret_cast<const char*>(o) + 16 * h, 16);
          *reinterpret_cast<u32x4_u*>(reinterpret_cast<char*>(w) + 16 * h) = v;
        }
      }
    }
  } else {
    for (int i = threadIdx.x; i < n; i += 256) q[i] = O::cast(I::one(p, i) * k);
  }
}

template <int TI>
__device__ __forceinline__ void scale_to(int out_type, const void* in, void* out, long long base, int n, float k) {
  if (out_type == DVAE_F32) scale_chunk<TI, DVAE_F32>(in, out, base, n, k);
  else if (out_type == DVAE_BF16) scale_chunk<TI, DVAE_BF16>(in, out, base, n, k);
  else scale_chunk<TI, DVAE_F16>(in, out, base, n, k);
}

// Chunks from the last to the first: the norm pass read the last ones last, so they are still in the 256 MB cache.  JOIN: every
// workgroup adds the partial sums, of one batch at most MAX_GRID (4 us less than a launch of their own), and the first writes
// norm and coefficient; else out2 holds them (with every batch's workgroups adding every batch's sums, work that grows with the
// square of the batches, 400 tensors of 400,000 fp32 took 470 us instead of 444).
template <bool JOIN>
__global__ __launch_bounds__(256) void scale_kernel(Batch b, const double* __restrict__ part, int n_part, double max_norm,
                                                    float* __restrict__ out2) {
  float k;
  if (JOIN) {
    const Sum sum = join(part, n_part, max_norm);
    k = (float)sum.coef;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      out2[0] = (float)sum.norm;
      out2[1] = k;
    }
  } else {
    k = out2[1];
  }
  const int chunks = b.start[b.count];
  const Lookup tensor_of(b);
  for (int c = chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const int t = tensor_of(c);
    if (k == 1.f && b.in[t] == b.out[t]) continue;              // in place, nothing to clip
    const long long base = (long long)(c - b.start[t]) * CHUNK;
    const int n = (int)min((long long)CHUNK, b.n[t] - base);
    if (b.in_type[t] == DVAE_F32) scale_to<DVAE_F32>(b.out_type[t], b.in[t], b.out[t], base, n, k);
    else if (b.in_type[t] == DVAE_BF16) scale_to<DVAE_BF16>(b.out_type[t], b.in[t], b.out[t], base, n, k);
    else scale_to<DVAE_F16>(b.out_type[t], b.in[t], b.out[t], base, n, k);
  }
}

struct Span { uintptr_t lo, hi; int tensor; bool write; };

// no output may overlap another tensor; an input may be its own output
int check_tensors(const dvae_tensor* t, int n, bool write, const char* who) {
  DVAE_REQUIRE(n >= 0 && (t || n == 0), "%s: null pointer", who);
  for (int i = 0; i < n; ++i) {
    DVAE_REQUIRE(t[i].n >= 0, "%s: tensor %d has %lld elements", who, i, t[i].n);
    DVAE_REQUIRE(t[i].in_type >= DVAE_F32 && t[i].in_type <= DVAE_F16, "%s: tensor %d has type %d", who, i, t[i].in_type);
    DVAE_REQUIRE(t[i].in || t[i].n == 0, "%s: tensor %d is null", who, i);
    DVAE_REQUIRE((uintptr_t)t[i].in % elem_bytes(t[i].in_type) == 0, "%s: tensor %d is not aligned to its type", who, i);
    if (!write) continue;
    DVAE_REQUIRE(t[i].out_type >= DVAE_F32 && t[i].out_type <= DVAE_F16, "%s: output %d has type %d", who, i, t[i].out_type);
    DVAE_REQUIRE(t[i].out || t[i].n == 0, "%s: output %d is null", who, i);
    DVAE_REQUIRE((uintptr_t)t[i].out % elem_bytes(t[i].out_type) == 0, "%s: output %d is not aligned to its type", who, i);
    DVAE_REQUIRE(t[i].n == 0 || t[i].in != t[i].out || t[i].in_type == t[i].out_type,
                 "%s: tensor %d is its own output in another type", who, i);
  }
  if (!write) return DVAE_OK;
  try {
    std::vector<Span> v;
    v.reserve((size_t)n * 2);
    for (int i = 0; i < n; ++i) {
      if (t[i].n == 0) continue;
      const uintptr_t o = (uintptr_t)t[i].out, p = (uintptr_t)t[i].in;
      v.push_back({o, o + (uintptr_t)t[i].n * elem_bytes(t[i].out_type), i, true});
      if (p != o) v.push_back({p, p + (uintptr_t)t[i].n * elem_bytes(t[i].in_type), i, false});
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

namespace {

// partial sums of all tensors -> ws; `used` their number, `batches` how many batches left them
int partials(const dvae_tensor* tensors, int n, double max_norm, const float* norm_coef, void* ws, int* used, int* batches,
             const char* who, hipStream_t st) {
  DVAE_REQUIRE(norm_coef && ws, "%s: null pointer", who);
  DVAE_REQUIRE(max_norm >= 0.0, "%s: max_norm must not be negative", who);
  double* part = (double*)ws;
  const size_t room = dvae_clip_ws_bytes(n) / sizeof(double);
  *used = *batches = 0;
  return for_batches(tensors, n, [&](const Batch& b, int grid) -> int {
    DVAE_REQUIRE((size_t)*used + grid <= room, "%s: too many batches", who);
    hipLaunchKernelGGL(norm_kernel, dim3(grid), dim3(256), 0, st, b, part + *used);
    DVAE_LAUNCH_CHECK();
    *used += grid;
    ++*batches;
    return DVAE_OK;
  });
}

}  // namespace

extern "C" int dvae_grad_norm(const dvae_tensor* tensors, int n, double max_norm, float* norm_coef, void* ws, void* stream) {
  DVAE_TRY(check_tensors(tensors, n, false, "grad_norm"));
  int used, batches;
  DVAE_TRY(partials(tensors, n, max_norm, norm_coef, ws, &used, &batches, "grad_norm", (hipStream_t)stream));
  hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, (const double*)ws, used, max_norm, norm_coef);
  DVAE_LAUNCH_CHECK();
  return DVAE_OK;
}

extern "C" int dvae_clip_grads(const dvae_tensor* tensors, int n, double max_norm, float* norm_coef, void* ws, void* stream) {
  DVAE_TRY(check_tensors(tensors, n, true, "clip_grads"));
  hipStream_t st = (hipStream_t)stream;
  int used, batches;
  DVAE_TRY(partials(tensors, n, max_norm, norm_coef, ws, &used, &batches, "clip_grads", st));
  if (batches != 1) {                   // several, or no elements at all
    hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(256), 0, st, (const double*)ws, used, max_norm, norm_coef);
    DVAE_LAUNCH_CHECK();
  }
  return for_batches(tensors, n, [&](const Batch& b, int grid) -> int {
    if (batches == 1)
      hipLaunchKernelGGL(scale_kernel<true>, dim3(grid), dim3(256), 0, st, b, (const double*)ws, used, max_norm, norm_coef);
    else
      hipLaunchKernelGGL(scale_kernel<false>, dim3(grid), dim3(256), 0, st, b, nullptr, 0, max_norm, norm_coef);
    DVAE_LAUNCH_CHECK();
    return DVAE_OK;
  });
}
