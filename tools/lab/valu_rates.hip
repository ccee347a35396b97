// Cycles a wave instruction takes on a full card (2048 workgroups of 4 waves, eight independent chains a lane): the rates behind
// the choice of doubles in csrc/rules.hip.
//   hipcc -O3 --offload-arch=gfx950 -Xclang -target-feature -Xclang -packed-fp32-ops tools/lab/valu_rates.hip -o valu_rates
#include <hip/hip_runtime.h>
#include <cstdio>

enum { FMA64, ADD64, MUL64, MAX64, EXP2F, FMA32, ADD32 };

template <int OP>
__global__ __launch_bounds__(256) void chains(double* out, double a, float fa, int n) {
  double x[8];
  float f[8];
  for (int i = 0; i < 8; ++i) {
    x[i] = a + i + threadIdx.x;
    f[i] = fa + i;
  }
  for (int r = 0; r < n; ++r) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (OP == FMA64) x[i] = fma(x[i], a, 0.5);
      if (OP == ADD64) x[i] = x[i] + a;
      if (OP == MUL64) x[i] = x[i] * a;
      if (OP == MAX64) x[i] = fmax(x[i], a);
      if (OP == EXP2F) f[i] = __builtin_amdgcn_exp2f(f[i]);
      if (OP == FMA32) f[i] = fmaf(f[i], fa, 0.5f);
      if (OP == ADD32) f[i] = f[i] + fa;
    }
  }
  double s = 0;
  for (int i = 0; i < 8; ++i) s += x[i] + f[i];
  out[blockIdx.x * 256 + threadIdx.x] = s;
}

template <int OP>
void run(const char* name, double* out) {
  const int n = 2000;
  hipEvent_t a, b;
  if (hipEventCreate(&a) != hipSuccess || hipEventCreate(&b) != hipSuccess) return;
  float ms = 0.f;
  for (int t = 0; t < 2; ++t) {
    (void)hipEventRecord(a);
    hipLaunchKernelGGL((chains<OP>), dim3(2048), dim3(256), 0, 0, out, 1.0000001, 0.9999f, n);
    (void)hipEventRecord(b);
    if (hipEventSynchronize(b) != hipSuccess) return;
    (void)hipEventElapsedTime(&ms, a, b);
  }
  const double per_simd = 2048.0 * 4 / 1024 * n * 8;          // wave instructions of one of the 1024 SIMDs
  printf("%-8s %.2f cycles at 2.4 GHz\n", name, ms * 1e-3 * 2.4e9 / per_simd);
}

int main() {
  double* out;
  if (hipMalloc(&out, 2048 * 256 * 8) != hipSuccess) return 1;
  run<FMA64>("fma64", out);
  run<ADD64>("add64", out);
  run<MUL64>("mul64", out);
  run<MAX64>("max64", out);
  run<EXP2F>("exp2f", out);
  run<FMA32>("fma32", out);
  run<ADD32>("add32", out);
  return 0;
}
