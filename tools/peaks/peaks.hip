// Measured peaks of the device this runs on, for pricing the roofline against what the machine delivers as well as
// against the vendor figures: HBM read, HBM copy (read + write) and dense bf16 MFMA (v_mfma_f32_32x32x16_bf16).
// Build: hipcc --offload-arch=gfx950 -Xclang -target-feature -Xclang -packed-fp32-ops -O3 -o tools/peaks/peaks tools/peaks/peaks.hip      Run: tools/peaks/peaks
#include <hip/hip_runtime.h>
#include <cstdio>
#include <cstdlib>

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

#define CHECK(x) do { hipError_t e_ = (x); if (e_ != hipSuccess) { fprintf(stderr, "%s: %s\n", #x, hipGetErrorString(e_)); exit(1); } } while (0)

__global__ __launch_bounds__(256) void copy_kernel(const f32x4* __restrict__ src, f32x4* __restrict__ dst, long long n4) {
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n4; i += (long long)gridDim.x * 256) dst[i] = src[i];
}

__global__ __launch_bounds__(256) void read_kernel(const f32x4* __restrict__ src, float* __restrict__ out, long long n4) {
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n4; i += (long long)gridDim.x * 256) a += src[i];
    if (a[0] + a[1] + a[2] + a[3] == 12345.678f) out[0] = 1.f;        // never true for the zero-filled buffer: keeps the loads alive
}

// every wave keeps four independent accumulator tiles in flight; operands never change (register resident)
__global__ __launch_bounds__(256) void mfma_kernel(float* __restrict__ out, int iters) {
    bf16x8 a, b;
    for (int j = 0; j < 8; ++j) { a[j] = (__bf16)(float)(threadIdx.x & 3); b[j] = (__bf16)0.5f; }
    f32x16 c0 = {}, c1 = {}, c2 = {}, c3 = {};
    for (int i = 0; i < iters; ++i) {
        c0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c0, 0, 0, 0);
        c1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c1, 0, 0, 0);
        c2 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c2, 0, 0, 0);
        c3 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c3, 0, 0, 0);
    }
    const f32x16 s = c0 + c1 + c2 + c3;
    float t = 0.f;
    for (int j = 0; j < 16; ++j) t += s[j];
    if (t == 12345.678f) out[0] = t;
}

static float time_ms(hipEvent_t e0, hipEvent_t e1) { float ms; CHECK(hipEventElapsedTime(&ms, e0, e1)); return ms; }

int main() {
    hipDeviceProp_t p;
    CHECK(hipGetDeviceProperties(&p, 0));
    const long long bytes = 2ll << 30;
    f32x4 *a, *b; float* o;
    CHECK(hipMalloc(&a, bytes)); CHECK(hipMalloc(&b, bytes)); CHECK(hipMalloc(&o, 64));
    CHECK(hipMemset(a, 0, bytes)); CHECK(hipMemset(b, 0, bytes));
    hipEvent_t e0, e1; CHECK(hipEventCreate(&e0)); CHECK(hipEventCreate(&e1));
    const long long n4 = bytes / 16;
    const int grid = p.multiProcessorCount * 8, reps = 10;
    double best_copy = 0, best_read = 0, best_mfma = 0;
    for (int r = 0; r < reps + 2; ++r) {
        CHECK(hipEventRecord(e0)); hipLaunchKernelGGL(copy_kernel, dim3(grid), dim3(256), 0, 0, a, b, n4); CHECK(hipEventRecord(e1)); CHECK(hipEventSynchronize(e1));
        const double gbs = 2.0 * bytes / (time_ms(e0, e1) * 1e-3) * 1e-9;
        if (r >= 2 && gbs > best_copy) best_copy = gbs;
        CHECK(hipEventRecord(e0)); hipLaunchKernelGGL(read_kernel, dim3(grid), dim3(256), 0, 0, a, o, n4); CHECK(hipEventRecord(e1)); CHECK(hipEventSynchronize(e1));
        const double gr = 1.0 * bytes / (time_ms(e0, e1) * 1e-3) * 1e-9;
        if (r >= 2 && gr > best_read) best_read = gr;
        const int iters = 4096, wgs = p.multiProcessorCount * 8;       // 8 workgroups x 4 waves per CU = 8 waves per SIMD
        CHECK(hipEventRecord(e0)); hipLaunchKernelGGL(mfma_kernel, dim3(wgs), dim3(256), 0, 0, o, iters); CHECK(hipEventRecord(e1)); CHECK(hipEventSynchronize(e1));
        const double flops = 2.0 * 32 * 32 * 16 * 4.0 * iters * (double)wgs * 4;
        const double tf = flops / (time_ms(e0, e1) * 1e-3) * 1e-12;
        if (r >= 2 && tf > best_mfma) best_mfma = tf;
    }
    printf("{\"device\": \"%s\", \"cus\": %d, \"hbm_read_GBs\": %.0f, \"hbm_copy_GBs\": %.0f, \"mfma_bf16_dense_TFLOPs\": %.0f, \"clock_MHz\": %d}\n",
           p.gcnArchName, p.multiProcessorCount, best_read, best_copy, best_mfma, p.clockRate / 1000);
    return 0;
}
