// How fast the 4-bit matrix instruction goes on this card: operands that stay in registers, and operands read from LDS for every product.
// Build: hipcc --offload-arch=gfx950 -O3 -Xclang -target-feature -Xclang -packed-fp32-ops -o /tmp/mx4_rate_probe tools/probe/mx4_rate_probe.hip
// One wave per SIMD, 16 accumulators of 32 x 32, on zeros and on random codes (the power the card draws depends on them).
#include <hip/hip_runtime.h>
#include <cstdio>
#include <cstdlib>
#include <vector>

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
#define CK(e) do { hipError_t _e = (e); if (_e != hipSuccess) { printf("%s, line %d\n", hipGetErrorString(_e), __LINE__); exit(1); } } while (0)

constexpr int GRID = 256, SLOT = 2048;                                      // v4i of an LDS slot; three of them
struct Acc { f16v c[4][4]; };
__device__ __forceinline__ void clear(Acc& a) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) a.c[i >> 2][i & 3][r] = 0.f;
}
__device__ __forceinline__ void products(Acc& a, const v4i (&A)[4], const v4i (&B)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const v8i x = {A[i][0], A[i][1], A[i][2], A[i][3], 0, 0, 0, 0}, y = {B[j][0], B[j][1], B[j][2], B[j][3], 0, 0, 0, 0};
            a.c[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, a.c[i][j], 4, 4, 0, 127, 0, 127);
        }
}
__device__ __forceinline__ float total(const Acc& a) {
    float s = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s += a.c[i >> 2][i & 3][r];
    return s;
}
__global__ void __launch_bounds__(256, 1) from_registers(const v4i* d, float* o, int n) {
    const int l = threadIdx.x;
    v4i A[4], B[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { A[i] = d[i * 256 + l]; B[i] = d[(4 + i) * 256 + l]; }
    Acc a;
    clear(a);
    for (int k = 0; k < n; ++k) products(a, A, B);
    o[blockIdx.x * 256 + l] = total(a);
}
__global__ void __launch_bounds__(256, 1) from_lds(const v4i* d, float* o, int n) {
    __shared__ v4i L[3 * SLOT];
    const int l = threadIdx.x, lane = l & 63, w = l >> 6;
    for (int i = l; i < 3 * SLOT; i += 256) L[i] = d[i];
    __syncthreads();
    v4i A[2][4], B[2][4];
    Acc a;
    clear(a);
    auto read = [&](int s, v4i (&x)[4], v4i (&y)[4]) {                      // (the largest index: 2 SLOT + 1024 + 512 + 256 + 3 * 64 + 63 < 3 SLOT)
        const v4i* p = L + s % 3 * SLOT + (s & 1) * 512 + lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[i] = p[(w >> 1) * 256 + i * 64]; y[i] = p[1024 + (w & 1) * 256 + i * 64]; }
    };
    read(0, A[0], B[0]);
    for (int k = 0; k < n; k += 2) {
        read(k + 1, A[1], B[1]);
        __builtin_amdgcn_sched_barrier(0);
        products(a, A[0], B[0]);
        __builtin_amdgcn_sched_barrier(0);
        read(k + 2, A[0], B[0]);
        __builtin_amdgcn_sched_barrier(0);
        products(a, A[1], B[1]);
        __builtin_amdgcn_sched_barrier(0);
    }
    o[blockIdx.x * 256 + l] = total(a);
}

int main() {
    std::vector<int> h(4 * 3 * SLOT);
    float* o;
    v4i* d;
    hipEvent_t e0, e1;
    CK(hipMalloc(&o, GRID * 256 * 4));
    CK(hipMalloc(&d, h.size() * 4));
    CK(hipEventCreate(&e0));
    CK(hipEventCreate(&e1));
    for (int random = 0; random < 2; ++random) {
        for (int& x : h) x = random ? rand() ^ (rand() << 16) : 0;
        CK(hipMemcpy(d, h.data(), h.size() * 4, hipMemcpyHostToDevice));
        for (int lds = 0; lds < 2; ++lds)
            for (int n : {2000, 2000, 20000}) {
                float ms;
                CK(hipEventRecord(e0));
                if (lds) from_lds<<<GRID, 256>>>(d, o, n);
                else from_registers<<<GRID, 256>>>(d, o, n);
                CK(hipEventRecord(e1));
                CK(hipEventSynchronize(e1));
                CK(hipEventElapsedTime(&ms, e0, e1));
                printf("%s operands from %s, %d steps: %.0f us, %.2f PFLOP/s\n", random ? "random" : "zero", lds ? "LDS" : "registers", n, ms * 1e3,
                       double(GRID) * 4 * n * 16 * 32 * 32 * 64 * 2 / ms / 1e12);
            }
    }
    return 0;
}
