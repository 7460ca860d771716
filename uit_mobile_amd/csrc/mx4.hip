// mx4.hip -- microscaled 4-bit floating point (OCP MXFP4): quantisation, the values back, and the linear layer on 4-bit operands.
//
//   quantize    block of 32: e = floor(log2 max |v|), scale 2^X, X = max(e - 2, -127); code = v / 2^X to the nearest e2m1 value, ties to
//               the even code, beyond 6 to 6.  (X = e - 2 puts the largest element into [4, 8): the top binade of e2m1.)
//   linear      out = residual + act(Q(x) W^T + bias); products of 4-bit operands are exact in fp32, their sum is held in fp32
// The layout of packed matrices: mx4_dev.h.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "../../include/uitk.h"
#include "mx4_dev.h"

namespace uitk {

int set_error(int code, const std::string& msg);                          // api.cpp: the thread's uitk_last_error text

// ------------------------------------------------------------------------------------------------------------------- quantize
// One wave per record: lane (r = l % 32, g = l / 32) owns the blocks (row 32 rt + r, elements 64 kh + 32 g ..) of the four fragments,
// so the maximum, the scale and the 16 bytes of a block never leave the lane, and a wave writes whole contiguous fragments.
template <typename T>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(const T* __restrict__ x, int64_t rows, int64_t K, int64_t ld, int vec, int64_t R, int64_t S,
                                                           char* __restrict__ codes, char* __restrict__ scales) {
    const int lane = threadIdx.x & 63, r = lane & 31, g = lane >> 5;
    const int64_t rec = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (rec >= R * S) return;
    const int64_t rg = rec / S, s = rec - rg * S;
    unsigned sc = 0;
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        const int64_t row = rg * MX4_ROWS + 32 * (f >> 1) + r, k = s * MX4_K + 64 * (f & 1) + 32 * g;
        Mx4Block b{mx_i4{0, 0, 0, 0}, 0};
        if (row < rows && k < K) {
            Mx4Src<T> src;
            src.load(x + row * ld + k, vec, (int)min((int64_t)32, K - k));
            b = src.pack();
        }
        *(mx_i4*)(codes + rec * MX4_CODES + f * 1024 + lane * 16) = b.codes;
        sc |= b.scale << (8 * f);
    }
    *(unsigned*)(scales + rec * MX4_SCALES + lane * 4) = sc;
}

template <typename T>
__global__ void __launch_bounds__(256) mx4_dequantize_kernel(const char* __restrict__ codes, const char* __restrict__ scales, int64_t rows, int64_t K, int64_t ld,
                                                             int64_t R, int64_t S, T* __restrict__ x) {
    const int lane = threadIdx.x & 63, r = lane & 31, g = lane >> 5;
    const int64_t rec = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (rec >= R * S) return;
    const int64_t rg = rec / S, s = rec - rg * S;
    const unsigned sc = *(const unsigned*)(scales + rec * MX4_SCALES + lane * 4);
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        const int64_t row = rg * MX4_ROWS + 32 * (f >> 1) + r, k = s * MX4_K + 64 * (f & 1) + 32 * g;
        if (row >= rows || k >= K) continue;
        const mx_i4 c = *(const mx_i4*)(codes + rec * MX4_CODES + f * 1024 + lane * 16);
        const unsigned byte = sc >> (8 * f) & 255u;
        const int n = (int)min((int64_t)32, K - k);
        T* out = x + row * ld + k;
        // 2^(byte - 127) in two steps: half of it is never subnormal for byte >= 2, and for byte < 2 the products stay exact
        for (int j = 0; j < n; ++j) {
            const unsigned code = (unsigned)c[j >> 3] >> (4 * (j & 7)) & 15u;
            const unsigned mag = code & 7u;
            const float m = mag < 2u ? 0.5f * mag : __uint_as_float(((mag >> 1) + 126u) << 23 | (mag & 1u) << 22);
            const float v = byte == 255u ? __uint_as_float(0x7fc00000u) : ldexpf(code & 8u ? -m : m, (int)byte - 127);
            out[j] = (T)v;
        }
    }
}

// --------------------------------------------------------------------------------------------------------------------- linear
struct Mx4LinearArgs {
    const void* x; int64_t M, K, ldx; int x_type, x_vec;                    // x_type MT_MX4: x = codes of a packed matrix, x_scales its scales
    const char* x_scales;
    const char* w; const char* w_scales;                                    // packed [N, K]
    int64_t N, S;                                                           // S = records along K
    const float* bias;
    int act;                                                                // 0 none, 1 ReLU, 2 exact GELU
    const void* residual; int64_t ldr;                                      // of the output's type, added last
    void* out; int64_t ldo; int out_type;                                   // MT_MX4: out = codes, out_scales its scales
    char* out_scales; int64_t out_S;
    unsigned ngroups;                                                       // groups of 64 columns
    int vec4;                                                               // every four-element group of bias / residual / out is aligned
};

// four consecutive outputs (row m, columns n ..): bias, activation, residual, one rounding, store
__device__ __forceinline__ void mx4_store4(const Mx4LinearArgs& a, int64_t m, int64_t n, float (&v)[4]) {
    const bool in_m = m < a.M;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (a.bias && n + i < a.N) v[i] += a.bias[n + i];
        if (a.act == 1) v[i] = v[i] > 0.f ? v[i] : (v[i] != v[i] ? v[i] : 0.f);              // a NaN stays one
        else if (a.act == 2) v[i] = mx4_gelu(v[i]);
    }
    if (a.out_type == MT_MX4) {                                             // (8 neighbouring lanes hold one block: no divergence up to here)
#pragma unroll
        for (int i = 0; i < 4; ++i) if (n + i >= a.N) v[i] = 0.f;
        unsigned sc;
        const unsigned two = mx4_pack_quads(v, &sc);
        if (!in_m || (n >> 7) >= a.out_S) return;
        const Mx4Place p = mx4_place(m, n >> 5, a.out_S);
        *(unsigned short*)((char*)a.out + p.code + ((n & 31) >> 1)) = (unsigned short)two;
        if ((n & 31) == 0) a.out_scales[p.scale] = (char)sc;
        return;
    }
    if (!in_m || n >= a.N) return;
    const bool four = a.vec4 && n + 4 <= a.N;
    if (a.out_type == MT_F32) {
        float* o = (float*)a.out + m * a.ldo + n;
        const float* r = a.residual ? (const float*)a.residual + m * a.ldr + n : nullptr;
        if (four) {
            mx_f4 t = {v[0], v[1], v[2], v[3]};
            if (r) t += *(const mx_f4*)r;
            *(mx_f4*)o = t;
        } else {
            for (int i = 0; i < 4; ++i) if (n + i < a.N) o[i] = r ? r[i] + v[i] : v[i];
        }
        return;
    }
    unsigned short* o = (unsigned short*)a.out + m * a.ldo + n;
    const unsigned short* r = a.residual ? (const unsigned short*)a.residual + m * a.ldr + n : nullptr;
    unsigned short t[4] = {0, 0, 0, 0};
    if (r) {
        if (four) { const mx_u2 u = *(const mx_u2*)r; t[0] = (unsigned short)u[0]; t[1] = (unsigned short)(u[0] >> 16); t[2] = (unsigned short)u[1]; t[3] = (unsigned short)(u[1] >> 16); }
        else for (int i = 0; i < 4; ++i) if (n + i < a.N) t[i] = r[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (a.out_type == MT_F16) {
            if (r) v[i] += (float)__builtin_bit_cast(_Float16, t[i]);
            t[i] = __builtin_bit_cast(unsigned short, (_Float16)v[i]);
        } else {
            if (r) v[i] += __uint_as_float((unsigned)t[i] << 16);
            t[i] = __builtin_bit_cast(unsigned short, (__bf16)v[i]);
        }
    }
    if (four) *(mx_u2*)o = mx_u2{(unsigned)t[0] | (unsigned)t[1] << 16, (unsigned)t[2] | (unsigned)t[3] << 16};
    else for (int i = 0; i < 4; ++i) if (n + i < a.N) o[i] = t[i];
}

// A workgroup computes 64 outputs (n) x 32 TT tokens (m); its waves take the records of K in turn, each with its own accumulators, and
// join them through LDS in a fixed order.  Operands go from memory to registers in fragment order; activations that are not packed yet
// are quantised by the lane that multiplies them (lane l of the B operand owns row l % 32, block l / 32: a whole block).
template <int TT, typename XT>
__device__ __forceinline__ void mx4_x_fragment(const Mx4LinearArgs& a, int64_t row, int64_t k, Mx4Block& b) {
    b.codes = mx_i4{0, 0, 0, 0}; b.scale = 0;
    if (row < a.M && k < a.K) {
        Mx4Src<XT> src;
        src.load((const XT*)a.x + row * a.ldx + k, a.x_vec, (int)min((int64_t)32, a.K - k));
        b = src.pack();
    }
}

template <int TT, typename XT, bool PACKED>
__global__ void __launch_bounds__(256) mx4_linear_kernel(Mx4LinearArgs a) {
    constexpr int NW = 4, LDT = 64 + 4;                                     // waves; floats per token row of the joining buffer
    __shared__ __attribute__((aligned(16))) float red[NW][32 * TT][LDT];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 31, g = lane >> 5;
    const int64_t ng = blockIdx.x % a.ngroups, m0 = (int64_t)(blockIdx.x / a.ngroups) * 32 * TT;
    mx_f16 acc[2][TT];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[rt][t][i] = 0.f;
    const int64_t nrec_rows = (a.N + MX4_ROWS - 1) / MX4_ROWS;
    if (ng < nrec_rows) {                                                   // (an out_type of 4 bits pads its columns to 128: such a group multiplies nothing)
        for (int64_t s = wave; s < a.S; s += NW) {
            const char* wc = a.w + (ng * a.S + s) * MX4_CODES;
            const int ws = *(const int*)(a.w_scales + (ng * a.S + s) * MX4_SCALES + lane * 4);
            mx_i4 wf[4];
#pragma unroll
            for (int f = 0; f < 4; ++f) wf[f] = *(const mx_i4*)(wc + f * 1024 + lane * 16);
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                if constexpr (PACKED) {
                    const int64_t row = m0 + 32 * t;                        // a multiple of 32: row tile (row / 32) % 2 of its record
                    if (row >= a.M) continue;
                    const int64_t rec = (row >> 6) * a.S + s;
                    const int rt = (int)(row >> 5) & 1;
                    const int xs = *(const int*)(a.x_scales + rec * MX4_SCALES + lane * 4) >> (16 * rt);
                    const char* xc = (const char*)a.x + rec * MX4_CODES + rt * 2048;
                    const mx_i4 x0 = *(const mx_i4*)(xc + lane * 16), x1 = *(const mx_i4*)(xc + 1024 + lane * 16);
                    acc[0][t] = mx4_mfma<0, 0>(wf[0], x0, acc[0][t], ws, xs);
                    acc[1][t] = mx4_mfma<2, 0>(wf[2], x0, acc[1][t], ws, xs);
                    acc[0][t] = mx4_mfma<1, 1>(wf[1], x1, acc[0][t], ws, xs);
                    acc[1][t] = mx4_mfma<3, 1>(wf[3], x1, acc[1][t], ws, xs);
                } else {
                    Mx4Block x0, x1;
                    mx4_x_fragment<TT, XT>(a, m0 + 32 * t + c, s * MX4_K + 32 * g, x0);
                    mx4_x_fragment<TT, XT>(a, m0 + 32 * t + c, s * MX4_K + 64 + 32 * g, x1);
                    acc[0][t] = mx4_mfma<0, 0>(wf[0], x0.codes, acc[0][t], ws, (int)x0.scale);
                    acc[1][t] = mx4_mfma<2, 0>(wf[2], x0.codes, acc[1][t], ws, (int)x0.scale);
                    acc[0][t] = mx4_mfma<1, 0>(wf[1], x1.codes, acc[0][t], ws, (int)x1.scale);
                    acc[1][t] = mx4_mfma<3, 0>(wf[3], x1.codes, acc[1][t], ws, (int)x1.scale);
                }
            }
        }
    }
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *(mx_f4*)&red[wave][32 * t + c][32 * rt + 8 * q + 4 * g] = mx_f4{acc[rt][t][4 * q], acc[rt][t][4 * q + 1], acc[rt][t][4 * q + 2], acc[rt][t][4 * q + 3]};
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * TT * 16; i += 256) {
        const int t = i >> 4, n4 = (i & 15) * 4;
        mx_f4 s = *(const mx_f4*)&red[0][t][n4];
#pragma unroll
        for (int w = 1; w < NW; ++w) s += *(const mx_f4*)&red[w][t][n4];
        float v[4] = {s[0], s[1], s[2], s[3]};
        mx4_store4(a, m0 + t, ng * 64 + n4, v);
    }
}

}  // namespace uitk

// --------------------------------------------------------------------------------------------------------------- host side + C ABI
using namespace uitk;

#define MX4_HIP(expr)                                                                                          \
    do {                                                                                                       \
        hipError_t _e = (expr);                                                                                \
        if (_e != hipSuccess) return set_error(UITK_ERR_HIP, std::string(#expr) + ": " + hipGetErrorString(_e)); \
    } while (0)

constexpr int64_t MX4_MAX_GRID = ((int64_t)1 << 32) / 256 - 1;            // workgroups of 256: a launch counts its threads in 32 bits
constexpr int64_t MX4_MAX_ROWS = (int64_t)1 << 31, MX4_MAX_K = (int64_t)1 << 20;

static int mx4_check_matrix(const char* what, int64_t rows, int64_t K) {
    if (rows < 0 || rows > MX4_MAX_ROWS) return set_error(UITK_ERR_INVALID_ARG, std::string(what) + ": the number of rows must be 0 .. 2^31");
    if (K < 1 || K > MX4_MAX_K) return set_error(UITK_ERR_INVALID_ARG, std::string(what) + ": the width must be 1 .. 2^20");
    return UITK_OK;
}
static int type_size(int t) { return t == UITK_T_F32 ? 4 : 2; }
static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int TT>
static void mx4_launch_linear(dim3 grid, const Mx4LinearArgs& a, hipStream_t s) {
    if (a.x_type == MT_MX4) hipLaunchKernelGGL((mx4_linear_kernel<TT, float, true>), grid, dim3(256), 0, s, a);
    else if (a.x_type == MT_F32) hipLaunchKernelGGL((mx4_linear_kernel<TT, float, false>), grid, dim3(256), 0, s, a);
    else if (a.x_type == MT_F16) hipLaunchKernelGGL((mx4_linear_kernel<TT, _Float16, false>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((mx4_linear_kernel<TT, __bf16, false>), grid, dim3(256), 0, s, a);
}

extern "C" {

int64_t uitk_mx4_bytes(int64_t rows, int64_t K) {
    if (rows < 0 || rows > MX4_MAX_ROWS || K < 1 || K > MX4_MAX_K) return -1;
    return mx4_bytes(rows, K);
}

int uitk_mx4_quantize(const void* x, int type, int64_t rows, int64_t K, int64_t ld, void* q, void* stream) {
    if (int rc = mx4_check_matrix("uitk_mx4_quantize", rows, K)) return rc;
    if (type < UITK_T_F32 || type > UITK_T_BF16) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_quantize: unknown type");
    if (rows == 0) return UITK_OK;
    if (!x || !q) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_quantize: null pointer");
    if (ld < K) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_quantize: rows overlap (ld < K)");
    if (!aligned16(q)) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_quantize: the packed buffer must be 16-byte aligned");
    const int64_t R = (rows + MX4_ROWS - 1) / MX4_ROWS, S = (K + MX4_K - 1) / MX4_K;
    char* codes = (char*)q;
    char* scales = codes + R * S * MX4_CODES;
    const int vec = aligned16(x) && (ld * type_size(type)) % 16 == 0;
    if ((R * S + 3) / 4 > MX4_MAX_GRID) return set_error(UITK_ERR_UNSUPPORTED, "uitk_mx4_quantize: more elements than one launch takes");
    const dim3 grid((unsigned)((R * S + 3) / 4)), block(256);
    hipStream_t s = (hipStream_t)stream;
    if (type == UITK_T_F32) hipLaunchKernelGGL(mx4_quantize_kernel<float>, grid, block, 0, s, (const float*)x, rows, K, ld, vec, R, S, codes, scales);
    else if (type == UITK_T_F16) hipLaunchKernelGGL(mx4_quantize_kernel<_Float16>, grid, block, 0, s, (const _Float16*)x, rows, K, ld, vec, R, S, codes, scales);
    else hipLaunchKernelGGL(mx4_quantize_kernel<__bf16>, grid, block, 0, s, (const __bf16*)x, rows, K, ld, vec, R, S, codes, scales);
    MX4_HIP(hipGetLastError());
    return UITK_OK;
}

int uitk_mx4_dequantize(const void* q, int64_t rows, int64_t K, void* x, int type, int64_t ld, void* stream) {
    if (int rc = mx4_check_matrix("uitk_mx4_dequantize", rows, K)) return rc;
    if (type < UITK_T_F32 || type > UITK_T_BF16) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_dequantize: unknown type");
    if (rows == 0) return UITK_OK;
    if (!x || !q) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_dequantize: null pointer");
    if (ld < K) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_dequantize: rows overlap (ld < K)");
    if (!aligned16(q)) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_dequantize: the packed buffer must be 16-byte aligned");
    const int64_t R = (rows + MX4_ROWS - 1) / MX4_ROWS, S = (K + MX4_K - 1) / MX4_K;
    if ((R * S + 3) / 4 > MX4_MAX_GRID) return set_error(UITK_ERR_UNSUPPORTED, "uitk_mx4_dequantize: more elements than one launch takes");
    const char* codes = (const char*)q;
    const char* scales = codes + R * S * MX4_CODES;
    const dim3 grid((unsigned)((R * S + 3) / 4)), block(256);
    hipStream_t s = (hipStream_t)stream;
    if (type == UITK_T_F32) hipLaunchKernelGGL(mx4_dequantize_kernel<float>, grid, block, 0, s, codes, scales, rows, K, ld, R, S, (float*)x);
    else if (type == UITK_T_F16) hipLaunchKernelGGL(mx4_dequantize_kernel<_Float16>, grid, block, 0, s, codes, scales, rows, K, ld, R, S, (_Float16*)x);
    else hipLaunchKernelGGL(mx4_dequantize_kernel<__bf16>, grid, block, 0, s, codes, scales, rows, K, ld, R, S, (__bf16*)x);
    MX4_HIP(hipGetLastError());
    return UITK_OK;
}

// Activations that are not packed: quantised inside the product (few rows) -- no workspace so far
int64_t uitk_mx4_linear_workspace(int64_t M, int64_t N, int64_t K, int x_type) {
    if (M < 0 || M > MX4_MAX_ROWS || N < 1 || N > MX4_MAX_K || K < 1 || K > MX4_MAX_K || x_type < UITK_T_F32 || x_type > UITK_T_MX4) return -1;
    return 0;
}

int uitk_mx4_linear(const uitk_mx4_linear_args* u, void* stream) {
    if (!u) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: null arguments");
    if (int rc = mx4_check_matrix("uitk_mx4_linear (x)", u->M, u->K)) return rc;
    if (u->N < 1 || u->N > MX4_MAX_K) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: N must be 1 .. 2^20");
    if (u->x_type < UITK_T_F32 || u->x_type > UITK_T_MX4) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: unknown x_type");
    if (u->out_type < UITK_T_F32 || u->out_type > UITK_T_MX4) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: unknown out_type");
    if (u->act < 0 || u->act > 2) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: act must be 0 (none), 1 (ReLU) or 2 (GELU)");
    if (u->residual && u->out_type == UITK_T_MX4) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: a residual needs an output of 16 or 32 bits");
    if (u->M == 0) return UITK_OK;
    if (!u->x || !u->w || !u->out) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: null pointer");
    if (!aligned16(u->w) || (u->x_type == UITK_T_MX4 && !aligned16(u->x)) || (u->out_type == UITK_T_MX4 && !aligned16(u->out)))
        return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: packed matrices must be 16-byte aligned");
    if (u->x_type != UITK_T_MX4 && u->ldx < u->K) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: rows of x overlap (ldx < K)");
    if (u->out_type != UITK_T_MX4 && u->ldo < u->N) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: rows of the output overlap (ldo < N)");
    if (u->residual && u->ldr < u->N) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: rows of the residual overlap (ldr < N)");
    Mx4LinearArgs a{};
    a.M = u->M; a.K = u->K; a.N = u->N; a.S = (u->K + MX4_K - 1) / MX4_K;
    a.x = u->x; a.x_type = u->x_type; a.ldx = u->ldx;
    if (u->x_type == UITK_T_MX4) a.x_scales = (const char*)u->x + mx4_records(u->M, u->K) * MX4_CODES;
    else a.x_vec = aligned16(u->x) && (u->ldx * type_size(u->x_type)) % 16 == 0;
    a.w = (const char*)u->w; a.w_scales = a.w + mx4_records(u->N, u->K) * MX4_CODES;
    a.bias = u->bias; a.act = u->act; a.residual = u->residual; a.ldr = u->ldr;
    a.out = u->out; a.ldo = u->ldo; a.out_type = u->out_type;
    if (u->out_type == UITK_T_MX4) { a.out_S = (u->N + MX4_K - 1) / MX4_K; a.out_scales = (char*)u->out + mx4_records(u->M, u->N) * MX4_CODES; }
    else {
        const int sz = type_size(u->out_type), grp = 4 * sz;
        a.vec4 = (uintptr_t)u->out % grp == 0 && u->ldo % 4 == 0 && (!u->residual || ((uintptr_t)u->residual % grp == 0 && u->ldr % 4 == 0));
    }
    const int64_t ngroups = u->out_type == UITK_T_MX4 ? 2 * a.out_S : (u->N + MX4_ROWS - 1) / MX4_ROWS;
    hipStream_t s = (hipStream_t)stream;
    const int tt = u->M <= 32 ? 1 : 2;
    const int64_t mt = (u->M + 32 * tt - 1) / (32 * tt);
    if (mt * ngroups > MX4_MAX_GRID) return set_error(UITK_ERR_UNSUPPORTED, "uitk_mx4_linear: more outputs than one launch takes");
    a.ngroups = (unsigned)ngroups;
    const dim3 grid((unsigned)(mt * ngroups));
    if (tt == 1) mx4_launch_linear<1>(grid, a, s); else mx4_launch_linear<2>(grid, a, s);
    MX4_HIP(hipGetLastError());
    return UITK_OK;
}

}  // extern "C"
