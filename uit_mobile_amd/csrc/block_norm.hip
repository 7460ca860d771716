// block_norm.hip -- the seam between two blocks of a transformer in one pass over the residual stream:
//
//     z  = post(y)                      norm behind the block (optional)
//     r' = r + gate * scale * z         gate: a row per sequence or per token (optional); scale: one gain per channel (LayerScale; optional)
//     h  = pre(r')                      norm in front of the next block (optional), 32, 16 or 4 bits (mx4_dev.h)
//
// post / pre: LayerNorm ((v - mean) / sqrt(var + eps)) or root mean square (v / sqrt(mean(v^2) + eps)), then gain and offset (each optional).
// All of it in fp32 from the inputs to the one rounding of each output; h is taken from the unrounded r'.  (models/uit.py:244-247: Block.forward,
// whose LayerScale is :78-85.)
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "../../include/uitk.h"
#include "mx4_dev.h"

namespace uitk {

int set_error(int code, const std::string& msg);                          // api.cpp: the thread's uitk_last_error text

struct BlockNormArgs {
    const void* y; int y_type; int64_t ldy;
    const void* r; int r_type; int64_t ldr;
    int64_t rows; int D;
    int rms; float eps;
    int post; const float* post_w; const float* post_b;
    const void* gate; int gate_type; int64_t ldg, gate_rows;
    const float* scale;
    void* ro; int64_t ldro;
    int pre; const float* pre_w; const float* pre_b;
    void* h; int h_type; int64_t ldh;
    char* h_scales; int64_t h_S;
    int vec;                                                                // every group of four elements of every operand is aligned
};

// four elements of a row, zeros behind its end
__device__ __forceinline__ void bn_load4(const void* base, int type, int64_t off, int n, int vec, float (&v)[4]) {
    if (type == MT_F32) {
        const float* p = (const float*)base + off;
        if (vec && n >= 4) { const mx_f4 t = *(const mx_f4*)p; v[0] = t[0]; v[1] = t[1]; v[2] = t[2]; v[3] = t[3]; }
        else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.f;
        }
        return;
    }
    const unsigned short* p = (const unsigned short*)base + off;
    unsigned short t[4];
    if (vec && n >= 4) { const mx_u2 u = *(const mx_u2*)p; t[0] = (unsigned short)u[0]; t[1] = (unsigned short)(u[0] >> 16); t[2] = (unsigned short)u[1]; t[3] = (unsigned short)(u[1] >> 16); }
    else {
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = i < n ? p[i] : (unsigned short)0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = type == MT_F16 ? (float)__builtin_bit_cast(_Float16, t[i]) : __uint_as_float((unsigned)t[i] << 16);
}

__device__ __forceinline__ void bn_store4(void* base, int type, int64_t off, int n, int vec, const float (&v)[4]) {
    if (type == MT_F32) {
        float* p = (float*)base + off;
        if (vec && n >= 4) *(mx_f4*)p = mx_f4{v[0], v[1], v[2], v[3]};
        else {
#pragma unroll
            for (int i = 0; i < 4; ++i) if (i < n) p[i] = v[i];
        }
        return;
    }
    unsigned short* p = (unsigned short*)base + off;
    unsigned short t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = type == MT_F16 ? __builtin_bit_cast(unsigned short, (_Float16)v[i]) : __builtin_bit_cast(unsigned short, (__bf16)v[i]);
    if (vec && n >= 4) *(mx_u2*)p = mx_u2{(unsigned)t[0] | (unsigned)t[1] << 16, (unsigned)t[2] | (unsigned)t[3] << 16};
    else {
#pragma unroll
        for (int i = 0; i < 4; ++i) if (i < n) p[i] = t[i];
    }
}

__device__ __forceinline__ float bn_block_sum(float v, float* red) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();                                                        // (the previous sum has been read)
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// mean and 1 / deviation of the row in LDS (its length D; the rest of the row buffer holds zeros)
__device__ __forceinline__ void bn_stats(const float* row, int D, int rms, float eps, float* red, float* mean, float* rstd) {
    *mean = 0.f;
    if (!rms) {
        float s = 0.f;
        for (int c = threadIdx.x; c < D; c += 256) s += row[c];
        *mean = bn_block_sum(s, red) / (float)D;
    }
    float q = 0.f;
    for (int c = threadIdx.x; c < D; c += 256) { const float d = row[c] - *mean; q += d * d; }
    *rstd = 1.0f / sqrtf(bn_block_sum(q, red) / (float)D + eps);
}

// one workgroup per row; the row stays in LDS between the passes
__global__ void __launch_bounds__(256) block_norm_kernel(BlockNormArgs a) {
    extern __shared__ __attribute__((aligned(16))) float row[];             // [D rounded up to 128]
    __shared__ float red[4];
    const int Dp = (a.D + 127) & ~127;
    for (int64_t m = blockIdx.x; m < a.rows; m += gridDim.x) {
        __syncthreads();
        float mean = 0.f, rstd = 1.f;
        if (a.y) {
            for (int c = 4 * threadIdx.x; c < Dp; c += 1024) {
                float v[4];
                bn_load4(a.y, a.y_type, m * a.ldy + c, a.D - c, a.vec, v);
#pragma unroll
                for (int i = 0; i < 4; ++i) row[c + i] = v[i];
            }
            __syncthreads();
            if (a.post) bn_stats(row, a.D, a.rms, a.eps, red, &mean, &rstd);
        }
        for (int c = 4 * threadIdx.x; c < Dp; c += 1024) {                  // (each thread reads and writes its own elements of the row)
            float v[4], z[4], g[4] = {1.f, 1.f, 1.f, 1.f};
            bn_load4(a.r, a.r_type, m * a.ldr + c, a.D - c, a.vec, v);
            if (a.y) {
                if (a.gate) bn_load4(a.gate, a.gate_type, (m / a.gate_rows) * a.ldg + c, a.D - c, a.vec, g);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    z[i] = row[c + i];
                    if (c + i < a.D) {
                        if (a.post) z[i] = (z[i] - mean) * rstd * (a.post_w ? a.post_w[c + i] : 1.f) + (a.post_b ? a.post_b[c + i] : 0.f);
                        if (a.gate) z[i] *= g[i];
                        if (a.scale) z[i] *= a.scale[c + i];
                    }
                    v[i] += z[i];
                }
                bn_store4(a.ro, a.r_type, m * a.ldro + c, a.D - c, a.vec, v);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) row[c + i] = v[i];
        }
        if (!a.pre) continue;
        __syncthreads();
        bn_stats(row, a.D, a.rms, a.eps, red, &mean, &rstd);
        for (int c = 4 * threadIdx.x; c < Dp; c += 1024) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = c + i < a.D ? (row[c + i] - mean) * rstd * (a.pre_w ? a.pre_w[c + i] : 1.f) + (a.pre_b ? a.pre_b[c + i] : 0.f) : 0.f;
            if (a.h_type == MT_MX4) {                                       // (Dp is a multiple of 128: whole groups of 8 lanes are here together)
                unsigned sc;
                const unsigned two = mx4_pack_quads(v, &sc);
                const Mx4Place p = mx4_place(m, c >> 5, a.h_S);
                *(unsigned short*)((char*)a.h + p.code + ((c & 31) >> 1)) = (unsigned short)two;
                if ((c & 31) == 0) a.h_scales[p.scale] = (char)sc;
            } else {
                bn_store4(a.h, a.h_type, m * a.ldh + c, a.D - c, a.vec, v);
            }
        }
    }
}

}  // namespace uitk

// --------------------------------------------------------------------------------------------------------------- host side + C ABI
using namespace uitk;

extern "C" int uitk_block_norm(const uitk_block_norm_args* u, void* stream) {
    auto bad = [](const char* s) { return set_error(UITK_ERR_INVALID_ARG, std::string("uitk_block_norm: ") + s); };
    if (!u) return bad("null arguments");
    if (u->rows < 0 || u->rows > (int64_t)1 << 31) return bad("the number of rows must be 0 .. 2^31");
    if (u->D < 1 || u->D > 16384) return bad("D must be 1 .. 16384");
    auto is_float = [](int t) { return t >= UITK_T_F32 && t <= UITK_T_BF16; };
    if (!is_float(u->r_type) || (u->y && !is_float(u->y_type)) || (u->gate && !is_float(u->gate_type))) return bad("y, residual and gate must be f32, f16 or bf16");
    if (u->kind != UITK_NORM_LAYER && u->kind != UITK_NORM_RMS) return bad("unknown kind of norm");
    if (!(u->eps >= 0.f)) return bad("eps must not be negative");
    if (u->pre && (u->h_type < UITK_T_F32 || u->h_type > UITK_T_MX4)) return bad("unknown h_type");
    if (!u->y && (u->post || u->gate || u->scale)) return bad("post, gate and scale need a block output y");
    if (!u->y && !u->pre) return bad("nothing to do: neither y nor pre");
    if (u->gate && u->gate_rows < 1) return bad("gate_rows must be positive");
    if (u->rows == 0) return UITK_OK;
    if (!u->residual || (u->y && !u->residual_out) || (u->pre && !u->h)) return bad("null pointer");
    if ((u->y && u->ldy < u->D) || u->ldr < u->D || (u->y && u->ldro < u->D) || (u->gate && u->ldg < u->D) || (u->pre && u->h_type != UITK_T_MX4 && u->ldh < u->D))
        return bad("rows overlap (a leading dimension below D)");
    if (u->pre && u->h_type == UITK_T_MX4 && ((uintptr_t)u->h & 15)) return bad("a packed h must be 16-byte aligned");
    BlockNormArgs a{};
    a.y = u->y; a.y_type = u->y_type; a.ldy = u->ldy; a.r = u->residual; a.r_type = u->r_type; a.ldr = u->ldr; a.rows = u->rows; a.D = u->D;
    a.rms = u->kind == UITK_NORM_RMS; a.eps = u->eps; a.post = u->post != 0; a.post_w = u->post_w; a.post_b = u->post_b;
    a.gate = u->gate; a.gate_type = u->gate_type; a.ldg = u->ldg; a.gate_rows = u->gate_rows; a.scale = u->scale;
    a.ro = u->residual_out; a.ldro = u->ldro; a.pre = u->pre != 0; a.pre_w = u->pre_w; a.pre_b = u->pre_b; a.h = u->h; a.h_type = u->h_type; a.ldh = u->ldh;
    if (a.pre && a.h_type == MT_MX4) { a.h_S = (a.D + MX4_K - 1) / MX4_K; a.h_scales = (char*)a.h + mx4_records(a.rows, a.D) * MX4_CODES; }
    auto ok4 = [](const void* p, int t, int64_t ld) { const int g = t == MT_F32 ? 16 : 8; return (uintptr_t)p % g == 0 && ld % 4 == 0; };
    a.vec = ok4(a.r, a.r_type, a.ldr) && (!a.y || (ok4(a.y, a.y_type, a.ldy) && ok4(a.ro, a.r_type, a.ldro))) && (!a.gate || ok4(a.gate, a.gate_type, a.ldg)) &&
            (!a.pre || a.h_type == MT_MX4 || ok4(a.h, a.h_type, a.ldh));
    const int grid = (int)std::min<int64_t>(a.rows, 1 << 20);
    hipLaunchKernelGGL(block_norm_kernel, dim3(grid), dim3(256), (size_t)((a.D + 127) & ~127) * 4, (hipStream_t)stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(UITK_ERR_HIP, std::string("uitk_block_norm: ") + hipGetErrorString(e));
    return UITK_OK;
}
