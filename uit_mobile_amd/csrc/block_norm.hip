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
};

// ---- L lanes per row (16, 64 or a workgroup of 256), the row in registers: E = 8 NCH elements a lane.
// VEC (D a multiple of 8, everything 16-byte aligned): lane t of the row owns elements 8 (ch L + t) .. + 7 of its NCH chunks, 16-byte accesses.
// Otherwise it owns elements i L + t, one at a time: neighbouring lanes still touch neighbouring elements, whatever the alignment.
template <int L, int NCH, bool VEC> struct BnRow {
    static constexpr int E = 8 * NCH;
    static __device__ __forceinline__ int col(int t, int i) { return VEC ? 8 * ((i >> 3) * L + t) + (i & 7) : i * L + t; }
    mx_u4 raw[NCH][2];                                                      // VEC: what has been asked for and is not converted yet

    __device__ __forceinline__ void ask(const void* base, int type, int64_t off, int t, int D) {
        if constexpr (VEC) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int k = 8 * (c * L + t);
                if (k >= D) continue;
                if (type == MT_F32) {
                    const mx_u4* p = (const mx_u4*)((const float*)base + off + k);
                    raw[c][0] = p[0]; raw[c][1] = p[1];
                } else {
                    raw[c][0] = *(const mx_u4*)((const unsigned short*)base + off + k);
                }
            }
        }
    }
    __device__ __forceinline__ void get(const void* base, int type, int64_t off, int t, int D, float (&v)[E]) {
        if constexpr (VEC) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                if (8 * (c * L + t) >= D) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[8 * c + i] = 0.f;
                } else if (type == MT_F32) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[8 * c + i] = __uint_as_float(raw[c][i >> 2][i & 3]);
                } else if (type == MT_BF16) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) { v[8 * c + 2 * i] = __uint_as_float(raw[c][0][i] << 16); v[8 * c + 2 * i + 1] = __uint_as_float(raw[c][0][i] & 0xffff0000u); }
                } else {
                    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
                    const h8 h = __builtin_bit_cast(h8, raw[c][0]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[8 * c + i] = (float)h[i];
                }
            }
        } else if (type == MT_F32) {
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = i * L + t < D ? ((const float*)base)[off + i * L + t] : 0.f;
        } else if (type == MT_BF16) {
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = i * L + t < D ? __uint_as_float((unsigned)((const unsigned short*)base)[off + i * L + t] << 16) : 0.f;
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = i * L + t < D ? (float)((const _Float16*)base)[off + i * L + t] : 0.f;
        }
    }
    static __device__ __forceinline__ void put(void* base, int type, int64_t off, int t, int D, const float (&v)[E]) {
        if constexpr (VEC) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int k = 8 * (c * L + t);
                if (k >= D) continue;
                if (type == MT_F32) {
                    mx_f4* p = (mx_f4*)((float*)base + off + k);
                    p[0] = mx_f4{v[8 * c], v[8 * c + 1], v[8 * c + 2], v[8 * c + 3]};
                    p[1] = mx_f4{v[8 * c + 4], v[8 * c + 5], v[8 * c + 6], v[8 * c + 7]};
                } else if (type == MT_BF16) {
                    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
                    b8 b;
#pragma unroll
                    for (int i = 0; i < 8; ++i) b[i] = (__bf16)v[8 * c + i];
                    *(b8*)((__bf16*)base + off + k) = b;
                } else {
                    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
                    h8 h;
#pragma unroll
                    for (int i = 0; i < 8; ++i) h[i] = (_Float16)v[8 * c + i];
                    *(h8*)((_Float16*)base + off + k) = h;
                }
            }
        } else if (type == MT_F32) {
#pragma unroll
            for (int i = 0; i < E; ++i) if (i * L + t < D) ((float*)base)[off + i * L + t] = v[i];
        } else if (type == MT_BF16) {
#pragma unroll
            for (int i = 0; i < E; ++i) if (i * L + t < D) ((__bf16*)base)[off + i * L + t] = (__bf16)v[i];
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) if (i * L + t < D) ((_Float16*)base)[off + i * L + t] = (_Float16)v[i];
        }
    }
    // the sum over a row; red: LDS of this sum alone (L = 256)
    static __device__ __forceinline__ float sum(float s, float* red) {
        s = mx_lanes_sum<(L < 64 ? L : 64)>(s);
        if constexpr (L == 256) {
            if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
            __syncthreads();
            s = (red[0] + red[1]) + (red[2] + red[3]);
        }
        return s;
    }
    // v = norm(v) * w + b; elements behind D stay what they are
    static __device__ __forceinline__ void norm(float (&v)[E], int t, const BlockNormArgs& a, const float* w, const float* b, float* red) {
        float mean = 0.f;
        if (!a.rms) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) s += v[i];                          // (zeros behind D)
            mean = sum(s, red) / (float)a.D;
        }
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) { const float d = col(t, i) < a.D ? v[i] - mean : 0.f; q = fmaf(d, d, q); }
        const float rstd = 1.0f / sqrtf(sum(q, red + 4) / (float)a.D + a.eps);
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = (v[i] - mean) * rstd;
        BnRow g;
        float u[E];
        if (w) {
            g.ask(w, MT_F32, 0, t, a.D);
            g.get(w, MT_F32, 0, t, a.D, u);
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] *= u[i];
        }
        if (b) {
            g.ask(b, MT_F32, 0, t, a.D);
            g.get(b, MT_F32, 0, t, a.D, u);
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] += u[i];
        }
    }
};

template <int L, int NCH, bool VEC>
__global__ void __launch_bounds__(256) block_norm_rows_kernel(BlockNormArgs a) {
    typedef BnRow<L, NCH, VEC> Row;
    __shared__ float red[16];                                               // four sums of a workgroup that shares a row
    const int t = threadIdx.x % L;
    const int64_t m = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (L < 256 && m >= a.rows) return;                                     // (whole groups of L lanes leave; L = 256: the grid is the rows)
    Row y, r, g;
    float v[Row::E];
    if (a.y) y.ask(a.y, a.y_type, m * a.ldy, t, a.D);
    r.ask(a.r, a.r_type, m * a.ldr, t, a.D);
    const int64_t goff = a.gate ? (a.gate_rows == 1 ? m : m / a.gate_rows) * a.ldg : 0;
    if (a.gate) g.ask(a.gate, a.gate_type, goff, t, a.D);
    if (a.y) {
        float z[Row::E];
        y.get(a.y, a.y_type, m * a.ldy, t, a.D, z);
        if (a.post) Row::norm(z, t, a, a.post_w, a.post_b, red);
        float u[Row::E];
        if (a.gate) {
            g.get(a.gate, a.gate_type, goff, t, a.D, u);
#pragma unroll
            for (int i = 0; i < Row::E; ++i) z[i] *= u[i];
        }
        if (a.scale) {
            y.ask(a.scale, MT_F32, 0, t, a.D);
            y.get(a.scale, MT_F32, 0, t, a.D, u);
#pragma unroll
            for (int i = 0; i < Row::E; ++i) z[i] *= u[i];
        }
        r.get(a.r, a.r_type, m * a.ldr, t, a.D, v);
#pragma unroll
        for (int i = 0; i < Row::E; ++i) v[i] = Row::col(t, i) < a.D ? v[i] + z[i] : 0.f;
        Row::put(a.ro, a.r_type, m * a.ldro, t, a.D, v);
    } else {
        r.get(a.r, a.r_type, m * a.ldr, t, a.D, v);
    }
    if (!a.pre) return;
    Row::norm(v, t, a, a.pre_w, a.pre_b, red + 8);
    if (a.h_type != MT_MX4) {
        Row::put(a.h, a.h_type, m * a.ldh, t, a.D, v);
    } else if constexpr (VEC) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int k = 8 * (c * L + t);
#pragma unroll
            for (int i = 0; i < 8; ++i) if (k >= a.D) v[8 * c + i] = 0.f;
            unsigned sc;
            const unsigned four = mx4_pack_octets(&v[8 * c], &sc);
            if (k < (int)(a.h_S * MX4_K)) {
                const Mx4Place p = mx4_place(m, k >> 5, a.h_S);
                *(unsigned*)((char*)a.h + p.code + ((k & 31) >> 1)) = four;
                if ((k & 31) == 0) a.h_scales[p.scale] = (char)sc;
            }
        }
    } else {
        // a block is 32 neighbouring lanes' i-th elements (L = 16: two i's of 16 lanes); eight lanes' codes make a dword
        constexpr int PER = L == 16 ? 2 : 1;
#pragma unroll
        for (int i = 0; i < Row::E; i += PER) {
            unsigned mx = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if ((i + j) * L + t >= a.D) v[i + j] = 0.f;
                mx = max(mx, __float_as_uint(v[i + j]) & 0x7fffffffu);
            }
            mx = mx_lanes_max<(L == 16 ? 16 : 32)>(mx);
            const unsigned sc = mx4_scale_byte(mx >> 23);
            const float f = mx4_scale_float(sc);
            const int k = i * L + t;
            const Mx4Place p = mx4_place(m, k >> 5, a.h_S);
            const bool in = k < (int)(a.h_S * MX4_K);
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const unsigned code = sc == 255u ? 0u : __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[i + j], 0.f, f, 0) & 15u;
                const unsigned eight = mx_lanes<8>(code << (4 * (t & 7)), [](unsigned x, unsigned y) { return x | y; });
                if (in && (t & 7) == 0) *(unsigned*)((char*)a.h + p.code + ((k & 31) >> 1) + 8 * j) = eight;
            }
            if (in && (k & 31) == 0) a.h_scales[p.scale] = (char)sc;
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
    hipStream_t s = (hipStream_t)stream;
    auto ok8 = [](const void* p, int t, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % (t == MT_F32 ? 4 : 8) == 0; };
    auto okv = [](const float* p) { return ((uintptr_t)p & 15) == 0; };
    const bool vec8 = a.D % 8 == 0 && ok8(a.r, a.r_type, a.ldr) && (!a.y || (ok8(a.y, a.y_type, a.ldy) && ok8(a.ro, a.r_type, a.ldro))) &&
                      (!a.gate || ok8(a.gate, a.gate_type, a.ldg)) && (!a.pre || a.h_type == MT_MX4 || ok8(a.h, a.h_type, a.ldh)) &&
                      okv(a.scale) && okv(a.post_w) && okv(a.post_b) && okv(a.pre_w) && okv(a.pre_b);
    // lanes per row, chunks of 8 elements per lane; a 4-bit h writes up to its row's end in records of 128
    const int Dp = a.pre && a.h_type == MT_MX4 ? (a.D + 127) & ~127 : a.D;
    auto launch = [&](auto vec_kernel, auto one_kernel, int lanes) {
        const int64_t grid = (a.rows + 256 / lanes - 1) / (256 / lanes);
        if (grid > ((int64_t)1 << 32) / 256 - 1) return false;
        hipLaunchKernelGGL(vec8 ? vec_kernel : one_kernel, dim3((unsigned)grid), dim3(256), 0, s, a);
        return true;
    };
    bool ok;
    if (Dp <= 128) ok = launch(block_norm_rows_kernel<16, 1, true>, block_norm_rows_kernel<16, 1, false>, 16);
    else if (Dp <= 512) ok = launch(block_norm_rows_kernel<64, 1, true>, block_norm_rows_kernel<64, 1, false>, 64);
    else if (Dp <= 1024) ok = launch(block_norm_rows_kernel<64, 2, true>, block_norm_rows_kernel<64, 2, false>, 64);
    else if (Dp <= 2048) ok = launch(block_norm_rows_kernel<256, 1, true>, block_norm_rows_kernel<256, 1, false>, 256);
    else if (Dp <= 4096) ok = launch(block_norm_rows_kernel<256, 2, true>, block_norm_rows_kernel<256, 2, false>, 256);
    else if (Dp <= 8192) ok = launch(block_norm_rows_kernel<256, 4, true>, block_norm_rows_kernel<256, 4, false>, 256);
    else ok = launch(block_norm_rows_kernel<256, 8, true>, block_norm_rows_kernel<256, 8, false>, 256);
    if (!ok) return set_error(UITK_ERR_UNSUPPORTED, "uitk_block_norm: more rows than one launch takes");
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(UITK_ERR_HIP, std::string("uitk_block_norm: ") + hipGetErrorString(e));
    return UITK_OK;
}
