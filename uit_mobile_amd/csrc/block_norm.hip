// block_norm.hip -- the seam between two blocks of a transformer in one pass over the residual stream:
//
//     z  = post(y)                      norm behind the block (optional)
//     r' = r + gate * scale * z         gate: a row per sequence or per token (optional); scale: one gain per channel (LayerScale; optional)
//     h  = pre(r')                      norm in front of the next block (optional), 32, 16 or 4 bits (mx4_dev.h)
//
// post / pre: LayerNorm ((v - mean) / sqrt(var + eps)) or root mean square (v / sqrt(mean(v^2) + eps)), then gain and offset (each optional).
// All of it in fp32 from the inputs to the one rounding of each output; h is taken from the unrounded r'.  (models/uit.py:245-248: Block.forward,
// whose LayerScale is :78-85.)
#include <hip/hip_runtime.h>
#include <stdint.h>

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

// ---- L lanes per row (16, 64 or a whole workgroup), the row in registers: lane t owns elements 8 (c L + t) .. + 7 of its NCH chunks, 16 bytes
// an access whatever the alignment; the chunk that D ends in goes element by element.  WIDE: the operand may be fp32 (a chunk is two
// accesses); 16-bit operands need half the registers.
template <int L, int NCH, bool WIDE> struct BnAsked {
    mx_u4 raw[NCH][WIDE ? 2 : 1];                                           // asked for, not converted yet

    __device__ __forceinline__ void ask(const void* base, int type, int64_t off, int t, int D) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int k = 8 * (c * L + t);
            if (k >= D) continue;
            if (WIDE && type == MT_F32) {
                const float* p = (const float*)base + off + k;
                if (k + 8 <= D) {
                    raw[c][0] = ((const mx_u4u*)p)[0];
                    raw[c][WIDE] = ((const mx_u4u*)p)[1];
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) raw[c][WIDE ? i >> 2 : 0][i & 3] = k + i < D ? __float_as_uint(p[i]) : 0u;
                }
            } else {
                const unsigned short* p = (const unsigned short*)base + off + k;
                if (k + 8 <= D) {
                    raw[c][0] = *(const mx_u4u*)p;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) raw[c][0][i] = (k + 2 * i < D ? (unsigned)p[2 * i] : 0u) | (k + 2 * i + 1 < D ? (unsigned)p[2 * i + 1] << 16 : 0u);
                }
            }
        }
    }
    // zeros behind D
    __device__ __forceinline__ void get(int type, int t, int D, float (&v)[8 * NCH]) const {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            if (8 * (c * L + t) >= D) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[8 * c + i] = 0.f;
            } else if (WIDE && type == MT_F32) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[8 * c + i] = __uint_as_float(raw[c][WIDE ? i >> 2 : 0][i & 3]);
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
    }
};

template <int L, int NCH> struct BnRow {
    static constexpr int E = 8 * NCH;
    static __device__ __forceinline__ int col(int t, int i) { return 8 * ((i >> 3) * L + t) + (i & 7); }
    // (streamed past the caches: 16128 x 768 fp32 43.0 / 40.5 us, 2 to 3 % of wider rows, and no loss where the next kernel reads it at once)
    static __device__ __forceinline__ void put(void* base, int type, int64_t off, int t, int D, const float (&v)[E]) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int k = 8 * (c * L + t);
            if (k >= D) continue;
            if (type == MT_F32) {
                float* p = (float*)base + off + k;
                if (k + 8 <= D) {
                    __builtin_nontemporal_store(mx_f4{v[8 * c], v[8 * c + 1], v[8 * c + 2], v[8 * c + 3]}, (mx_f4u*)p);
                    __builtin_nontemporal_store(mx_f4{v[8 * c + 4], v[8 * c + 5], v[8 * c + 6], v[8 * c + 7]}, (mx_f4u*)p + 1);
                } else {
#pragma unroll
                    for (int i = 0; i < 7; ++i) if (k + i < D) p[i] = v[8 * c + i];
                }
            } else if (type == MT_BF16) {
                typedef __bf16 b8 __attribute__((ext_vector_type(8), aligned(2)));
                b8 b;
#pragma unroll
                for (int i = 0; i < 8; ++i) b[i] = (__bf16)v[8 * c + i];
                __bf16* p = (__bf16*)base + off + k;
                if (k + 8 <= D) __builtin_nontemporal_store(b, (b8*)p);
                else {
#pragma unroll
                    for (int i = 0; i < 7; ++i) if (k + i < D) p[i] = b[i];
                }
            } else {
                typedef _Float16 h8 __attribute__((ext_vector_type(8), aligned(2)));
                h8 h;
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] = (_Float16)v[8 * c + i];
                _Float16* p = (_Float16*)base + off + k;
                if (k + 8 <= D) __builtin_nontemporal_store(h, (h8*)p);
                else {
#pragma unroll
                    for (int i = 0; i < 7; ++i) if (k + i < D) p[i] = h[i];
                }
            }
        }
    }
    // the sum over a row; red: LDS of this sum alone (L > 64)
    static __device__ __forceinline__ float sum(float s, float* red) {
        s = mx_lanes_sum<(L < 64 ? L : 64)>(s);
        if constexpr (L > 64) {
            if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
            __syncthreads();
            s = 0.f;
#pragma unroll
            for (int i = 0; i < L / 64; ++i) s += red[i];
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
        const float rstd = 1.0f / sqrtf(sum(q, red + L / 64) / (float)a.D + a.eps);
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = (v[i] - mean) * rstd;
        BnAsked<L, NCH, true> g;
        float u[E];
        if (w) {
            g.ask(w, MT_F32, 0, t, a.D);
            g.get(MT_F32, t, a.D, u);
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] *= u[i];
        }
        if (b) {
            g.ask(b, MT_F32, 0, t, a.D);
            g.get(MT_F32, t, a.D, u);
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] += u[i];
        }
    }
};

// One pass: y, the residual and a per-token gate are asked for at once and the row never leaves the registers again, so the kernel moves what it
// has to and is bound by HBM: 16 x 4096 rows of 2048 bf16, add + RMS norm 5.9 TB/s; 64 x 252 rows of 768 fp32, scale + add + LayerNorm 40 us, 4.9 TB/s;
// 8 x 4096 rows of 4096 bf16, both norms, gate and scale 235 us, 4.6 TB/s (its five parameter rows pass L1 for every row).  Mean and variance are
// two sums over the row (the variance of what is left after the mean: no cancellation against a large mean).
template <int L, int NCH, bool Y32, bool R32>
__global__ void __launch_bounds__(L < 256 ? 256 : L) block_norm_rows_kernel(BlockNormArgs a) {
    typedef BnRow<L, NCH> Row;
    constexpr int RPW = L < 256 ? 256 / L : 1;                              // rows of a workgroup
    __shared__ float red[L < 64 ? 1 : 4 * L / 64];                          // four sums of a workgroup that shares a row
    const int t = threadIdx.x % L;
    const int64_t m = (int64_t)blockIdx.x * RPW + threadIdx.x / L;
    if (RPW > 1 && m >= a.rows) return;                                     // (whole groups of L lanes leave; one row a workgroup: the grid is the rows)
    float v[Row::E];
    BnAsked<L, NCH, R32> r;
    if (a.y) {
        float z[Row::E], u[Row::E];
        BnAsked<L, NCH, true> g;
        {
            BnAsked<L, NCH, Y32> y;
            y.ask(a.y, a.y_type, m * a.ldy, t, a.D);
            r.ask(a.r, a.r_type, m * a.ldr, t, a.D);
            y.get(a.y_type, t, a.D, z);
        }
        if (a.gate) g.ask(a.gate, a.gate_type, (a.gate_rows == 1 ? m : m / a.gate_rows) * a.ldg, t, a.D);
        if (a.post) Row::norm(z, t, a, a.post_w, a.post_b, red);
        if (a.gate) {
            g.get(a.gate_type, t, a.D, u);
#pragma unroll
            for (int i = 0; i < Row::E; ++i) z[i] *= u[i];
        }
        if (a.scale) {
            g.ask(a.scale, MT_F32, 0, t, a.D);
            g.get(MT_F32, t, a.D, u);
#pragma unroll
            for (int i = 0; i < Row::E; ++i) z[i] *= u[i];
        }
        r.get(a.r_type, t, a.D, v);
#pragma unroll
        for (int i = 0; i < Row::E; ++i) v[i] = Row::col(t, i) < a.D ? v[i] + z[i] : 0.f;
        Row::put(a.ro, a.r_type, m * a.ldro, t, a.D, v);
    } else {
        r.ask(a.r, a.r_type, m * a.ldr, t, a.D);
        r.get(a.r_type, t, a.D, v);
    }
    if (!a.pre) return;
    Row::norm(v, t, a, a.pre_w, a.pre_b, red + 2 * (L / 64));
    if (a.h_type != MT_MX4) {
        Row::put(a.h, a.h_type, m * a.ldh, t, a.D, v);
        return;
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int k = 8 * (c * L + t);
#pragma unroll
        for (int i = 0; i < 8; ++i) if (k + i >= a.D) v[8 * c + i] = 0.f;
        unsigned sc;
        const unsigned four = mx4_pack_octets(&v[8 * c], &sc);
        if (k < (int)(a.h_S * MX4_K)) {
            const Mx4Place p = mx4_place(m, k >> 5, a.h_S);
            *(unsigned*)((char*)a.h + p.code + ((k & 31) >> 1)) = four;
            if ((k & 31) == 0) a.h_scales[p.scale] = (char)sc;
        }
    }
}

template <int L, int NCH>
static bool bn_launch(const BlockNormArgs& a, hipStream_t s) {
    constexpr int THREADS = L < 256 ? 256 : L, RPW = THREADS / L;
    const int64_t grid = (a.rows + RPW - 1) / RPW;
    if (grid > ((int64_t)1 << 32) / THREADS - 1) return false;              // a launch counts its threads in 32 bits
    const bool y32 = a.y && a.y_type == MT_F32, r32 = a.r_type == MT_F32;
    auto kernel = y32 ? (r32 ? block_norm_rows_kernel<L, NCH, true, true> : block_norm_rows_kernel<L, NCH, true, false>)
                      : (r32 ? block_norm_rows_kernel<L, NCH, false, true> : block_norm_rows_kernel<L, NCH, false, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(THREADS), 0, s, a);
    return true;
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
    auto off = [](const void* p, int t) { return (uintptr_t)p % (t == UITK_T_F32 ? 4 : 2) != 0; };
    if (off(u->residual, u->r_type) || (u->y && (off(u->y, u->y_type) || off(u->residual_out, u->r_type))) || (u->gate && off(u->gate, u->gate_type)) ||
        (u->pre && u->h_type != UITK_T_MX4 && off(u->h, u->h_type)) || off(u->scale, 0) || off(u->post_w, 0) || off(u->post_b, 0) || off(u->pre_w, 0) || off(u->pre_b, 0))
        return bad("a pointer is not aligned to its elements");
    BlockNormArgs a{};
    a.y = u->y; a.y_type = u->y_type; a.ldy = u->ldy; a.r = u->residual; a.r_type = u->r_type; a.ldr = u->ldr; a.rows = u->rows; a.D = u->D;
    a.rms = u->kind == UITK_NORM_RMS; a.eps = u->eps; a.post = u->post != 0; a.post_w = u->post_w; a.post_b = u->post_b;
    a.gate = u->gate; a.gate_type = u->gate_type; a.ldg = u->ldg; a.gate_rows = u->gate_rows; a.scale = u->scale;
    a.ro = u->residual_out; a.ldro = u->ldro; a.pre = u->pre != 0; a.pre_w = u->pre_w; a.pre_b = u->pre_b; a.h = u->h; a.h_type = u->h_type; a.ldh = u->ldh;
    if (a.pre && a.h_type == MT_MX4) { a.h_S = (a.D + MX4_K - 1) / MX4_K; a.h_scales = (char*)a.h + mx4_records(a.rows, a.D) * MX4_CODES; }
    hipStream_t s = (hipStream_t)stream;
    // Lanes per row, chunks of 8 elements per lane (a 4-bit h writes up to its row's end in records of 128).  A wave per row needs no barrier and
    // keeps 12 to 32 rows of a CU on their way; a workgroup per row is what the registers ask for beyond 2048.  64 x 1024 rows of 1500, everything
    // on, 64 lanes x 3 chunks / 256 x 1: 288 / 406 us; of 2048: 263 / 278; 8 x 4096 rows of 4096, 128 x 4 / 256 x 2: 260 / 246; one row of 2048: 7.0 / 3.9.
    // By the width alone: a row's result does not depend on how many others there are.
    const int Dp = a.pre && a.h_type == MT_MX4 ? (a.D + 127) & ~127 : a.D;
    const bool ok = Dp <= 128    ? bn_launch<16, 1>(a, s)
                    : Dp <= 512  ? bn_launch<64, 1>(a, s)
                    : Dp <= 1024 ? bn_launch<64, 2>(a, s)
                    : Dp <= 1536 ? bn_launch<64, 3>(a, s)
                    : Dp <= 2048 ? bn_launch<64, 4>(a, s)
                    : Dp <= 4096 ? bn_launch<256, 2>(a, s)
                    : Dp <= 8192 ? bn_launch<512, 2>(a, s)
                                 : bn_launch<1024, 2>(a, s);
    if (!ok) return set_error(UITK_ERR_UNSUPPORTED, "uitk_block_norm: more rows than one launch takes");
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(UITK_ERR_HIP, std::string("uitk_block_norm: ") + hipGetErrorString(e));
    return UITK_OK;
}
