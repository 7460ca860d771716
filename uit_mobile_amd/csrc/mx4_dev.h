// mx4_dev.h -- microscaled 4-bit floating point (OCP MXFP4) on gfx950: the packed layout and the device code that reads and writes it.
//
// A row of K elements is cut into blocks of 32; a block holds 32 e2m1 codes (4 bits: +-{0, .5, 1, 1.5, 2, 3, 4, 6}) and one e8m0 scale
// (a byte b: 2^(b - 127); 255: NaN, the whole block is NaN).  Packed matrices keep the order in which
// v_mfma_scale_f32_32x32x64_f8f6f4 takes its operands: lane l of a wave holds row l % 32 of a 32 x 64 fragment, elements
// 32 (l / 32) .. + 31 -- exactly one block, 16 bytes -- and supplies that block's scale.  A RECORD is 64 rows x 128 elements:
//     codes   4096 B = [row tile rt 0..1][k half kh 0..1][lane 0..63][16 B], element j of a block in nibble j % 2 of byte j / 2
//     scales   256 B = [lane 0..63][byte 2 rt + kh]: one dword per lane serves the record's four fragments (op_sel picks the byte)
// A packed matrix of `rows` x `K`: the codes of all records [rows / 64][K / 128], then all their scales in the same order (both
// counts rounded up).  Elements behind K are code 0 under a finite scale, so they add nothing to a product; rows behind `rows` may
// hold anything: a product's rows and columns do not mix, and what they yield is not stored.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace uitk {

constexpr int MX4_ROWS = 64, MX4_K = 128, MX4_CODES = 4096, MX4_SCALES = 256;

enum Mx4Type { MT_F32 = 0, MT_F16 = 1, MT_BF16 = 2, MT_MX4 = 3 };          // == uitk_type (include/uitk.h)

__host__ __device__ inline int64_t mx4_records(int64_t rows, int64_t K) { return ((rows + MX4_ROWS - 1) / MX4_ROWS) * ((K + MX4_K - 1) / MX4_K); }
__host__ __device__ inline int64_t mx4_bytes(int64_t rows, int64_t K) { return mx4_records(rows, K) * (MX4_CODES + MX4_SCALES); }

typedef int mx_i4 __attribute__((ext_vector_type(4)));
typedef int mx_i8 __attribute__((ext_vector_type(8)));
typedef float mx_f2 __attribute__((ext_vector_type(2)));
typedef float mx_f4 __attribute__((ext_vector_type(4)));
typedef float mx_f16 __attribute__((ext_vector_type(16)));
typedef _Float16 mx_h2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_b2 __attribute__((ext_vector_type(2)));
typedef unsigned mx_u4 __attribute__((ext_vector_type(4)));
typedef unsigned mx_u2 __attribute__((ext_vector_type(2)));
// the same at the alignment of their elements: global memory takes 16-byte accesses at any address, so a row that starts anywhere (an odd
// width, a slice) still goes 16 bytes a lane (quantize 32768 x 4095 bf16, element by element / like this: 453 / 102 us; 4096 wide: 72)
typedef unsigned mx_u4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned mx_u2u __attribute__((ext_vector_type(2), aligned(2)));
typedef float mx_f4u __attribute__((ext_vector_type(4), aligned(4)));

struct Mx4Block { mx_i4 codes; unsigned scale; };                          // 32 elements: 16 bytes of codes, the scale byte

// scale byte of a block whose largest magnitude has the float32 exponent field e (255: the block holds an infinity or a NaN)
__device__ __forceinline__ unsigned mx4_scale_byte(unsigned e) { return e == 255u ? 255u : (e > 2u ? e - 2u : 0u); }
// 2^(b - 127) as a float; b = 0 is the subnormal 2^-127, which the conversions take as what it is
__device__ __forceinline__ float mx4_scale_float(unsigned b) { return __uint_as_float(b == 0u ? 0x00400000u : b << 23); }

// ---- 32 elements of a row in registers, by type
template <typename T> struct Mx4Src;

template <> struct Mx4Src<float> {
    float v[32];
    __device__ __forceinline__ void load(const float* p, int n) {                           // n valid elements
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (4 * i + 4 <= n) {
                const mx_f4 t = *(const mx_f4u*)(p + 4 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * i + j] = t[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * i + j] = 4 * i + j < n ? p[4 * i + j] : 0.f;
            }
        }
    }
    __device__ __forceinline__ Mx4Block pack() const {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        Mx4Block b;
        b.scale = mx4_scale_byte(m >> 23);
        const float s = mx4_scale_float(b.scale);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            unsigned w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[8 * d + 0], v[8 * d + 1], s, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[8 * d + 2], v[8 * d + 3], s, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[8 * d + 4], v[8 * d + 5], s, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[8 * d + 6], v[8 * d + 7], s, 3);
            b.codes[d] = b.scale == 255u ? 0 : (int)w;
        }
        return b;
    }
};

// the two 16-bit types: 16 dwords of two elements each
template <typename T> struct Mx4Src16 {
    unsigned v[16];
    __device__ __forceinline__ void load(const T* p, int n) {
        const unsigned short* q = (const unsigned short*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (8 * i + 8 <= n) {
                const mx_u4 t = *(const mx_u4u*)(q + 8 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * i + j] = t[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int e = 8 * i + 2 * j;
                    v[4 * i + j] = (e < n ? (unsigned)q[e] : 0u) | (e + 1 < n ? (unsigned)q[e + 1] << 16 : 0u);
                }
            }
        }
    }
    __device__ __forceinline__ unsigned amax() const {                                      // the largest |element|'s 15 bits
        typedef unsigned short us2 __attribute__((ext_vector_type(2)));
        us2 m = {0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, v[i] & 0x7fff7fffu));
        return max((unsigned)m[0], (unsigned)m[1]);
    }
};
template <> struct Mx4Src<_Float16> : Mx4Src16<_Float16> {
    __device__ __forceinline__ Mx4Block pack() const {
        Mx4Block b;
        b.scale = mx4_scale_byte(__float_as_uint((float)__builtin_bit_cast(_Float16, (unsigned short)amax())) >> 23);
        const float s = mx4_scale_float(b.scale);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            unsigned w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(mx_h2, v[4 * d + 0]), s, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(mx_h2, v[4 * d + 1]), s, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(mx_h2, v[4 * d + 2]), s, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(mx_h2, v[4 * d + 3]), s, 3);
            b.codes[d] = b.scale == 255u ? 0 : (int)w;
        }
        return b;
    }
};
template <> struct Mx4Src<__bf16> : Mx4Src16<__bf16> {
    __device__ __forceinline__ Mx4Block pack() const {
        Mx4Block b;
        b.scale = mx4_scale_byte(amax() >> 7);
        const float s = mx4_scale_float(b.scale);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            unsigned w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(mx_b2, v[4 * d + 0]), s, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(mx_b2, v[4 * d + 1]), s, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(mx_b2, v[4 * d + 2]), s, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(mx_b2, v[4 * d + 3]), s, 3);
            b.codes[d] = b.scale == 255u ? 0 : (int)w;
        }
        return b;
    }
};

// ---- 8 elements of a row, four neighbouring lanes a block
template <typename T> struct Mx4Oct;
template <> struct Mx4Oct<float> {
    mx_f4 v[2];
    __device__ __forceinline__ void load(const float* p, int n) {                           // n valid elements (0 or less: none)
        if (n >= 8) { v[0] = ((const mx_f4u*)p)[0]; v[1] = ((const mx_f4u*)p)[1]; return; }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i >> 2][i & 3] = i < n ? p[i] : 0.f;
    }
    __device__ __forceinline__ unsigned exponent() const;                                   // of the block's largest magnitude, as a float32 exponent field
    __device__ __forceinline__ unsigned pack(float s) const {
        unsigned w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0][0], v[0][1], s, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0][2], v[0][3], s, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[1][0], v[1][1], s, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[1][2], v[1][3], s, 3);
    }
};
template <typename T> struct Mx4Oct16 {
    mx_u4 v;
    __device__ __forceinline__ void load(const T* p, int n) {
        if (n >= 8) { v = *(const mx_u4u*)p; return; }
        const unsigned short* q = (const unsigned short*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (2 * i < n ? (unsigned)q[2 * i] : 0u) | (2 * i + 1 < n ? (unsigned)q[2 * i + 1] << 16 : 0u);
    }
    __device__ __forceinline__ unsigned amax() const;                                       // the 15 bits of the block's largest magnitude
};
template <> struct Mx4Oct<_Float16> : Mx4Oct16<_Float16> {
    __device__ __forceinline__ unsigned exponent() const { return __float_as_uint((float)__builtin_bit_cast(_Float16, (unsigned short)amax())) >> 23; }
    __device__ __forceinline__ unsigned pack(float s) const {
        typedef _Float16 h8 __attribute__((ext_vector_type(8)));
        const h8 h = __builtin_bit_cast(h8, v);
        unsigned w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, mx_h2{h[0], h[1]}, s, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, mx_h2{h[2], h[3]}, s, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, mx_h2{h[4], h[5]}, s, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, mx_h2{h[6], h[7]}, s, 3);
    }
};
template <> struct Mx4Oct<__bf16> : Mx4Oct16<__bf16> {
    __device__ __forceinline__ unsigned exponent() const { return amax() >> 7; }
    __device__ __forceinline__ unsigned pack(float s) const {
        typedef __bf16 b8 __attribute__((ext_vector_type(8)));
        const b8 h = __builtin_bit_cast(b8, v);
        unsigned w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, mx_b2{h[0], h[1]}, s, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, mx_b2{h[2], h[3]}, s, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, mx_b2{h[4], h[5]}, s, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, mx_b2{h[6], h[7]}, s, 3);
    }
};

// ---- reductions over neighbouring lanes without LDS: DPP within 16 lanes, row swaps beyond
template <int CTRL> __device__ __forceinline__ unsigned mx_dpp(unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140;
// every lane gets the result over its group of N lanes (4, 8, 16, 32 or 64)
template <int N, typename F> __device__ __forceinline__ unsigned mx_lanes(unsigned v, F f) {
    static_assert(N >= 4 && N <= 64 && (N & (N - 1)) == 0, "");
    v = f(v, mx_dpp<DPP_XOR1>(v));
    v = f(v, mx_dpp<DPP_XOR2>(v));
    if constexpr (N >= 8) v = f(v, mx_dpp<DPP_HALF_MIRROR>(v));
    if constexpr (N >= 16) v = f(v, mx_dpp<DPP_MIRROR>(v));
    if constexpr (N >= 32) { const auto t = __builtin_amdgcn_permlane16_swap(v, v, false, false); v = f(t[0], t[1]); }
    if constexpr (N >= 64) { const auto t = __builtin_amdgcn_permlane32_swap(v, v, false, false); v = f(t[0], t[1]); }
    return v;
}
template <int N> __device__ __forceinline__ unsigned mx_lanes_max(unsigned v) { return mx_lanes<N>(v, [](unsigned a, unsigned b) { return max(a, b); }); }
template <int N> __device__ __forceinline__ float mx_lanes_sum(float v) {
    return __uint_as_float(mx_lanes<N>(__float_as_uint(v), [](unsigned a, unsigned b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}

__device__ __forceinline__ unsigned Mx4Oct<float>::exponent() const {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i >> 2][i & 3]) & 0x7fffffffu);
    return mx_lanes_max<4>(m) >> 23;
}
template <typename T> __device__ __forceinline__ unsigned Mx4Oct16<T>::amax() const {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    us2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) { const unsigned a = v[i] & 0x7fff7fffu; m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, a)); }
    return mx_lanes_max<4>(max((unsigned)m[0], (unsigned)m[1]));
}

// ---- packing inside an epilogue: 8 neighbouring lanes hold 4 consecutive elements of a block each.  -> the lane's two bytes of codes
// and the block's scale byte (the same on the 8 lanes)
__device__ __forceinline__ unsigned mx4_pack_quads(const float (&v)[4], unsigned* scale) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = mx_lanes_max<8>(m);
    const unsigned b = mx4_scale_byte(m >> 23);
    const float s = mx4_scale_float(b);
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
    *scale = b;
    return b == 255u ? 0u : w & 0xffffu;
}

// the same for 4 neighbouring lanes with 8 consecutive elements each -> the lane's four bytes of codes
__device__ __forceinline__ unsigned mx4_pack_octets(const float* v, unsigned* scale) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = mx_lanes_max<4>(m);
    const unsigned b = mx4_scale_byte(m >> 23);
    const float s = mx4_scale_float(b);
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
    *scale = b;
    return b == 255u ? 0u : w;
}

// where block kb (32 elements) of row r lives in a packed matrix of S records per row group
struct Mx4Place { int64_t code, scale; };                                   // byte offsets into the codes / the scales
__device__ __forceinline__ Mx4Place mx4_place(int64_t r, int64_t kb, int64_t S) {
    const int64_t rec = (r >> 6) * S + (kb >> 2);
    const int rt = (int)(r >> 5) & 1, kh = (int)(kb >> 1) & 1, lane = (int)(r & 31) + 32 * (int)(kb & 1);
    return Mx4Place{rec * MX4_CODES + (2 * rt + kh) * 1024 + lane * 16, rec * MX4_SCALES + lane * 4 + 2 * rt + kh};
}

// D = A (32 x 64) . B (64 x 32) + C, both operands 4-bit; SA / SB: which byte of the lane's scale dword belongs to this fragment.
// Lane l, register r holds D[8 (r / 4) + 4 (l / 32) + r % 4][l % 32].  (The 32 x 32 x 64 form: 9.4 PFLOP/s over the card against 5.4
// for 16 x 16 x 128, both from registers, one wave per SIMD.)
template <int SA, int SB>
__device__ __forceinline__ mx_f16 mx4_mfma(mx_i4 a, mx_i4 b, mx_f16 c, int sa, int sb) {
    const mx_i8 a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, SA, sa, SB, sb);
}

// GELU, x Phi(x), with Phi(x) = 1 / (1 + exp(-x P(x^2))): x P(x^2) is the logit of Phi, an odd function; P a polynomial of degree 6 that
// minimises the largest error of x Phi on [0, 5.5]: 7e-8 there, evaluated in fp32 2.3e-7 max(1, |y|).  Beyond, P stays at its last value:
// the exponent keeps growing, so the tails go to x and to 0.  An absolute error: beside y itself it is 3e-4 at x = -4, 4 % at -5 and 42 % at
// -5.5 (where y is -1e-7; 0.5 x (1 + erf(x / sqrt 2)) in fp32: 3e-4, 4 %, 57 %).  12 instructions, two of them transcendental (erff: ~40); the
// coefficients carry the factor -log2(e).
__device__ __forceinline__ float mx4_gelu(float x) {
    const float u = fminf(x * x, 30.25f);
    float p = -5.282749793e-09f;
    p = fmaf(p, u, 3.889133779e-07f);
    p = fmaf(p, u, -1.152892673e-05f);
    p = fmaf(p, u, 1.601013355e-04f);
    p = fmaf(p, u, 9.235717152e-05f);
    p = fmaf(p, u, -1.048319191e-01f);
    p = fmaf(p, u, -2.302212000e+00f);
    return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(p * x));
}

}  // namespace uitk
