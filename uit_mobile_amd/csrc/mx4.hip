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
#include <type_traits>

#include "../../include/uitk.h"
#include "mx4_dev.h"
#include "mx4_plan.h"

namespace uitk {

int set_error(int code, const std::string& msg);                          // api.cpp: the thread's uitk_last_error text

// ------------------------------------------------------------------------------------------------------------------- quantize
// One wave per record; 16 lanes share a row, a lane rounds 8 of its elements and four neighbours a block: a wave reads 128 consecutive elements
// of four rows at a time, whatever their alignment, and finds a block's maximum in two lane exchanges.  (A whole block per lane needs no
// exchange, but its 16-byte reads lie 64 or 128 bytes apart: 32768 x 4096 bf16 75 / 72 us (4.7 TB/s), 16384 x 4096 fp32 82 / 58, 32768 x 4095 bf16 137 / 102.)
// SPLIT: the four waves of a workgroup share a record, 16 rows each: few records are a matter of latency.
template <typename T, bool SPLIT>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(const T* __restrict__ x, int64_t rows, int64_t K, int64_t ld, int64_t R, int64_t S,
                                                           char* __restrict__ codes, char* __restrict__ scales) {
    __shared__ unsigned char sc[SPLIT ? 1 : 4][MX4_SCALES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, kb = l16 >> 2;       // the lane's block: half kb / 2, group kb % 2
    const int64_t rec = SPLIT ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
    if (rec >= R * S) return;
    const int64_t rg = rec / S, s = rec - rg * S, k = s * MX4_K + l16 * 8;
    const int n = (int)min((int64_t)8, K - k);                              // (negative: no element of the row)
    const int nrow = (int)min((int64_t)MX4_ROWS, rows - rg * MX4_ROWS);
    const T* p = x + (rg * MX4_ROWS + (lane >> 4)) * ld + k;
    char* c = codes + rec * MX4_CODES + (kb >> 1) * 1024 + ((kb & 1) * 32 + (lane >> 4)) * 16 + (l16 & 3) * 4;
    unsigned char* my = sc[SPLIT ? 0 : wave];
    constexpr int BATCH = sizeof(T) == 4 || SPLIT ? 4 : 8;                  // reads on their way at a time
#pragma unroll
    for (int b0 = 0; b0 < (SPLIT ? 4 : 16); b0 += BATCH) {
        const int i0 = SPLIT ? 4 * wave : b0;
        if (4 * i0 >= nrow) break;                                          // (rows behind the matrix are left as they are)
        Mx4Oct<T> v[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) v[i].load(p + (i0 + i) * 4 * ld, (i0 + i) * 4 + (lane >> 4) < nrow ? n : 0);
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int r = (i0 + i) * 4;                                     // + lane / 16: the row of the record
            const unsigned b = mx4_scale_byte(v[i].exponent());
            const unsigned w = v[i].pack(mx4_scale_float(b));
            *(unsigned*)(c + (r >> 5) * 2048 + (r & 31) * 16) = b == 255u ? 0u : w;
            if ((l16 & 3) == 0) my[((kb & 1) * 32 + (r & 31) + (lane >> 4)) * 4 + 2 * (r >> 5) + (kb >> 1)] = (unsigned char)b;
        }
    }
    if constexpr (SPLIT) {
        __syncthreads();
        if (wave) return;
    } else {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");              // (LDS serves a wave in order: what is left to do is to keep the compiler's)
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    *(unsigned*)(scales + rec * MX4_SCALES + lane * 4) = *(const unsigned*)&my[lane * 4];
}

// One wave per record here too; a lane turns the codes of 16 bytes of output into them, so that neighbouring lanes store neighbouring
// bytes of a row (a whole block per lane stored 16-byte pieces 64 or 128 bytes apart; 32768 x 4096 bf16: 56 us, 6.1 TB/s).
template <typename T, bool STREAM>
__global__ void __launch_bounds__(256) mx4_dequantize_kernel(const char* __restrict__ codes, const char* __restrict__ scales, int64_t rows, int64_t K, int64_t ld,
                                                             int64_t R, int64_t S, T* __restrict__ x) {
    constexpr int P = 16 / sizeof(T), LPR = MX4_K / P, RPI = 64 / LPR;      // elements of a lane, lanes of a row, rows at a time
    typedef T TP __attribute__((ext_vector_type(P)));
    typedef T TPu __attribute__((ext_vector_type(P), aligned(sizeof(T))));
    const int lane = threadIdx.x & 63, lr = lane % LPR, row0 = lane / LPR, kb = lr * P >> 5;          // the lane's block: half kb / 2, group kb % 2
    const int64_t rec = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (rec >= R * S) return;
    const int64_t rg = rec / S, s = rec - rg * S, k = s * MX4_K + lr * P;
    const int n = (int)min((int64_t)P, K - k), nrow = (int)min((int64_t)MX4_ROWS, rows - rg * MX4_ROWS);
    const char* c = codes + rec * MX4_CODES + (kb >> 1) * 1024 + (kb & 1) * 512 + ((lr * P & 31) >> 1);
    const unsigned char* sc = (const unsigned char*)scales + rec * MX4_SCALES + (kb & 1) * 128 + (kb >> 1);
    if (n <= 0) return;
    constexpr int BATCH = 8;                                                // rows asked for at a time
#pragma unroll
    for (int i0 = 0; i0 < MX4_ROWS / RPI; i0 += BATCH) {
        if (i0 * RPI >= nrow) return;
        unsigned w[BATCH], b[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int r = (i0 + i) * RPI + row0;
            const char* q = c + (r >> 5) * 2048 + (r & 31) * 16;
            w[i] = P == 8 ? *(const unsigned*)q : *(const unsigned short*)q;
            b[i] = sc[(r & 31) * 4 + 2 * (r >> 5)];
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int r = (i0 + i) * RPI + row0;
            const float f = mx4_scale_float(b[i]);
            const mx_f2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], f, 1),
                                __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], f, 3)};
            TP t;
#pragma unroll
            for (int j = 0; j < P; ++j) t[j] = (T)(b[i] == 255u ? __uint_as_float(0x7fc00000u) : v[j >> 1][j & 1]);
            if (r >= nrow) continue;
            T* o = x + (rg * MX4_ROWS + r) * ld + k;
            if (n == P) {
                if constexpr (STREAM) __builtin_nontemporal_store(t, (TPu*)o);
                else *(TPu*)o = t;
            } else {
#pragma unroll
                for (int j = 0; j < P - 1; ++j) if (j < n) o[j] = t[j];
            }
        }
    }
}

// --------------------------------------------------------------------------------------------------------------------- linear
struct Mx4LinearArgs {
    const void* x; int64_t M, K, ldx; int x_type;                           // x_type MT_MX4: x = codes of a packed matrix, x_scales its scales
    const char* x_scales;
    const char* w; const char* w_scales;                                    // packed [N, K]
    int64_t N, S;                                                           // S = records along K
    const float* bias;
    int act;                                                                // 0 none, 1 ReLU, 2 GELU (mx4_gelu)
    const void* residual; int64_t ldr;                                      // of the output's type, added last
    void* out; int64_t ldo; int out_type;                                   // MT_MX4: out = codes, out_scales its scales
    char* out_scales; int64_t out_S;
    unsigned ngroups; int chains;                                           // rows kernel: column groups; waves that share K (not more than its records)
};

__device__ __forceinline__ mx_f4 mx4_bias4(const Mx4LinearArgs& a, int64_t n) {
    mx_f4 b = {0.f, 0.f, 0.f, 0.f};
    if (a.bias && n + 4 <= a.N) b = *(const mx_f4u*)(a.bias + n);
    else if (a.bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i) if (n + i < a.N) b[i] = a.bias[n + i];
    }
    return b;
}

// four consecutive outputs of a type: add a residual, round once, store
template <int OUT> struct Mx4Out;
template <> struct Mx4Out<MT_F32> {
    typedef float T;
    static __device__ __forceinline__ void add4(float (&v)[4], const float* r) { const mx_f4 t = *(const mx_f4u*)r; v[0] += t[0]; v[1] += t[1]; v[2] += t[2]; v[3] += t[3]; }
    static __device__ __forceinline__ void put4(float* o, const float (&v)[4]) { *(mx_f4u*)o = mx_f4{v[0], v[1], v[2], v[3]}; }
    static __device__ __forceinline__ void stream4(float* o, const float (&v)[4]) { __builtin_nontemporal_store(mx_f4{v[0], v[1], v[2], v[3]}, (mx_f4u*)o); }
};
template <> struct Mx4Out<MT_F16> {
    typedef _Float16 T;
    static __device__ __forceinline__ void add4(float (&v)[4], const _Float16* r) {
        typedef _Float16 h4 __attribute__((ext_vector_type(4), aligned(2)));            // (a bit cast of ONE element of a vector reads element 0, whichever was named)
        const h4 t = *(const h4*)r;
        v[0] += (float)t[0]; v[1] += (float)t[1]; v[2] += (float)t[2]; v[3] += (float)t[3];
    }
    static __device__ __forceinline__ mx_u2 pack4(const float (&v)[4]) {
        const mx_h2 a = {(_Float16)v[0], (_Float16)v[1]}, b = {(_Float16)v[2], (_Float16)v[3]};
        return mx_u2{__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b)};
    }
    static __device__ __forceinline__ void put4(_Float16* o, const float (&v)[4]) { *(mx_u2u*)o = pack4(v); }
    static __device__ __forceinline__ void stream4(_Float16* o, const float (&v)[4]) { __builtin_nontemporal_store(pack4(v), (mx_u2u*)o); }
};
template <> struct Mx4Out<MT_BF16> {
    typedef __bf16 T;
    static __device__ __forceinline__ void add4(float (&v)[4], const __bf16* r) {
        const mx_u2 t = *(const mx_u2u*)r;
        v[0] += __uint_as_float(t[0] << 16); v[1] += __uint_as_float(t[0] & 0xffff0000u); v[2] += __uint_as_float(t[1] << 16); v[3] += __uint_as_float(t[1] & 0xffff0000u);
    }
    static __device__ __forceinline__ mx_u2 pack4(const float (&v)[4]) {
        const mx_b2 a = {(__bf16)v[0], (__bf16)v[1]}, b = {(__bf16)v[2], (__bf16)v[3]};
        return mx_u2{__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b)};
    }
    static __device__ __forceinline__ void put4(__bf16* o, const float (&v)[4]) { *(mx_u2u*)o = pack4(v); }
    static __device__ __forceinline__ void stream4(__bf16* o, const float (&v)[4]) { __builtin_nontemporal_store(pack4(v), (mx_u2u*)o); }
};
// n of the four are inside the row
template <int OUT>
__device__ __forceinline__ void mx4_finish4(void* out, int64_t o, const void* residual, int64_t r, int n, float (&v)[4]) {
    typedef typename Mx4Out<OUT>::T T;
    T* po = (T*)out + o;
    const T* pr = residual ? (const T*)residual + r : nullptr;
    if (n >= 4) {
        if (pr) Mx4Out<OUT>::add4(v, pr);
        Mx4Out<OUT>::put4(po, v);
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < n) po[i] = (T)(pr ? v[i] + (float)pr[i] : v[i]);
    }
}

template <int ACT> __device__ __forceinline__ float mx4_act(float v) {
    if constexpr (ACT == 1) return v < 0.f ? 0.f : v;                       // (a NaN stays one)
    else if constexpr (ACT == 2) return mx4_gelu(v);
    else return v;
}

// four consecutive outputs (row m, columns n ..): bias, activation, residual, one rounding, store
__device__ __forceinline__ void mx4_store4(const Mx4LinearArgs& a, int64_t m, int64_t n, const mx_f4& bias, float (&v)[4]) {
    const bool in_m = m < a.M;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] += bias[i];
        v[i] = a.act == 0 ? v[i] : a.act == 1 ? mx4_act<1>(v[i]) : mx4_act<2>(v[i]);
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
    const int in = (int)min((int64_t)4, a.N - n);
    if (a.out_type == MT_F32) mx4_finish4<MT_F32>(a.out, m * a.ldo + n, a.residual, m * a.ldr + n, in, v);
    else if (a.out_type == MT_F16) mx4_finish4<MT_F16>(a.out, m * a.ldo + n, a.residual, m * a.ldr + n, in, v);
    else mx4_finish4<MT_BF16>(a.out, m * a.ldo + n, a.residual, m * a.ldr + n, in, v);
}

// ---- few rows, or few tiles: latency.  A workgroup computes 32 NT outputs (n) x 32 tokens (m); its NW waves (or the first of them alone: a.chains)
// take the records of K in turn, each with its own accumulators, and join them through LDS in a fixed order.  Operands go from memory to
// registers in fragment order, a record of weights ahead of its product; activations that are not packed yet are quantised by the lane that
// multiplies them (lane l of the B operand owns row l % 32, block l / 32: a whole block).  Bound by reading the weights where there are many (13 x 8192 x 8192, packed x:
// 10.8 us, 3.3 TB/s of weights; 13 x 8192 x 8320: 8.1 us, 4.5 TB/s -- rows of records a power of two apart are read in step, likely from few
// channels), by the latency of a launch and one trip to memory where there are few (1 x 2304 x 768: 3.1 us).
template <typename XT>
__device__ __forceinline__ Mx4Block mx4_x_fragment(const Mx4LinearArgs& a, int64_t row, int64_t k) {
    Mx4Block b{mx_i4{0, 0, 0, 0}, 0};
    if (row < a.M && k < a.K) {
        Mx4Src<XT> src;
        src.load((const XT*)a.x + row * a.ldx + k, (int)min((int64_t)32, a.K - k));
        b = src.pack();
    }
    return b;
}

template <int NT, int NW, typename XT, bool PACKED>
__global__ void __launch_bounds__(64 * NW) mx4_rows_kernel(Mx4LinearArgs a) {
    constexpr int LDT = 32 * NT + 4;                                        // floats per token row of the joining buffer
    extern __shared__ __attribute__((aligned(16))) float red[];             // [NW][32][LDT]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 31, g = lane >> 5;
    const int64_t nt = blockIdx.x % a.ngroups, m0 = (int64_t)(blockIdx.x / a.ngroups) * 32;
    const int64_t ng = NT == 2 ? nt : nt >> 1;                              // the record's row group, and with NT = 1 the half of it
    const int half = NT == 2 ? 0 : (int)(nt & 1);
    mx_f16 acc[NT];
#pragma unroll
    for (int rt = 0; rt < NT; ++rt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[rt][i] = 0.f;
    mx_i4 wf[NT * 2];
    int ws = 0;
    auto weights = [&](int64_t s) {
        const int64_t rec = ng * a.S + s;
        const char* wc = a.w + rec * MX4_CODES + half * 2048 + lane * 16;
#pragma unroll
        for (int f = 0; f < NT * 2; ++f) wf[f] = *(const mx_i4*)(wc + f * 1024);
        ws = *(const int*)(a.w_scales + rec * MX4_SCALES + lane * 4) >> (16 * half);
    };
    if (ng * MX4_ROWS + 32 * half < a.N && wave < a.chains) {               // (an out_type of 4 bits pads its columns to 128: such a group multiplies nothing)
        weights(wave);
        for (int64_t s = wave; s < a.S; s += a.chains) {
            mx_i4 w[NT * 2];
#pragma unroll
            for (int f = 0; f < NT * 2; ++f) w[f] = wf[f];
            const int wsc = ws;
            if (s + a.chains < a.S) weights(s + a.chains);
            Mx4Block x0, x1;                                                // the two halves of the record; their scales in bytes 0 and 1 where packed
            if constexpr (PACKED) {
                const int64_t rec = (m0 >> 6) * a.S + s;
                const int rt = (int)(m0 >> 5) & 1;
                const char* xc = (const char*)a.x + rec * MX4_CODES + rt * 2048 + lane * 16;
                x0.codes = *(const mx_i4*)xc;
                x1.codes = *(const mx_i4*)(xc + 1024);
                x0.scale = x1.scale = *(const unsigned*)(a.x_scales + rec * MX4_SCALES + lane * 4) >> (16 * rt);
            } else {
                x0 = mx4_x_fragment<XT>(a, m0 + c, s * MX4_K + 32 * g);
                x1 = mx4_x_fragment<XT>(a, m0 + c, s * MX4_K + 64 + 32 * g);
            }
            acc[0] = mx4_mfma<0, 0>(w[0], x0.codes, acc[0], wsc, (int)x0.scale);
            if constexpr (NT == 2) acc[1] = mx4_mfma<2, 0>(w[2], x0.codes, acc[1], wsc, (int)x0.scale);
            acc[0] = mx4_mfma<1, PACKED ? 1 : 0>(w[1], x1.codes, acc[0], wsc, (int)x1.scale);
            if constexpr (NT == 2) acc[1] = mx4_mfma<3, PACKED ? 1 : 0>(w[3], x1.codes, acc[1], wsc, (int)x1.scale);
        }
    }
    float* mine = red + wave * 32 * LDT;
#pragma unroll
    for (int rt = 0; rt < NT; ++rt)
#pragma unroll
        for (int q = 0; q < 4; ++q) *(mx_f4*)&mine[c * LDT + 32 * rt + 8 * q + 4 * g] = mx_f4{acc[rt][4 * q], acc[rt][4 * q + 1], acc[rt][4 * q + 2], acc[rt][4 * q + 3]};
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * 8 * NT; i += 64 * NW) {              // (whole waves: the 4-bit store exchanges maxima between lanes)
        const int t = i / (8 * NT), n4 = i % (8 * NT) * 4;
        const float* p = red + t * LDT + n4;
        mx_f4 s = *(const mx_f4*)p;
        for (int w = 1; w < a.chains; ++w) s += *(const mx_f4*)(p + w * 32 * LDT);
        float v[4] = {s[0], s[1], s[2], s[3]};
        const int64_t n = nt * 32 * NT + n4;
        mx4_store4(a, m0 + t, n, mx4_bias4(a, n), v);
    }
}

// ---- many rows: both operands packed, a workgroup computes BN outputs x BM tokens from LDS.
// A stage holds 128 elements of K: BN / 64 + BM / 64 records, brought in by LDS-DMA in the order they have in memory (a record IS its
// LDS image: every fragment read is 1 KB of consecutive bytes, no bank conflicts, no address arithmetic).  Two slots: stage s + 1 is on
// its way while s is multiplied, s + 2 follows into the slot of s once the second half of s is in registers.  One barrier per stage,
// between the two halves, and every load issued behind a product, so that the matrix pipe has work throughout.  (A third slot costs a
// workgroup per CU and is slower: 16128 x 2304 x 768, 128 x 128 tile, 3 / 2 slots 32.5 / 28.7 us; 8192^3, 256 x 128: 265 / 262; loads behind products instead of in one go: 254.)
// 8192^3: 4.3 PFLOP/s at 1.7 GHz, the matrix pipe busy in 56 % of the cycles.  The clock is the card's power limit; the pipe's idle time is not: products
// alone, on random operands, reach 6.2 PFLOP/s from registers (95 % busy, 1.55 GHz) and 5.7 from LDS (81 %, 1.68 GHz).  Narrow K: bound by writing the output (16128 x 2304 x 768: 81 MB, 2.9 TB/s).
__device__ __forceinline__ void mx4_dma16(unsigned lds, unsigned off, const char* src) {       // 64 lanes x 16 B -> 1 KB at lds
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(src) : "memory", "m0");
}
__device__ __forceinline__ void mx4_dma4(unsigned lds, unsigned off, const char* src) {        // 64 lanes x 4 B -> 256 B at lds
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(src) : "memory", "m0");
}
template <int N> __device__ __forceinline__ void mx4_wait_dma() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

template <int BN, int BM, int WN, int WM>                                   // WN x WM waves
struct Mx4Tile {
    static constexpr int NW = WN * WM, THREADS = 64 * NW;
    static constexpr int RN = BN / 64, RM = BM / 64, REC = RN + RM;         // records of a stage
    static constexpr int TN = BN / WN / 32, TM = BM / WM / 32;              // 32 x 32 tiles of a wave
    static constexpr int STAGE = REC * (MX4_CODES + MX4_SCALES);
    static constexpr int SLOTS = 2;
    static constexpr int CP = REC * 4 / NW, SP = (REC + NW - 1) / NW;       // pieces of codes (1 KB) / of scales (256 B) a wave brings in per stage
    static constexpr int LOADS = CP + SP;
    static constexpr int LDE = TN * 32 + 4;                                 // floats per token row of the epilogue's buffer
    static constexpr int EPI = NW * 32 * LDE * 4;
    static constexpr int LDS = SLOTS * STAGE > EPI ? SLOTS * STAGE : EPI;
    static_assert(REC * 4 % NW == 0, "every wave brings in the same number of pieces");
};

// ---- a wave's 32 tokens x 32 TN outputs, from its part of LDS to memory.  n0, m0: the first column / row; bias added, activation, residual
// added, one rounding, 16 bytes of output a lane (16-bit outputs, 8 bytes / 16 a lane: 16128 x 2304 x 768 29 / 27.5 us).
template <int OUT, int COLS, int LDE, int ACT>
__device__ __forceinline__ void mx4_store_tile(const Mx4LinearArgs& a, const float* ep, int64_t m0, int64_t n0) {
    const int lane = threadIdx.x & 63;
    if constexpr (OUT == MT_MX4) {
        // eight columns a lane, four lanes a block; m0 is a multiple of 32, so a lane's blocks lie 16 bytes a row apart
        constexpr int L8 = COLS / 8, R8 = 64 / L8;
        const int64_t n = n0 + (lane % L8) * 8;
        if (n0 >= a.out_S * MX4_K || m0 >= a.M) return;
        const mx_f4 b0 = mx4_bias4(a, n), b1 = mx4_bias4(a, n + 4);
        const bool inside = n0 + COLS <= a.N;
        const Mx4Place p = mx4_place(m0 + lane / L8, n >> 5, a.out_S);
        char* code = (char*)a.out + p.code + ((n & 31) >> 1);
        char* scale = a.out_scales + p.scale;
        const int rows = (int)min((int64_t)32, a.M - m0);
#pragma unroll 2
        for (int it = 0; it < 32 / R8; ++it) {
            const int t = it * R8 + lane / L8;
            const mx_f4 w0 = *(const mx_f4*)&ep[t * LDE + (lane % L8) * 8], w1 = *(const mx_f4*)&ep[t * LDE + (lane % L8) * 8 + 4];
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] = mx4_act<ACT>(w0[i] + b0[i]); v[4 + i] = mx4_act<ACT>(w1[i] + b1[i]); }
            if (!inside) {
#pragma unroll
                for (int i = 0; i < 8; ++i) if (n + i >= a.N) v[i] = 0.f;
            }
            unsigned sc;
            const unsigned four = mx4_pack_octets(v, &sc);                  // (every lane is here: the 4 lanes of a block exchange their maxima)
            if (t < rows) {
                *(unsigned*)(code + it * R8 * 16) = four;
                if ((n & 31) == 0) scale[it * R8 * 4] = (char)sc;
            }
        }
    } else {
        typedef typename Mx4Out<OUT>::T T;
        if (m0 >= a.M || n0 >= a.N) return;
        // as many columns a lane as 16 bytes of output hold
        constexpr int C = 16 / sizeof(T), LR = COLS / C, RI = 64 / LR;
        const int64_t n = n0 + (lane % LR) * C;
        const int row = lane / LR, in = (int)min((int64_t)C, a.N - n);
        mx_f4 bias[C / 4];
#pragma unroll
        for (int q = 0; q < C / 4; ++q) bias[q] = mx4_bias4(a, n + 4 * q);
        int64_t o = (m0 + row) * a.ldo + n, r = (m0 + row) * a.ldr + n;
        const bool whole = n0 + COLS <= a.N && m0 + 32 <= a.M;              // (of the wave)
        const int rows = (int)min((int64_t)32, a.M - m0);
#pragma unroll 2
        for (int it = 0; it < 32 / RI; ++it, o += RI * a.ldo, r += RI * a.ldr) {
            float v[C / 4][4];
#pragma unroll
            for (int q = 0; q < C / 4; ++q) {
                const mx_f4 w = *(const mx_f4*)&ep[(it * RI + row) * LDE + (lane % LR) * C + 4 * q];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[q][i] = mx4_act<ACT>(w[i] + bias[q][i]);
            }
            if (whole) {
                if (a.residual) {
#pragma unroll
                    for (int q = 0; q < C / 4; ++q) Mx4Out<OUT>::add4(v[q], (const T*)a.residual + r + 4 * q);
                }
                if constexpr (C == 4) Mx4Out<OUT>::stream4((T*)a.out + o, v[0]);
                else {
                    const mx_u2 lo = Mx4Out<OUT>::pack4(v[0]), hi = Mx4Out<OUT>::pack4(v[C / 4 - 1]);
                    __builtin_nontemporal_store(mx_u4{lo[0], lo[1], hi[0], hi[1]}, (mx_u4u*)((T*)a.out + o));
                }
            } else if (it * RI + row < rows) {
#pragma unroll
                for (int q = 0; q < C / 4; ++q) if (in > 4 * q) mx4_finish4<OUT>(a.out, o + 4 * q, a.residual, r + 4 * q, in - 4 * q, v[q]);
            }
        }
    }
}

template <int BN, int BM, int WN, int WM, int OUT>
__global__ void __launch_bounds__(64 * WN * WM, 2) mx4_tile_kernel(Mx4LinearArgs a, int ntiles, int mtiles) {
    typedef Mx4Tile<BN, BM, WN, WM> T;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // tiles in the order of their XCD (workgroup b runs on XCD b % 8), eight rows of tiles by columns: what an XCD works on at a time
    // shares its operands in that XCD's L2
    const int total = ntiles * mtiles;
    int id = blockIdx.x;
    { const int per = total / 8, rest = total % 8, x = id % 8; id = x * per + min(x, rest) + id / 8; }
    constexpr int GRP = 8;
    const int band = id / (GRP * ntiles), in_band = id - band * GRP * ntiles, bh = min(GRP, mtiles - band * GRP);
    const int mt = band * GRP + in_band % bh, nt = in_band / bh;
    const int S = (int)a.S;
    const int64_t nrec = (a.N + MX4_ROWS - 1) / MX4_ROWS, mrec = (a.M + MX4_ROWS - 1) / MX4_ROWS;
    // the pieces this wave brings in, at the same place of every stage (a tile's missing rows read the last record)
    auto record = [&](int rec, bool scales) {
        const bool is_w = rec < T::RN;
        const int64_t g = is_w ? min((int64_t)nt * T::RN + rec, nrec - 1) : min((int64_t)mt * T::RM + rec - T::RN, mrec - 1);
        return scales ? (is_w ? a.w_scales : a.x_scales) + g * S * MX4_SCALES : (is_w ? a.w : (const char*)a.x) + g * S * MX4_CODES;
    };
    const char* src_codes[T::CP];
    const char* src_scales[T::SP];
#pragma unroll
    for (int i = 0; i < T::CP; ++i) src_codes[i] = record((wave * T::CP + i) / 4, false) + (wave * T::CP + i) % 4 * 1024;
#pragma unroll
    for (int i = 0; i < T::SP; ++i) src_scales[i] = record(min(wave * T::SP + i, T::REC - 1), true);
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    const unsigned off16 = lane * 16, off4 = lane * 4;
    // piece i of what this wave brings in for stage s: CP pieces of codes, then SP of scales
    auto bring = [&](int s, int i) {
        const unsigned slot = lds0 + (s % T::SLOTS) * T::STAGE;
        if (i < T::CP) mx4_dma16(slot + (wave * T::CP + i) * 1024, off16, src_codes[i] + (int64_t)s * MX4_CODES);
        else {
            const int j = i - T::CP;
            mx4_dma4(slot + T::REC * MX4_CODES + min(wave * T::SP + j, T::REC - 1) * MX4_SCALES, off4, src_scales[j] + (int64_t)s * MX4_SCALES);
        }
    };
    const int wn = wave / WM, wm = wave % WM;                               // the wave's place in the tile
    // row tile j of the wave: rows 32 (wn TN + j) of the tile = record (..) / 2, half (..) % 2 of it.  TN and TM are even or the wave's
    // first row tile is at an even place, so the byte of the scale dword is known at compile time
    static_assert(T::TN % 2 == 0 && T::TM % 2 == 0, "a wave owns whole records");
    mx_i4 fa[2][T::TN], fb[2][T::TM];
    int sa[T::TN / 2], sb[T::TM / 2];
    // fragment i of half kh of a stage: the first of each operand first, so that a product can start
    constexpr int FRAGS = T::TN + T::TM, SCALES = (T::TN + T::TM) / 2;
    auto fetch = [&](const char* slot, int kh, int i, mx_i4 (&A)[T::TN], mx_i4 (&B)[T::TM]) {
        const int j = i < 2 * T::TM ? i / 2 : i - T::TM;                    // (TM <= TN: A0 B0 A1 B1 .. then the rest of A)
        if (i < 2 * T::TM && i % 2) B[j] = *(const mx_i4*)(slot + (T::RN + wm * T::TM / 2 + j / 2) * MX4_CODES + (2 * (j & 1) + kh) * 1024 + lane * 16);
        else A[j] = *(const mx_i4*)(slot + (wn * T::TN / 2 + j / 2) * MX4_CODES + (2 * (j & 1) + kh) * 1024 + lane * 16);
    };
    auto fetch_scale = [&](const char* slot, int i, int (&A)[T::TN / 2], int (&B)[T::TM / 2]) {
        if (i < T::TN / 2) A[i] = *(const int*)(slot + T::REC * MX4_CODES + (wn * T::TN / 2 + i) * MX4_SCALES + lane * 4);
        else B[i - T::TN / 2] = *(const int*)(slot + T::REC * MX4_CODES + (T::RN + wm * T::TM / 2 + i - T::TN / 2) * MX4_SCALES + lane * 4);
    };
    mx_f16 acc[T::TN][T::TM];
#pragma unroll
    for (int i = 0; i < T::TN; ++i)
#pragma unroll
        for (int j = 0; j < T::TM; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    // one half of a stage; between(i) is what else is issued behind product i: the matrix pipe is busy for 32 cycles with each, and a wave
    // that issues its loads in one go instead leaves it idle meanwhile
    constexpr int PROD = T::TN * T::TM;
    auto multiply = [&](auto KH, mx_i4 (&A)[T::TN], mx_i4 (&B)[T::TM], int (&SA)[T::TN / 2], int (&SB)[T::TM / 2], auto between) {
        constexpr int kh = decltype(KH)::value;
#pragma unroll
        for (int i = 0; i < T::TN; i += 2)
#pragma unroll
            for (int j = 0; j < T::TM; j += 2) {
                const int p = (i / 2 * (T::TM / 2) + j / 2) * 4;
                acc[i][j] = mx4_mfma<kh, kh>(A[i], B[j], acc[i][j], SA[i / 2], SB[j / 2]);
                between(p);
                acc[i + 1][j] = mx4_mfma<2 + kh, kh>(A[i + 1], B[j], acc[i + 1][j], SA[i / 2], SB[j / 2]);
                between(p + 1);
                acc[i][j + 1] = mx4_mfma<kh, 2 + kh>(A[i], B[j + 1], acc[i][j + 1], SA[i / 2], SB[j / 2]);
                between(p + 2);
                acc[i + 1][j + 1] = mx4_mfma<2 + kh, 2 + kh>(A[i + 1], B[j + 1], acc[i + 1][j + 1], SA[i / 2], SB[j / 2]);
                between(p + 3);
            }
    };
    std::integral_constant<int, 0> K0;
    std::integral_constant<int, 1> K1;
    // ---- the pipeline
    for (int s = 0; s < T::SLOTS && s < S; ++s) {
#pragma unroll
        for (int i = 0; i < T::LOADS; ++i) bring(s, i);
    }
    if (S > 1) mx4_wait_dma<T::LOADS>(); else mx4_wait_dma<0>();            // stage 0 is here
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < FRAGS; ++i) fetch(lds, 0, i, fa[0], fb[0]);
#pragma unroll
    for (int i = 0; i < SCALES; ++i) fetch_scale(lds, i, sa, sb);
    constexpr int PER_F = (FRAGS + PROD - 1) / PROD, PER_S = (SCALES + PROD - 1) / PROD, PER_L = (T::LOADS + PROD - 1) / PROD;
    auto step = [&](int s, auto MORE) {                                     // MORE: stage s + 2 exists
        const char* slot = lds + s % T::SLOTS * T::STAGE;
        const char* next = lds + (s + 1) % T::SLOTS * T::STAGE;
        multiply(K0, fa[0], fb[0], sa, sb, [&](int p) {
#pragma unroll
            for (int i = p * PER_F; i < (p + 1) * PER_F; ++i) if (i < FRAGS) fetch(slot, 1, i, fa[1], fb[1]);
            __builtin_amdgcn_sched_barrier(0);
        });
        // stage s + 1 has landed (this wave's part; the barrier says so for all), and this wave is done reading the slot of s
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        int oa[T::TN / 2], ob[T::TM / 2];                                   // the scales of the half that is still to be multiplied
#pragma unroll
        for (int i = 0; i < T::TN / 2; ++i) oa[i] = sa[i];
#pragma unroll
        for (int i = 0; i < T::TM / 2; ++i) ob[i] = sb[i];
        multiply(K1, fa[1], fb[1], oa, ob, [&](int p) {
#pragma unroll
            for (int i = p * PER_F; i < (p + 1) * PER_F; ++i) if (i < FRAGS) fetch(next, 0, i, fa[0], fb[0]);
#pragma unroll
            for (int i = p * PER_S; i < (p + 1) * PER_S; ++i) if (i < SCALES) fetch_scale(next, i, sa, sb);
            if constexpr (decltype(MORE)::value) {
#pragma unroll
                for (int i = p * PER_L; i < (p + 1) * PER_L; ++i) if (i < T::LOADS) bring(s + T::SLOTS, i);
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    {
        int s = 0;
        for (; s + T::SLOTS < S; ++s) step(s, std::true_type{});
        for (; s + 1 < S; ++s) step(s, std::false_type{});
        const char* slot = lds + (S - 1) % T::SLOTS * T::STAGE;
#pragma unroll
        for (int i = 0; i < FRAGS; ++i) fetch(slot, 1, i, fa[1], fb[1]);
        multiply(K0, fa[0], fb[0], sa, sb, [](int) {});
        multiply(K1, fa[1], fb[1], sa, sb, [](int) {});
    }
    __syncthreads();                                                        // every wave has left the ring
    // ---- epilogue: 32 tokens at a time through the wave's own part of LDS, so that a lane holds four consecutive outputs of a token and
    // a wave stores whole rows (straight from the accumulators a row would leave in pieces of 16 bytes)
    float* ep = (float*)lds + wave * 32 * T::LDE;
    const int c = lane & 31, g = lane >> 5;
    const int64_t n0 = (int64_t)nt * BN + wn * T::TN * 32, mw = (int64_t)mt * BM + wm * T::TM * 32;
#pragma unroll
    for (int j = 0; j < T::TM; ++j) {
#pragma unroll
        for (int i = 0; i < T::TN; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *(mx_f4*)&ep[c * T::LDE + 32 * i + 8 * q + 4 * g] = mx_f4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");              // (LDS serves a wave in order: what is left to do is to keep the compiler's)
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (a.act == 0) mx4_store_tile<OUT, T::TN * 32, T::LDE, 0>(a, ep, mw + 32 * j, n0);
        else if (a.act == 1) mx4_store_tile<OUT, T::TN * 32, T::LDE, 1>(a, ep, mw + 32 * j, n0);
        else mx4_store_tile<OUT, T::TN * 32, T::LDE, 2>(a, ep, mw + 32 * j, n0);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
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
static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static bool on_element(const void* p, int type) { return (uintptr_t)p % (type == UITK_T_F32 ? 4 : 2) == 0; }

template <int NT, int NW>
static hipError_t mx4_launch_rows(Mx4LinearArgs& a, bool one_chain, hipStream_t s) {
    const int64_t cols = a.out_type == MT_MX4 ? a.out_S * MX4_K : a.N;
    const int64_t ngroups = (cols + 32 * NT - 1) / (32 * NT), mt = (a.M + 31) / 32;
    if (mt * ngroups > ((int64_t)1 << 32) / (64 * NW) - 1) return hipErrorInvalidConfiguration;
    a.ngroups = (unsigned)ngroups;
    a.chains = one_chain ? 1 : (int)std::min<int64_t>(NW, a.S);
    const dim3 grid((unsigned)(mt * ngroups));
    constexpr int lds = NW * 32 * (32 * NT + 4) * 4;
    auto go = [&](auto kernel) {
        if (lds > 64 * 1024)                                                // (of the current device: set at every call, not once per process)
            if (hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds); e != hipSuccess) return e;
        hipLaunchKernelGGL(kernel, grid, dim3(64 * NW), lds, s, a);
        return hipGetLastError();
    };
    if (a.x_type == MT_MX4) return go(mx4_rows_kernel<NT, NW, float, true>);
    if (a.x_type == MT_F32) return go(mx4_rows_kernel<NT, NW, float, false>);
    if (a.x_type == MT_F16) return go(mx4_rows_kernel<NT, NW, _Float16, false>);
    return go(mx4_rows_kernel<NT, NW, __bf16, false>);
}

template <int BN, int BM, int WN, int WM, int OUT>
static hipError_t mx4_launch_tile_as(const Mx4LinearArgs& a, hipStream_t s) {
    typedef Mx4Tile<BN, BM, WN, WM> T;
    const int64_t cols = a.out_type == MT_MX4 ? a.out_S * MX4_K : a.N;
    const int64_t nt = (cols + BN - 1) / BN, mt = (a.M + BM - 1) / BM;
    if (nt * mt > ((int64_t)1 << 32) / T::THREADS - 1) return hipErrorInvalidConfiguration;
    if (T::LDS > 64 * 1024)                                                 // (of the current device: set at every call, not once per process)
        if (hipError_t e = hipFuncSetAttribute((const void*)mx4_tile_kernel<BN, BM, WN, WM, OUT>, hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS); e != hipSuccess) return e;
    hipLaunchKernelGGL((mx4_tile_kernel<BN, BM, WN, WM, OUT>), dim3((unsigned)(nt * mt)), dim3(T::THREADS), T::LDS, s, a, (int)nt, (int)mt);
    return hipGetLastError();
}
template <int BN, int BM, int WN, int WM>
static hipError_t mx4_launch_tile(const Mx4LinearArgs& a, hipStream_t s) {
    if (a.out_type == MT_F32) return mx4_launch_tile_as<BN, BM, WN, WM, MT_F32>(a, s);
    if (a.out_type == MT_F16) return mx4_launch_tile_as<BN, BM, WN, WM, MT_F16>(a, s);
    if (a.out_type == MT_BF16) return mx4_launch_tile_as<BN, BM, WN, WM, MT_BF16>(a, s);
    return mx4_launch_tile_as<BN, BM, WN, WM, MT_MX4>(a, s);
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
    if (!on_element(x, type)) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_quantize: x is not aligned to its elements");
    if (!aligned16(q)) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_quantize: the packed buffer must be 16-byte aligned");
    const int64_t R = (rows + MX4_ROWS - 1) / MX4_ROWS, S = (K + MX4_K - 1) / MX4_K;
    char* codes = (char*)q;
    char* scales = codes + R * S * MX4_CODES;
    if ((R * S + 3) / 4 > MX4_MAX_GRID) return set_error(UITK_ERR_UNSUPPORTED, "uitk_mx4_quantize: more elements than one launch takes");
    // a record to a workgroup / to a wave, us: bf16 1021 x 1000 (128 records) 3.4 / 6.8, 2048 x 4096 (1024) 4.1 / 4.8, 8192 x 4096 (4096) 13.6 / 17.1; fp32
    // 1021 x 1000 3.4 / 7.2, 16128 x 768 (1512) 9.8 / 9.7
    const bool split = R * S <= 1024;
    const dim3 grid((unsigned)(split ? R * S : (R * S + 3) / 4)), block(256);
    hipStream_t s = (hipStream_t)stream;
    auto launch = [&](auto kernel, const auto* p) { hipLaunchKernelGGL(kernel, grid, block, 0, s, p, rows, K, ld, R, S, codes, scales); };
    if (type == UITK_T_F32) split ? launch(mx4_quantize_kernel<float, true>, (const float*)x) : launch(mx4_quantize_kernel<float, false>, (const float*)x);
    else if (type == UITK_T_F16) split ? launch(mx4_quantize_kernel<_Float16, true>, (const _Float16*)x) : launch(mx4_quantize_kernel<_Float16, false>, (const _Float16*)x);
    else split ? launch(mx4_quantize_kernel<__bf16, true>, (const __bf16*)x) : launch(mx4_quantize_kernel<__bf16, false>, (const __bf16*)x);
    MX4_HIP(hipGetLastError());
    return UITK_OK;
}

int uitk_mx4_dequantize(const void* q, int64_t rows, int64_t K, void* x, int type, int64_t ld, void* stream) {
    if (int rc = mx4_check_matrix("uitk_mx4_dequantize", rows, K)) return rc;
    if (type < UITK_T_F32 || type > UITK_T_BF16) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_dequantize: unknown type");
    if (rows == 0) return UITK_OK;
    if (!x || !q) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_dequantize: null pointer");
    if (ld < K) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_dequantize: rows overlap (ld < K)");
    if (!on_element(x, type)) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_dequantize: x is not aligned to its elements");
    if (!aligned16(q)) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_dequantize: the packed buffer must be 16-byte aligned");
    const int64_t R = (rows + MX4_ROWS - 1) / MX4_ROWS, S = (K + MX4_K - 1) / MX4_K;
    if ((R * S + 3) / 4 > MX4_MAX_GRID) return set_error(UITK_ERR_UNSUPPORTED, "uitk_mx4_dequantize: more elements than one launch takes");
    const char* codes = (const char*)q;
    const char* scales = codes + R * S * MX4_CODES;
    const dim3 grid((unsigned)((R * S + 3) / 4)), block(256);
    hipStream_t s = (hipStream_t)stream;
    // whole 16-byte pieces go past the caches (32768 x 4096 bf16 73 / 56 us), pieces across their borders must not (4095 wide: 104 / 126)
    const bool nt = aligned16(x) && ld * (type == UITK_T_F32 ? 4 : 2) % 16 == 0;
    auto launch = [&](auto kernel, auto* p) { hipLaunchKernelGGL(kernel, grid, block, 0, s, codes, scales, rows, K, ld, R, S, p); };
    if (type == UITK_T_F32) nt ? launch(mx4_dequantize_kernel<float, true>, (float*)x) : launch(mx4_dequantize_kernel<float, false>, (float*)x);
    else if (type == UITK_T_F16) nt ? launch(mx4_dequantize_kernel<_Float16, true>, (_Float16*)x) : launch(mx4_dequantize_kernel<_Float16, false>, (_Float16*)x);
    else nt ? launch(mx4_dequantize_kernel<__bf16, true>, (__bf16*)x) : launch(mx4_dequantize_kernel<__bf16, false>, (__bf16*)x);
    MX4_HIP(hipGetLastError());
    return UITK_OK;
}

int64_t uitk_mx4_linear_workspace(int64_t M, int64_t N, int64_t K, int x_type) {
    if (M < 0 || M > MX4_MAX_ROWS || N < 1 || N > MX4_MAX_K || K < 1 || K > MX4_MAX_K || x_type < UITK_T_F32 || x_type > UITK_T_MX4) return -1;
    return mx4_plan(M, N, K, x_type == UITK_T_MX4).quantize_first ? mx4_bytes(M, K) : 0;
}

int uitk_mx4_linear(const uitk_mx4_linear_args* u, void* stream) { return mx4_linear(u, mx4_plan, stream); }

}  // extern "C"

int uitk::mx4_linear(const uitk_mx4_linear_args* u, Mx4Plan (*rule)(int64_t, int64_t, int64_t, bool), void* stream) {
    if (!u) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: null arguments");
    if (int rc = mx4_check_matrix("uitk_mx4_linear (x)", u->M, u->K)) return rc;
    if (u->N < 1 || u->N > MX4_MAX_K) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: N must be 1 .. 2^20");
    if (u->x_type < UITK_T_F32 || u->x_type > UITK_T_MX4) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: unknown x_type");
    if (u->out_type < UITK_T_F32 || u->out_type > UITK_T_MX4) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: unknown out_type");
    if (u->act < 0 || u->act > 2) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: act must be 0 (none), 1 (ReLU) or 2 (GELU)");
    if (u->residual && u->out_type == UITK_T_MX4) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: a residual needs an output of 16 or 32 bits");
    if (u->reserved) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: reserved must be 0");
    if (u->M == 0) return UITK_OK;
    if (!u->x || !u->w || !u->out) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: null pointer");
    if (!aligned16(u->w) || (u->x_type == UITK_T_MX4 && !aligned16(u->x)) || (u->out_type == UITK_T_MX4 && !aligned16(u->out)))
        return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: packed matrices must be 16-byte aligned");
    if (!on_element(u->bias, UITK_T_F32) || (u->x_type != UITK_T_MX4 && !on_element(u->x, u->x_type)) ||
        (u->out_type != UITK_T_MX4 && (!on_element(u->out, u->out_type) || !on_element(u->residual, u->out_type))))
        return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: a pointer is not aligned to its elements");
    if (u->x_type != UITK_T_MX4 && u->ldx < u->K) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: rows of x overlap (ldx < K)");
    if (u->out_type != UITK_T_MX4 && u->ldo < u->N) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: rows of the output overlap (ldo < N)");
    if (u->residual && u->ldr < u->N) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: rows of the residual overlap (ldr < N)");
    Mx4LinearArgs a{};
    a.M = u->M; a.K = u->K; a.N = u->N; a.S = (u->K + MX4_K - 1) / MX4_K;
    a.x = u->x; a.x_type = u->x_type; a.ldx = u->ldx;
    if (u->x_type == UITK_T_MX4) a.x_scales = (const char*)u->x + mx4_records(u->M, u->K) * MX4_CODES;
    a.w = (const char*)u->w; a.w_scales = a.w + mx4_records(u->N, u->K) * MX4_CODES;
    a.bias = u->bias; a.act = u->act; a.residual = u->residual; a.ldr = u->ldr;
    a.out = u->out; a.ldo = u->ldo; a.out_type = u->out_type;
    if (u->out_type == UITK_T_MX4) { a.out_S = (u->N + MX4_K - 1) / MX4_K; a.out_scales = (char*)u->out + mx4_records(u->M, u->N) * MX4_CODES; }
    hipStream_t s = (hipStream_t)stream;
    const Mx4Plan plan = rule(u->M, u->N, u->K, u->x_type == UITK_T_MX4);
    if (plan.quantize_first) {
        if (!u->workspace || !aligned16(u->workspace)) return set_error(UITK_ERR_INVALID_ARG, "uitk_mx4_linear: needs a 16-byte aligned workspace (uitk_mx4_linear_workspace)");
        if (int rc = uitk_mx4_quantize(u->x, u->x_type, u->M, u->K, u->ldx, u->workspace, stream)) return rc;
        a.x = u->workspace; a.x_type = MT_MX4; a.x_scales = (const char*)u->workspace + mx4_records(u->M, u->K) * MX4_CODES;
    }
    const hipError_t e = plan.kernel == MX4_TILE256   ? mx4_launch_tile<256, 128, 2, 2>(a, s)
                         : plan.kernel == MX4_TILE128 ? mx4_launch_tile<128, 128, 2, 2>(a, s)
                         : plan.kernel == MX4_ROWS64  ? mx4_launch_rows<2, 8>(a, plan.one_chain, s)
                         : plan.kernel == MX4_ROWS16  ? mx4_launch_rows<1, 16>(a, plan.one_chain, s)
                                                      : mx4_launch_rows<1, 8>(a, plan.one_chain, s);
    if (e == hipErrorInvalidConfiguration) return set_error(UITK_ERR_UNSUPPORTED, "uitk_mx4_linear: more outputs than one launch takes");
    MX4_HIP(e);
    return UITK_OK;
}
