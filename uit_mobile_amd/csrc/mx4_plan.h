// mx4_plan.h -- which kernel of mx4.hip a product of 4-bit matrices runs on, and whether its activations are quantised in a launch of their own.
// Host code, by sizes alone.
#pragma once
#include <stdint.h>

struct uitk_mx4_linear_args;

namespace uitk {

// us on the GPU, packed x unless said otherwise:
// * rows against tiles: 128 x 128 tiles need more than 128 of them (rows / 128 x 128: 512 x 4096 x 4096: 12.5 / 13.1; 128 x 16384 x 4096: 15.7 / 19.2;
//   300 x 8192 x 512: 7.7 / 6.1; 2048 x 4096 x 2048: 31 / 16), 256 x 128 ones two workgroups on every CU and a K that outweighs their longer
//   epilogue (128 x 128 / 256 x 128: 16128 x 2304 x 768: 28.7 / 36.8; 16128 x 2304 x 2048: 50.4 / 55.2; 4096 x 4096 x 4096: 41.3 / 40.1; 8192 x 8192 x 8192: 270 / 254).
// * rows: 8 waves share K, 16 where a wave would still have two records or more (13 x 8192 x 8192, 8 / 16: 12.5 / 11.9); with more than 512
//   workgroups 64 columns each instead of 32 (128 x 8192 x 8192, 32 / 64: 21.4 / 17.5).
// * quantising inside repeats the work in every column group, about 65 vector instructions per 32 x 64 fragment; a launch of its own costs
//   2.6 us of the GPU, and a caller that does not replay a graph 3 us of the host and a workspace.  bf16 inside / packed, GPU: 1 x 2304 x 768 (864
//   fragments) 4.4 / 3.2, 252 x 768 x 768 (2304) 4.9 / 3.4, 1003 x 537 x 1000 (8704) 11 / 5.1, 64 x 4096 x 4096 (16384) 12.4 / 6.0, 13 x 8192 x 8192 (32768) 17.7 / 11.9.
enum { MX4_ROWS8 = 0, MX4_ROWS16, MX4_ROWS64, MX4_TILE128, MX4_TILE256 };
struct Mx4Plan { int kernel; bool quantize_first, one_chain; };           // one_chain: a rows kernel gives all of K to one wave
inline Mx4Plan mx4_plan(int64_t M, int64_t N, int64_t K, bool packed) {
    const int64_t m128 = (M + 127) / 128, S = (K + 127) / 128, groups = ((N + 31) / 32) * ((M + 31) / 32);       // S: records along K
    Mx4Plan p{MX4_ROWS8, !packed, false};
    if (M > 64 && m128 * ((N + 127) / 128) > 128) p.kernel = m128 * ((N + 255) / 256) >= 512 && K >= 4096 ? MX4_TILE256 : MX4_TILE128;
    else if (groups > 512) p.kernel = MX4_ROWS64;
    else if (S >= 32) p.kernel = MX4_ROWS16;
    if (p.kernel < MX4_TILE128 && 2 * groups * S <= 10240) p.quantize_first = false;
    return p;
}

// The same for a caller whose rows must not see how many others there are (the general engine: a clip's result is the same in any batch, shard or
// chunk).  The tile kernels add along K in one chain; the rows kernels join 8 or 16, and are told here to give all of K to one wave, which
// adds in the tiles' order.  General engine, 8 or 16 chains / one, ms: 768 wide, 1 ten-second clip 8.37 / 8.56, 4 clips 8.76 / 8.87, 64 clips
// 11.6 / 11.6; 96 wide, 1 to 64 clips no difference.  (Tiles whatever the rows: 8.75 for 1 clip; 96 wide 0.22 -> 0.24 for 1, 0.28 -> 0.33 for 64.)
inline Mx4Plan mx4_plan_one_chain(int64_t M, int64_t N, int64_t K, bool packed) {
    Mx4Plan p = mx4_plan(M, N, K, packed);
    if (p.kernel == MX4_ROWS16) p.kernel = MX4_ROWS8;
    p.one_chain = p.kernel < MX4_TILE128;
    return p;
}

// uitk_mx4_linear by either rule
int mx4_linear(const uitk_mx4_linear_args* u, Mx4Plan (*rule)(int64_t, int64_t, int64_t, bool), void* stream);

}  // namespace uitk
