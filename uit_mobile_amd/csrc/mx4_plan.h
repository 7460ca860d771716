// mx4_plan.h -- which kernel of mx4.hip a product of 4-bit matrices runs on, and whether its activations are quantised in a launch of their own.
// Host code, by sizes alone.
#pragma once
#include <stdint.h>

struct uitk_mx4_linear_args;

namespace uitk {

// us on the GPU (calls inside a replayed graph), packed x unless said otherwise; more shapes in profiles/operators/plan_sweep.log.
// * rows against tiles: 128 x 128 tiles need more than 128 of them.  Rows / tiles: 36 tiles (252 x 2304 x 768) 4.0 / 6.2, 96 (2016 x 768 x 768) 6.0 / 6.0,
//   128 (252 x 8192 x 1024) 7.7 / 7.1, 144 (1008 x 2304 x 768) 8.1 / 6.4, 256 (2048 x 2048 x 1024) 12.5 / 6.9.  256 x 128 ones need two workgroups on every CU
//   and a K that outweighs their longer epilogue (128 x 128 / 256 x 128: 16128 x 2304 x 768: 28.7 / 36.8; 16128 x 2304 x 2048: 50.4 / 55.2;
//   4096 x 4096 x 4096: 41.3 / 40.1; 8192 x 8192 x 8192: 270 / 254).
// * rows: 64 columns a workgroup instead of 32 with more than 512 workgroups of 32 (groups, 32 / 64 columns: 100 x 4096 x 768, 512: 3.6 / 3.6;
//   128 x 8192 x 768, 1024: 4.4 / 4.3; 32 x 20480 x 2048, 640: 7.0 / 5.7; 128 x 8192 x 8192, 1024: 29 / 13).  From K = 4096 on they are faster below 512
//   too (64 x 8192 x 4096, 512: 10.0 / 5.8; 32 x 8192 x 4096, 256: 7.4 / 5.6), which this rule leaves unused.
// * rows of 32 columns: 8 waves share K, 16 from 32 records on (8 / 16: 1 x 2304 x 4096 4.0 / 4.2, 13 x 8192 x 5120 5.0 / 5.2, 32 x 4096 x 8192 8.0 / 7.2,
//   1 x 2304 x 16384 7.7 / 7.4): nothing either way at the threshold, the gain is in the long ones.
// * quantising inside repeats the work in every column group, about 65 vector instructions per 32 x 64 fragment (two to three times that for fp32); a launch of
//   its own costs 2.6 us of the GPU, and a caller that does not replay a graph 3 us of the host and a workspace.  The rule counts fragments in
//   columns of 32, twice what the 64-column kernel has.  Inside / first, 16-bit x (fragments that are quantised): 1 x 2304 x 768 (864) 4.1 / 6.0,
//   252 x 768 x 768 (2304) 4.7 / 5.8, 1003 x 537 x 1000 (4608, counted as 8704) 7.1 / 7.9, 128 x 4096 x 1024 (8192) 7.4 / 6.4, 64 x 4096 x 4096 (16384) 12.2 / 7.7,
//   13 x 8192 x 8192 (32768) 16.2 / 13.6; fp32: 4.8 / 6.0, 6.2 / 5.9, 16.4 / 7.8, 15.9 / 6.4, 22.3 / 7.7, 23.3 / 13.6.
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
