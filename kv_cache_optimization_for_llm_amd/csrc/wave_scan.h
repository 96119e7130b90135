// Prefixes over the 64 lanes of a wavefront in the vector ALU, of 32 and 64-bit whole numbers (a shuffle's trip through LDS is as
// long as two of these steps).
#pragma once
#include "common.h"

typedef unsigned long long u64;

// Numbers from lanes in front of this one, or `none` where there is no such lane.
template <int CTRL, int ROWS>
__device__ inline unsigned wave_from(unsigned v, unsigned none) {
    return __builtin_amdgcn_update_dpp(none, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ inline u64 wave_from(u64 v, u64 none) {
    return (u64)wave_from<CTRL, ROWS>((unsigned)(v >> 32), (unsigned)(none >> 32)) << 32 | wave_from<CTRL, ROWS>((unsigned)v, (unsigned)none);
}
// Inclusive prefix of the wavefront in the vector ALU: 1, 2, 4 and 8 lanes up inside rows of 16, then the last lane of a row to the
// next one, then that of the first half to the second.
template <typename T, typename OP>
__device__ inline T wave_scan(T v, T none, OP op) {
    v = op(v, wave_from<0x111, 0xf>(v, none));
    v = op(v, wave_from<0x112, 0xf>(v, none));
    v = op(v, wave_from<0x114, 0xf>(v, none));
    v = op(v, wave_from<0x118, 0xf>(v, none));
    v = op(v, wave_from<0x142, 0xa>(v, none));
    return op(v, wave_from<0x143, 0xc>(v, none));
}
template <typename T>
__device__ inline T wave_prefix(T v) {
    return wave_scan(v, (T)0, [](T a, T b) { return a + b; });
}
__device__ inline unsigned wave_last(unsigned v) { return __builtin_amdgcn_readlane(v, KVA_WAVE - 1); }
__device__ inline u64 wave_last(u64 v) { return (u64)wave_last((unsigned)(v >> 32)) << 32 | wave_last((unsigned)v); }
