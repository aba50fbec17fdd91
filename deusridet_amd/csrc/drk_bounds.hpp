// drk_bounds.hpp -- the bounds buffer's layout and the power of two of its codes, shared by the
// kernels that write the bounds and the ones that score queries against them.
#pragma once

#include "drk_common.hpp"

namespace drk {

// codes int8 [layers][blocks][kv heads][2][D], then exponents int8 [layers][blocks][kv heads]
inline size_t bounds_exps_offset(const Lay &a) { return (size_t)a.L * a.NB * a.KVH * 2 * a.D; }
int bounds_lay(const drk_kv_layout *g, Lay *a, const char *who);      // make_lay + the head_dims that have bounds

// The smallest e in [-40, 40] with amax <= 127 * 2^e.  amax = s * 2^x with s in [1, 2): 127 * 2^e is
// 127/64 * 2^(e+6), so e = x - 6 when s <= 127/64 -- the 23 fraction bits at most 63/64 of their range -- and
// x - 5 otherwise.  Zero and numbers below 2^-34 give -40, infinity 40.
__device__ __forceinline__ int bounds_exponent(float amax)
{
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 6 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return e < -40 ? -40 : (e > 40 ? 40 : e);
}

} // namespace drk
