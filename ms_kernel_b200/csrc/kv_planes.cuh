// The planes of one packed cache and a plain read of one element.
#pragma once

#include "msaq_common.cuh"

namespace msaq {

struct KvPlanes {
    const int8_t* s;
    const uint8_t* u;
    const uint8_t* h;
};

// One dequantised element (block-local index k) of the record at `slot`.
__device__ __forceinline__ float kv_element(const KvPlanes& p, int64_t slot, int k, const Fmt& f) {
    const uint8_t* ub = p.u + slot * f.UB;
    const int bit = k * f.wbits, by = bit >> 3, off = bit & 7;
    uint32_t v = ub[by] >> off;
    if (off + f.wbits > 8) v |= (uint32_t)ub[by + 1] << (8 - off);
    const int up = sext(v, f.wbits);
    const uint8_t* sb = p.h + slot * f.SB;
    const int sbit = (k >> f.lg_gs) * f.u, sby = sbit >> 3, soff = sbit & 7;
    uint32_t w = sb[sby] >> soff;
    if (soff + f.u > 8) w |= (uint32_t)sb[sby + 1] << (8 - soff);
    const int sh = sext(w, f.u);
    return (float)(up * (1 << f.u) + sh) * exp2_int((int)p.s[slot]);
}

}  // namespace msaq
