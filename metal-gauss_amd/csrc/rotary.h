// Angles of rotary positions, for the kernels that turn heads by them. Internal
// header.
#pragma once

#include "mg_types.h"

namespace mg {

// Which axis of a token's position each pair goes by, handed over in the
// kernel's arguments. Pairs past this many go by equal runs alone.
constexpr int kAxisPairs = 256;
struct AxisTable {
    uint8_t axis[kAxisPairs];
};

// The axis of every pair: as the caller says (axis_of, `pairs` values below
// `axes`), or equal runs (NULL). False where a value is out of range.
inline bool fill_axes(AxisTable &t, const uint8_t *axis_of, int pairs, int axes) {
    for (int i = 0; i < pairs; ++i) {
        t.axis[i] = axis_of ? axis_of[i] : (uint8_t)(i / (pairs / axes));
        if (t.axis[i] >= axes) return false;
    }
    return true;
}

// Cosine and sine (times `sign`) of position * frequency. The angle's whole turns
// leave it in float64.
__device__ __forceinline__ float2 turn_of(double position, double frequency, float sign) {
    const double turns = position * frequency * 0.15915494309189533577;
    float sn, cs;
    // turns - rint(turns) in [-1/2, 1/2]; sincospi takes half turns.
    sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
    return make_float2(cs, sign * sn);
}

}  // namespace mg
