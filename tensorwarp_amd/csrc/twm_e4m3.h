// A row's values in units of their block's scale, for e4m3 codes.  No device code: a host compiler takes it as it is.
#pragma once

namespace twm {

constexpr float kFp8Max = 448.0f;
// Scales from which on units_of takes the place of a division: its remainder is exact down to 2^-93
constexpr float kFp8LeastExact = 0x1p-90f;

// v / scale as f32 rounds it, or a neighbour of that on the same side of every border between two e4m3 codes, where scale is
// amax / 448, inverse 448 / amax, both rounded to f32, and |v| at most amax: the product with the inverse and one step by its remainder.
// Shown by trying it with every mantissa of amax at every border, on the five f32 values around it: none of 5.3e9 is off.  (The product
// alone puts one in seven of those on the wrong side, and of f16 rows a code in thirty thousand.)
// (A constexpr template, which either compiler takes for its side.)
template <typename Float> constexpr Float units_of(Float v, Float scale, Float inverse)
{
    const Float near = v * inverse;
    return __builtin_fmaf(__builtin_fmaf(-near, scale, v), inverse, near);
}

}  // namespace twm
