// What the kernels of the gated delta rule share (its arguments and formulas are explained in rwkv_hip.h and delta.hip).
#pragma once

#include "mixers.h"

namespace rwkv {

constexpr int DELTA_CHUNK = 64;                                 // tokens of a chunk
// A log decay below this is a decay of 0: e^-104 lies below half of fp32's least number.
constexpr float DELTA_NONE = -104.f;

// What becomes of a token: padding leaves the state as it is; a cut lets nothing of it through.
struct DeltaToken { bool real, cut; };
DEVINL DeltaToken delta_token(const int* doc, const int64_t row, const int t, const int T) {
    if (t >= T) return {false, false};
    if (doc == nullptr) return {true, false};
    const int d = doc[row + t];
    return {d >= 0, d >= 0 && t > 0 && doc[row + t - 1] != d};
}

}  // namespace rwkv
