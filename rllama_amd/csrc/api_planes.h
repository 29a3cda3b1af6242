// api_planes.h -- tensors as the kernels of long contexts and of many answers see them (entry points only).
#pragma once

#include "api_internal.h"
#include "f8.h"
#include "longctx.h"

inline rlh::PlaneRef plane_of(const rlh_tensor *t) {
    rlh::PlaneRef r{t->p, nullptr};
    if (t->dtype == RLH_Q4) r.pairs = reinterpret_cast<uint32_t *>(static_cast<char *>(t->p) + rlh::q4_pairs_offset(t->count()));
    return r;
}
inline int plane_type(const rlh_tensor *t) { return t->dtype == RLH_F16 ? rlh::kPlaneF16 : t->dtype == RLH_F32 ? rlh::kPlaneF32 : rlh::kPlaneQ4; }
inline bool holds_plane(const rlh_tensor *t) { return t->is_float() || t->dtype == RLH_Q4; }
inline rlh::EightRef eight_of(const rlh_tensor *t) {
    return {static_cast<uint8_t *>(t->p), reinterpret_cast<float *>(static_cast<char *>(t->p) + t->count()), t->dtype == RLH_F8 ? 1 : rlh::kF8Block};
}
inline bool shaped(const rlh_tensor *t, int64_t rows, int64_t cols) { return t->rows == rows && t->cols == cols; }
