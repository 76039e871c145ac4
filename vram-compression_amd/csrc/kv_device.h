// What the key-value cache's kernels share: the 4-bit format's conversions and
// the checks of a cache's descriptor.  Everything sits in an anonymous
// namespace: each .hip file is a translation unit of its own.  The layout is
// documented in include/vramc_kv.h.
#ifndef VRAMC_KV_DEVICE_H
#define VRAMC_KV_DEVICE_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/vramc_kv.h"

namespace {

constexpr int kMxBlock = 32;  // values to a scale byte
constexpr int64_t kMaxTokens = 1 << 29;  // that a row of the table has room for
constexpr int64_t kMaxThreads = UINT32_MAX;  // of a launch

template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// Two values of a byte of codes (the lower half first) times 2^(scale - 127).
template <typename T, int BYTE>
__device__ __forceinline__ uint32_t mx_pair(uint32_t codes, uint32_t scale) {
    const float unit = __uint_as_float(scale << 23);  // the conversion reads the exponent alone
    if constexpr (std::is_same_v<T, __bf16>)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, unit, BYTE));
    else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, unit, BYTE));
}
template <typename T>
__device__ __forceinline__ uint32_t mx_pair_at(uint32_t codes, uint32_t scale, int byte) {
    switch (byte) {  // constant after unrolling
        case 0: return mx_pair<T, 0>(codes, scale);
        case 1: return mx_pair<T, 1>(codes, scale);
        case 2: return mx_pair<T, 2>(codes, scale);
        default: return mx_pair<T, 3>(codes, scale);
    }
}

// The sum over a wave's lanes up to and with this one: within rows of 16 lanes,
// then each row's last lane into the rows behind it.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);   // row_shr:2
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);   // row_shr:4
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);   // row_shr:8
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
    return x;
}

// The checks of every entry point.
inline int check_cache(const vramc_kv_cache* c) {
    if (!c || !c->k || !c->v || c->pages <= 0 || c->kv_heads <= 0) return RANS_EARG;
    switch (c->page_size) {
        case 16: case 32: case 64: case 128: case 256: break;
        default: return RANS_EUNSUPPORTED;
    }
    switch (c->head_dim) {
        case 64: case 96: case 128: case 192: case 256: break;
        default: return RANS_EUNSUPPORTED;
    }
    if (c->dtype != RANS_X_F32 && c->dtype != RANS_X_BF16 && c->dtype != RANS_X_F16)
        return RANS_EUNSUPPORTED;
    if (c->mx && c->dtype == RANS_X_F32) return RANS_EUNSUPPORTED;
    if (c->mx && (!c->k_scale || !c->v_scale)) return RANS_EARG;
    if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->mass | (uintptr_t)c->position) % 16) return RANS_EARG;
    if (!c->mass != !c->position) return RANS_EARG;
    return 0;
}

}  // namespace

#endif  // VRAMC_KV_DEVICE_H
