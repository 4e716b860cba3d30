// The paged key / value cache: layout, addresses and the codes of its three types.
//
// One buffer holds the keys, another the values, of n_pages pages of page_tokens tokens. Plane 0 holds the codes
// [page][kv head][token of the page][row], plane 1 (Q8_0, Q4_0) the f16 block scales [page][kv head][token][head_dim / 32].
// A slot is page · page_tokens + token of the page. A row of a head is head_dim elements: F16 as they are, Q8_0 one int8 per
// element, Q4_0 16 bytes per block of 32 (byte j: element j low, element 16 + j high, both biased by 8). An element stands
// for scale · code rounded to f16, so every type reaches the matrix cores as f16 without a further rounding.
#pragma once

#include "common.h"
#include "fastdiv.h"

namespace jamhip {

__host__ __device__ constexpr int kv_row_bytes(int type, int dim) { return type == F16 ? 2 * dim : type == Q8_0 ? dim : dim / 2; }
__host__ __device__ constexpr int kv_scales(int type, int dim) { return type == F16 ? 0 : dim / 32; }

struct KvView {
    uint8_t* k;
    uint8_t* v;
    int64_t scale_off;   // byte offset of plane 1
    int kv, dim, n_pages;
    FastDiv page;        // page.d = tokens per page
    __device__ int64_t slots() const { return (int64_t) n_pages * page.d; }
    // index of (slot, head) in units of rows, slot in [0, slots())
    __device__ int64_t row(int64_t slot, int head) const {
        const int p = page.div((int) slot), t = (int) slot - p * page.d;
        return ((int64_t) p * kv + head) * page.d + t;
    }
};

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
typedef float float4_t __attribute__((ext_vector_type(4)));

JAMHIP_DEV half2_t as_half2(uint32_t v) { return __builtin_bit_cast(half2_t, v); }
JAMHIP_DEV uint32_t as_u32(half2_t v) { return __builtin_bit_cast(uint32_t, v); }

// Bytes (0, 1) or (2, 3) of w under the exponent byte 0x64: two f16 of 1024 + byte, exact.
JAMHIP_DEV half2_t bytes01_1024(uint32_t w) { return as_half2(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)); }
JAMHIP_DEV half2_t bytes23_1024(uint32_t w) { return as_half2(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)); }

// 4 int8 codes -> 4 f16 of scale · code, each product rounded once: 1024 + (code + 128) - 1152 is exact.
JAMHIP_DEV void q8_word(uint32_t w, half2_t scale, half2_t* out) {
    const half2_t bias = {(_Float16) 1152.0f, (_Float16) 1152.0f};
    const uint32_t u = w ^ 0x80808080u;
    out[0] = (bytes01_1024(u) - bias) * scale;
    out[1] = (bytes23_1024(u) - bias) * scale;
}
// the 4 low nibbles of w's bytes -> 4 f16 of scale · (nibble - 8)
JAMHIP_DEV void q4_word(uint32_t w, half2_t scale, half2_t* out) {
    const half2_t bias = {(_Float16) 1032.0f, (_Float16) 1032.0f};
    const uint32_t u = w & 0x0F0F0F0Fu;
    out[0] = (bytes01_1024(u) - bias) * scale;
    out[1] = (bytes23_1024(u) - bias) * scale;
}

// 4 consecutive elements e .. e + 3 (e % 4 == 0) of one row; `row` from KvView::row.
template <int TYPE> JAMHIP_DEV float4_t kv_load4(const uint8_t* buf, int64_t scale_off, int dim, int64_t row, int e) {
    half2_t h[2];
    if constexpr (TYPE == F16) {
        const uint2_t w = *reinterpret_cast<const uint2_t*>(buf + (row * dim + e) * 2);
        h[0] = as_half2(w[0]), h[1] = as_half2(w[1]);
    } else {
        const int nb = dim / 32;
        const _Float16 s = *reinterpret_cast<const _Float16*>(buf + scale_off + (row * nb + e / 32) * 2);
        const half2_t scale = {s, s};
        if constexpr (TYPE == Q8_0) {
            q8_word(*reinterpret_cast<const uint32_t*>(buf + row * dim + e), scale, h);
        } else {
            const int in = e % 32;
            const uint32_t w = *reinterpret_cast<const uint32_t*>(buf + row * (dim / 2) + e / 32 * 16 + in % 16);
            q4_word(in < 16 ? w : w >> 4, scale, h);
        }
    }
    return float4_t{(float) h[0][0], (float) h[0][1], (float) h[1][0], (float) h[1][1]};
}

}  // namespace jamhip
