// The 4-bit KV cache's layout and number format, on the device.
//
// A value is a 4-bit float (e2m1) times a power of two shared by 32
// consecutive dimensions of a head (all 16 where hd is 16).  The scale s is
// the smallest power of two with max|x| <= 7 s: at 7 s the clamp to the
// largest magnitude, 6, is off by as much as rounding between 4 and 6 is, so
// no value is off by more than half the spacing of the codes around it.
// s is kept within [2^-100, 2^125]: 6 s and every step below are finite
// normal f32, and smaller groups read as zeros.  A group that holds an
// infinity or a NaN gets the scale byte 255 and reads back as NaN.
//
// x / s is exact (s a power of two) and so are the thresholds, so the codes
// follow from the definition without a rounding of ours; code * s has at most
// two significant bits and is exact in bf16.
#pragma once

#include "common.cuh"
#include "kernels.hpp"

namespace tmg {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kKv4BadScale = 255, kKv4MaxScale = 252;

// One sequence's planes: a row is (kv head, position).
template <int HD>
struct Kv4Planes {
    static constexpr int NG = kv4_groups(HD);
    uint8_t *kc, *vc;  // [nkv][cap][HD / 2] codes, the even dimension in the low half byte
    uint8_t *ks, *vs;  // [nkv][cap][NG] scale bytes
    __device__ Kv4Planes(const Kv4Cache &c, int seq) {
        const size_t rows = (size_t)c.nkv * c.cap;
        kc = c.data + (size_t)seq * c.seq_stride;
        vc = kc + rows * (HD / 2);
        ks = vc + rows * (HD / 2);
        vs = ks + rows * NG;
    }
};

// A sequence's first row position, or -1 where it takes no part: an idle
// slot, or rows that would pass the capacity.
__device__ __forceinline__ int kv4_pos(int p, int rows, uint32_t cap) {
    return p < 0 || (int64_t)p + rows > (int64_t)cap ? -1 : p;
}
__device__ __forceinline__ int kv4_pos(const int *pos_dev, int pos, int seq, int rows, uint32_t cap) {
    return kv4_pos(pos_dev ? pos_dev[seq] : pos, rows, cap);
}

// Scale byte of a group whose largest |x| has these f32 bits.
__device__ __forceinline__ uint32_t kv4_scale_byte(uint32_t bits) {
    const int e = (int)(bits >> 23) - 2 + ((bits & 0x7FFFFFu) > 0x600000u);
    return bits >= 0x7F800000u ? kKv4BadScale : (uint32_t)min(max(e, 27), 252);
}

// The f32 scale of a byte; infinity, for a marked group, makes the conversions
// give NaN.
__device__ __forceinline__ float kv4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight consecutive dimensions of a row, of which LANES consecutive lanes
// hold a group: their codes, and the group's scale byte in every lane.
template <int LANES>
__device__ __forceinline__ uint32_t kv4_quantize8(const float (&x)[8], uint32_t *byte) {
    static_assert(LANES == 2 || LANES == 4, "a group is two or four lanes");
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    m = max(m, dpp_mov<kDppXor1>(m));
    if (LANES == 4) m = max(m, dpp_mov<kDppXor2>(m));
    const uint32_t b = kv4_scale_byte(m);
    *byte = b;
    if (b == kKv4BadScale) return 0;
    const float s = kv4_scale(b);
    // v_cvt_scalef32_pk_fp4_f32: x / s to the nearest code, halves to even,
    // saturating at 6
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], s, 3);
    return c;
}

}  // namespace tmg
