// Rows written into the 4-bit KV cache and read back as f32 (the format:
// kv4.cuh).  A lane takes eight consecutive dimensions of a row: 32 bytes of
// f32 on one side, four bytes of codes on the other; hd / 8 lanes are a row
// of a head, and consecutive rows of one head are consecutive lanes, so the
// codes of a workgroup are one contiguous run of the cache.  The cache's rows
// are head by head, as the attention reads them; the f32 rows are position by
// position, as the projections write them.
//
// Bound by the f32 rows' traffic, 4 bytes a value against 0.53: 8192 rows of 8
// heads of 128 (76 MB) are written in 13-19 us (4.0-5.8 TB/s) and read back in
// 16-22 us (3.5-4.8 TB/s); a row or a few by the launch, 2.6 us.
#include "kv4.cuh"

namespace tmg {
namespace {

// Grid: x over the lanes of a head's rows, y = 2 g + (0 keys, 1 values), z =
// sequence.
template <int HD>
__global__ __launch_bounds__(kBlock) void kv4_write_kernel(const Kv4WriteArgs a) {
    constexpr int LPR = HD / 8, NG = kv4_groups(HD), LPG = LPR / NG;
    const int seq = blockIdx.z, g = blockIdx.y >> 1;
    const bool val = blockIdx.y & 1;
    const int p = kv4_pos(a.pos_dev, a.pos, seq, a.rows, a.c.cap);
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    const int64_t t = i / LPR;
    const int lane = (int)(i % LPR);
    if (p < 0 || t >= a.rows) return;  // whole groups leave together
    const float *src = (val ? a.v : a.k) + ((size_t)seq * a.rows + t) * a.row_stride + (size_t)g * HD + lane * 8;
    float x[8];
    *reinterpret_cast<f32x4 *>(x) = *reinterpret_cast<const f32x4 *>(src);
    *reinterpret_cast<f32x4 *>(x + 4) = *reinterpret_cast<const f32x4 *>(src + 4);
    uint32_t byte;
    const uint32_t code = kv4_quantize8<LPG>(x, &byte);
    const Kv4Planes<HD> pl(a.c, seq);
    const size_t row = (size_t)g * a.c.cap + p + t;
    *reinterpret_cast<uint32_t *>((val ? pl.vc : pl.kc) + row * (HD / 2) + lane * 4) = code;
    if (lane % LPG == 0) (val ? pl.vs : pl.ks)[row * NG + lane / LPG] = (uint8_t)byte;
}

// The same grid over the planes that are asked for.
template <int HD>
__global__ __launch_bounds__(kBlock) void kv4_read_kernel(const Kv4ReadArgs a) {
    constexpr int LPR = HD / 8, NG = kv4_groups(HD), LPG = LPR / NG;
    const int seq = blockIdx.z, g = blockIdx.y >> 1;
    const bool val = blockIdx.y & 1;
    float *const plane = val ? a.v : a.k;
    const int p = kv4_pos(a.pos_dev, a.pos, seq, a.rows, a.c.cap);
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    const int64_t t = i / LPR;
    const int lane = (int)(i % LPR);
    if (!plane || t >= a.rows) return;
    f32x4 lo{0.f, 0.f, 0.f, 0.f}, hi{0.f, 0.f, 0.f, 0.f};
    if (p >= 0) {
        const Kv4Planes<HD> pl(a.c, seq);
        const size_t row = (size_t)g * a.c.cap + p + t;
        const uint32_t c = *reinterpret_cast<const uint32_t *>((val ? pl.vc : pl.kc) + row * (HD / 2) + lane * 4);
        const uint32_t b = (val ? pl.vs : pl.ks)[row * NG + lane / LPG];
        const float s = kv4_scale(b > kKv4MaxScale ? kKv4BadScale : b);
        const f32x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0);
        const f32x2 v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
        const f32x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2);
        const f32x2 v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
        lo = f32x4{v0.x, v0.y, v1.x, v1.y};
        hi = f32x4{v2.x, v2.y, v3.x, v3.y};
    }
    float *dst = plane + ((size_t)seq * a.rows + t) * a.row_stride + (size_t)g * HD + lane * 8;
    *reinterpret_cast<f32x4 *>(dst) = lo;
    *reinterpret_cast<f32x4 *>(dst + 4) = hi;
}

dim3 rows_grid(const Kv4Cache &c, int rows) {
    const int64_t lanes = (int64_t)rows * (c.hd / 8);
    return dim3((unsigned)((lanes + kBlock - 1) / kBlock), 2 * c.nkv, c.n_seq);
}

}  // namespace

hipError_t launch_kv4_write(const Kv4WriteArgs &a, hipStream_t s) {
    const dim3 grid = rows_grid(a.c, a.rows);
    switch (a.c.hd) {
        case 16: hipLaunchKernelGGL((kv4_write_kernel<16>), grid, dim3(kBlock), 0, s, a); break;
        case 32: hipLaunchKernelGGL((kv4_write_kernel<32>), grid, dim3(kBlock), 0, s, a); break;
        case 64: hipLaunchKernelGGL((kv4_write_kernel<64>), grid, dim3(kBlock), 0, s, a); break;
        case 128: hipLaunchKernelGGL((kv4_write_kernel<128>), grid, dim3(kBlock), 0, s, a); break;
        case 256: hipLaunchKernelGGL((kv4_write_kernel<256>), grid, dim3(kBlock), 0, s, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4ReadArgs &a, hipStream_t s) {
    const dim3 grid = rows_grid(a.c, a.rows);
    switch (a.c.hd) {
        case 16: hipLaunchKernelGGL((kv4_read_kernel<16>), grid, dim3(kBlock), 0, s, a); break;
        case 32: hipLaunchKernelGGL((kv4_read_kernel<32>), grid, dim3(kBlock), 0, s, a); break;
        case 64: hipLaunchKernelGGL((kv4_read_kernel<64>), grid, dim3(kBlock), 0, s, a); break;
        case 128: hipLaunchKernelGGL((kv4_read_kernel<128>), grid, dim3(kBlock), 0, s, a); break;
        case 256: hipLaunchKernelGGL((kv4_read_kernel<256>), grid, dim3(kBlock), 0, s, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace tmg
