// Causal GQA attention over the 4-bit KV cache (the format: kv4.cuh).
//
//   S = q K^T / sqrt(hd),  P = softmax of S over positions 0 .. the row's own,
//   O = P V
//
// Scores.  The cache's codes and scale bytes are what
// v_mfma_scale_f32_16x16x128_f8f6f4 takes, so keys go from memory into the
// matrix instruction as they are.  The query, scaled to log2 units, is the
// sum of six 6-bit floats (e2m3) a dimension: part n holds what the parts
// before it leave, at a sixteenth of the scale (each rounding leaves at most
// a quarter of its part's step of 1/8 .. 1/2), so 2^-24 of the largest of 32
// dimensions is left out, as f32 itself would.  A 4-bit and a 6-bit operand
// run at four times the bf16 rate: six parts cost half of three bf16 ones.
//
// Values.  A value's scale belongs to a (position, 32 dimensions), which the
// instruction cannot take along its contracted axis, so values are widened to
// bf16 (exact) and multiplied on the bf16 MFMA with P as three bf16 parts
// (2^-26 of a probability left out).
//
// Layouts (lane l: r = l & 15, lg = l >> 4).  S^T = K Q^T: lane (r, lg)
// supplies dims 32 lg .. +31 of key r and of column r, and receives keys
// 4 lg + i of column r.  O^T = V^T P^T: the contraction's slot (lg, j) is the
// key 16 (j / 4) + 4 lg + j % 4 of a unit of 32, which is what the two score
// tiles left in this lane, so P needs no exchange between lanes.  V^T's row r
// of tile t is the dimension r HD / 16 + t: a lane reads HD / 16 consecutive
// dimensions of its eight keys.
//
// A column is a (query row, query head) pair of one KV head: column c of a
// sequence is row c / group, head c % group.
#include <algorithm>

#include "kv4.cuh"

namespace tmg {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x6 __attribute__((ext_vector_type(6)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x32 __attribute__((ext_vector_type(32)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kQParts = 6;

// A column's query in a lane: 128-dimension halves, parts, scale bytes.
template <int HD>
struct Kv4Query {
    static constexpr int KH = (HD + 127) / 128;
    u32x6 part[KH][kQParts];
    uint32_t scale[KH][2];  // part n's byte: byte n & 3 of word n >> 2

    // src: the column's HD floats, or null for a column that does not exist
    __device__ __forceinline__ void load(const float *src, int lg, float mul) {
#pragma unroll
        for (int h = 0; h < KH; h++) {
            f32x16 ev, od;
#pragma unroll
            for (int i = 0; i < 16; i++) ev[i] = od[i] = 0.f;
            const int d0 = 128 * h + 32 * lg;
            if (src && d0 < HD) {
#pragma unroll
                for (int i = 0; i < (HD < 32 ? HD : 32) / 4; i++) {
                    const f32x4 v = *reinterpret_cast<const f32x4 *>(src + d0 + 4 * i);
                    ev[2 * i] = v.x * mul;
                    od[2 * i] = v.y * mul;
                    ev[2 * i + 1] = v.z * mul;
                    od[2 * i + 1] = v.w * mul;
                }
            }
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 16; i++)
                m = max(m, max(__float_as_uint(ev[i]) & 0x7FFFFFFFu, __float_as_uint(od[i]) & 0x7FFFFFFFu));
            // the largest magnitude within (3.75, 7.5] of the first part's scale
            int e = (int)(m >> 23) - 2 + ((m & 0x7FFFFFu) > 0x700000u);
            e = min(max(e, 27), 252);
            const bool bad = m >= 0x7F800000u;
            scale[h][0] = bad ? 0xFFFFFFFFu : (uint32_t)(e | (e - 4) << 8 | (e - 8) << 16 | (e - 12) << 24);
            scale[h][1] = bad ? 0xFFFFFFFFu : (uint32_t)((e - 16) | (e - 20) << 8);
#pragma unroll
            for (int n = 0; n < kQParts; n++) {
                const float s = __uint_as_float((uint32_t)(e - 4 * n) << 23);
                part[h][n] = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(ev, od, s);
                if (n + 1 < kQParts) {
                    const f32x32 v = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(part[h][n], s);
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        ev[i] -= v[2 * i];
                        od[i] -= v[2 * i + 1];
                    }
                }
            }
        }
    }
};

template <int HD>
struct Kv4Key {
    static constexpr int KH = (HD + 127) / 128;
    u32x4 code[KH];
    uint32_t scale[KH];

    __device__ __forceinline__ void load(const Kv4Planes<HD> &pl, size_t row, int lg) {
#pragma unroll
        for (int h = 0; h < KH; h++) {
            code[h] = u32x4{0, 0, 0, 0};
            scale[h] = 127;
            if (128 * h + 32 * lg < HD) {
                const uint8_t *p = pl.kc + row * (HD / 2) + 64 * h + 16 * lg;
                if constexpr (HD == 16) {
                    const uint2 c = *reinterpret_cast<const uint2 *>(p);
                    code[h].x = c.x;
                    code[h].y = c.y;
                } else {
                    code[h] = *reinterpret_cast<const u32x4 *>(p);
                }
                scale[h] = pl.ks[row * kv4_groups(HD) + 4 * h + lg];
            }
        }
    }
};

template <int N, int HD>
__device__ __forceinline__ void score_part(const i32x8 &k, uint32_t ks, const Kv4Query<HD> &q, int h, f32x4 &s) {
    const u32x6 p = q.part[h][N];
    const i32x8 b = {(int)p[0], (int)p[1], (int)p[2], (int)p[3], (int)p[4], (int)p[5], 0, 0};
    s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, b, s, 4 /* fp4 */, 2 /* fp6 e2m3 */, 0, (int)ks, N & 3,
                                                         (int)q.scale[h][N >> 2]);
}

// Scores (log2 units) of 16 keys and 16 columns; the smallest parts first.
template <int HD>
__device__ __forceinline__ f32x4 kv4_scores(const Kv4Key<HD> &k, const Kv4Query<HD> &q) {
    f32x4 s{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < Kv4Key<HD>::KH; h++) {
        const i32x8 a = {(int)k.code[h].x, (int)k.code[h].y, (int)k.code[h].z, (int)k.code[h].w, 0, 0, 0, 0};
        score_part<5>(a, k.scale[h], q, h, s);
        score_part<4>(a, k.scale[h], q, h, s);
        score_part<3>(a, k.scale[h], q, h, s);
        score_part<2>(a, k.scale[h], q, h, s);
        score_part<1>(a, k.scale[h], q, h, s);
        score_part<0>(a, k.scale[h], q, h, s);
    }
    return s;
}

// A lane's HD / 16 dimensions of its eight keys of a unit of 32.
template <int HD>
struct Kv4Values {
    static constexpr int DPL = HD / 16;                // dimensions, tiles
    static constexpr int W = HD == 256 ? 2 : 1;        // words of codes a key
    uint32_t code[8][W];
    uint32_t scale[8];

    // row0: the head's first row; keys past `last` repeat it
    __device__ __forceinline__ void load(const Kv4Planes<HD> &pl, size_t row0, int key0, int last, int r, int lg) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const size_t row = row0 + min(key0 + 16 * (j >> 2) + 4 * lg + (j & 3), last);
            const uint8_t *p = pl.vc + row * (HD / 2);
            if constexpr (HD == 256) {
                const uint2 c = *reinterpret_cast<const uint2 *>(p + 8 * r);
                code[j][0] = c.x;
                code[j][1] = c.y;
            } else if constexpr (HD == 128) {
                code[j][0] = *reinterpret_cast<const uint32_t *>(p + 4 * r);
            } else if constexpr (HD == 64) {
                code[j][0] = *reinterpret_cast<const uint16_t *>(p + 2 * r);
            } else if constexpr (HD == 32) {
                code[j][0] = p[r];
            } else {
                code[j][0] = (uint32_t)p[r >> 1] >> (4 * (r & 1));
            }
            scale[j] = pl.vs[row * kv4_groups(HD) + r * DPL / 32];
        }
    }

    // Whether some group of this lane's keys is marked as not finite; its
    // values are then taken as finite ones (a masked key's weight of zero
    // must not meet a NaN), and nan_values puts the NaN where it belongs.
    __device__ __forceinline__ bool take_bad(uint32_t *bits) {
        uint32_t b = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (scale[j] == kKv4BadScale) {
                b |= 1u << j;
                scale[j] = 127;
            }
        }
        *bits = b;
        return __builtin_amdgcn_ballot_w64(b != 0) != 0;
    }

    // The bf16 operands of two neighbouring tiles: dimensions 2 i and 2 i + 1
    // of the lane's, eight keys each.
    template <int I>
    __device__ __forceinline__ void widen(u32x4 &even, u32x4 &odd) const {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            w[j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(
                                                    code[j][I / 4], kv4_scale(scale[j]), I & 3));
#pragma unroll
        for (int j = 0; j < 4; j++) {
            even[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x05040100u);
            odd[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x07060302u);
        }
    }
};

// P as bf16 parts, each what the ones before leave.
template <int PARTS>
__device__ __forceinline__ void split_p(const float (&p)[8], bf16x8 (&out)[PARTS]) {
    float rest[8];
#pragma unroll
    for (int j = 0; j < 8; j++) rest[j] = p[j];
#pragma unroll
    for (int n = 0; n < PARTS; n++) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            out[n][j] = (__bf16)rest[j];
            rest[j] -= (float)out[n][j];
        }
    }
}

template <int PARTS>
__device__ __forceinline__ f32x4 mfma_pv(const u32x4 &v, const bf16x8 (&p)[PARTS], f32x4 o) {
#pragma unroll
    for (int n = PARTS - 1; n >= 0; n--)
        o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v), p[n], o, 0, 0, 0);
    return o;
}

// o += V^T P^T of a unit of 32 keys.
template <int HD, int PARTS, int I = 0>
__device__ __forceinline__ void kv4_values(const Kv4Values<HD> &v, const bf16x8 (&p)[PARTS], f32x4 (&o)[HD / 16]) {
    if constexpr (2 * I < HD / 16) {
        u32x4 even, odd;
        v.template widen<I>(even, odd);
        o[2 * I] = mfma_pv(even, p, o[2 * I]);
        if constexpr (2 * I + 1 < HD / 16) o[2 * I + 1] = mfma_pv(odd, p, o[2 * I + 1]);
        kv4_values<HD, PARTS, I + 1>(v, p, o);
    }
}

// NaN into the outputs of the columns that see a marked group's key: lane
// (r, lg) holds dimensions (4 lg + i) HD / 16 + t of column r, which are those
// of the lanes (4 lg + i, any) of `bits`.
template <int HD>
__device__ __forceinline__ void nan_values(uint32_t bits, int key0, int qpos, int lg, f32x4 (&o)[HD / 16]) {
#pragma unroll 1
    for (int j = 0; j < 8; j++) {
        const unsigned long long marked = __builtin_amdgcn_ballot_w64((bits >> j) & 1);
#pragma unroll 1
        for (int kl = 0; kl < 4; kl++) {
            if (key0 + 16 * (j >> 2) + 4 * kl + (j & 3) > qpos) continue;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if ((marked >> (16 * kl + 4 * lg + i)) & 1)
#pragma unroll
                    for (int t = 0; t < HD / 16; t++) o[t][i] = __builtin_nanf("");
        }
    }
}

// Running softmax state of a lane's column over the keys its wavefront took.
template <int HD>
struct Kv4State {
    float m = -INFINITY, l = 0.f;
    f32x4 o[HD / 16];
    __device__ Kv4State() {
#pragma unroll
        for (int t = 0; t < HD / 16; t++) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // The scores of a unit's two key tiles become weights.  The maximum is
    // raised in steps of at least 2^8 only: weights up to 2^8 cost no
    // precision in f32, and most units then leave the sums as they are.
    __device__ __forceinline__ void weights(const f32x4 (&s)[2], float (&p)[8]) {
        float mx = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
        mx = fmaxf(mx, fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = max_xor16_32(mx);
        const bool raise = mx > m + 8.0f;
        if (__builtin_amdgcn_ballot_w64(raise)) {
            const float corr = raise ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
            m = raise ? mx : m;
            l *= corr;
#pragma unroll
            for (int t = 0; t < HD / 16; t++) o[t] *= corr;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            p[j] = __builtin_amdgcn_exp2f(s[j >> 2][j & 3] - ref);
            l += p[j];
        }
    }
};

// An output element, as f32 or as the split-bf16 planes of a following GEMM.
__device__ __forceinline__ void kv4_store(const Kv4AttnArgs &a, int seq, int row, int d, float v) {
    const size_t i = ((size_t)seq * a.rows + row) * a.out_stride + d;
    if (a.out) a.out[i] = v;
    if (a.out_hi) split_bf16(v, a.out_hi + i, a.out_lo + i);
}

// The blocks [b0, b1) of nb that split `sp` takes of `active`.
__device__ __forceinline__ int split_begin(int nb, int sp, int active) { return (int)((int64_t)nb * sp / active); }

// Few columns: a workgroup owns a tile of 16 columns and a run of blocks of
// 128 keys, of which each wavefront takes a unit of 32, with a softmax state
// of its own; the wavefronts are merged through LDS, the runs (splits) by
// kv4_combine_kernel.
//
// Bound by the latency of its loads and of the merge for one sequence, by the
// cache's bytes for many.
template <int HD>
__global__ __launch_bounds__(kBlock, 2) void kv4_attn_rows_kernel(const Kv4AttnArgs a) {
    constexpr int DPL = HD / 16, PAD = 4;
    __shared__ __attribute__((aligned(16))) float s_o[4][16][HD + PAD];
    __shared__ float s_m[4][16], s_l[4][16];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, r = lane & 15, lg = lane >> 4;
    const int group = a.nq / a.c.nkv, ncol = a.rows * group, ntile = (ncol + 15) / 16;
    const int g = (int)(blockIdx.x % (unsigned)a.c.nkv);
    unsigned rest = blockIdx.x / (unsigned)a.c.nkv;
    const int sp = (int)(rest % (unsigned)a.nsplit);
    rest /= (unsigned)a.nsplit;
    const int tile = (int)(rest % (unsigned)ntile), seq = (int)(rest / (unsigned)ntile);
    const int cols = min(16, ncol - 16 * tile);
    const int pos = kv4_pos(a.pos_dev, a.pos, seq, a.rows, a.c.cap);
    const int row_r = (16 * tile + min(r, cols - 1)) / group, head_r = (16 * tile + min(r, cols - 1)) % group;
    const int last = pos + (16 * tile + cols - 1) / group;  // the tile's last position
    const int nb = pos < 0 ? 0 : last / kKv4Block + 1;
    const int active = min(a.nsplit, nb);
    if (sp >= max(active, 1) || (pos < 0 && a.nsplit > 1)) return;  // idle rows of split launches: the merge's

    Kv4State<HD> st;
    if (pos >= 0) {
        const Kv4Planes<HD> pl(a.c, seq);
        const size_t row0 = (size_t)g * a.c.cap;
        const int qpos = r < cols ? pos + row_r : -1;
        const int first_pos = pos + 16 * tile / group;
        const int b1 = split_begin(nb, sp + 1, active);
        Kv4Key<HD> k[2];
        Kv4Values<HD> v;
        auto load = [&](int key0) {
            k[0].load(pl, row0 + min(key0 + r, last), lg);
            k[1].load(pl, row0 + min(key0 + 16 + r, last), lg);
            v.load(pl, row0, key0, last, r, lg);
        };
        int key0 = split_begin(nb, sp, active) * kKv4Block + 32 * wave;
        const int end = min(b1 * kKv4Block, last + 1);
        if (key0 < end) load(key0);
        Kv4Query<HD> q;
        q.load(r < cols ? a.q + ((size_t)seq * a.rows + row_r) * a.q_stride + (size_t)(g * group + head_r) * HD : nullptr,
               lg, a.scale * 1.4426950408889634f);
        for (; key0 < end; key0 += kKv4Block) {
            f32x4 s[2] = {kv4_scores(k[0], q), kv4_scores(k[1], q)};
            Kv4Values<HD> vn = v;
            if (key0 + kKv4Block < end) load(key0 + kKv4Block);
            if (key0 + 31 > first_pos || cols < 16) {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (key0 + 16 * (j >> 2) + 4 * lg + (j & 3) > qpos) s[j >> 2][j & 3] = -INFINITY;
            }
            float p[8];
            st.weights(s, p);
            bf16x8 pp[3];
            split_p(p, pp);
            uint32_t bad;
            const bool any_bad = vn.take_bad(&bad);
            kv4_values(vn, pp, st.o);
            if (any_bad) nan_values<HD>(bad, key0, qpos, lg, st.o);
        }
    }
    // the wavefronts' states
    st.l = add_xor32(add_xor16(st.l));
    if (r < cols) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int d = 0; d < DPL; d++) s_o[wave][r][(4 * lg + i) * DPL + d] = st.o[d][i];
        if (lg == 0) {
            s_m[wave][r] = st.m;
            s_l[wave][r] = st.l;
        }
    }
    __syncthreads();
    const size_t pbase = ((((size_t)seq * ntile + tile) * a.c.nkv + g) * a.nsplit + sp) * a.part_cols;
    for (int idx = t; idx < cols * HD; idx += kBlock) {
        const int c = idx / HD, d = idx % HD;
        float M = s_m[0][c];
#pragma unroll
        for (int w = 1; w < 4; w++) M = fmaxf(M, s_m[w][c]);
        float L = 0.f, O = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            // a wavefront without a finite maximum still brings its sums: they
            // are zeros, or NaN
            const float f = s_m[w][c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[w][c] - M);
            L = fmaf(s_l[w][c], f, L);
            O = fmaf(s_o[w][c][d], f, O);
        }
        if (active <= 1) {
            const int row = (16 * tile + c) / group, h = (16 * tile + c) % group;
            kv4_store(a, seq, row, (g * group + h) * HD + d, L == 0.f ? 0.f : O / L);
        } else {
            a.part[(pbase + c) * HD + d] = O;
            if (d == 0) {
                a.part_ml[(pbase + c) * 2] = M;
                a.part_ml[(pbase + c) * 2 + 1] = L;
            }
        }
    }
}

// Merge of the splits of a tile of columns: workgroup (column, (sequence,
// tile, KV head)).
__global__ __launch_bounds__(kBlock) void kv4_combine_kernel(const Kv4AttnArgs a) {
    const int group = a.nq / a.c.nkv, ncol = a.rows * group, ntile = (ncol + a.tile_cols - 1) / a.tile_cols;
    const int g = (int)(blockIdx.x % (unsigned)a.c.nkv);
    unsigned rest = blockIdx.x / (unsigned)a.c.nkv;
    const int tile = (int)(rest % (unsigned)ntile), seq = (int)(rest / (unsigned)ntile);
    const int cols = min(a.tile_cols, ncol - a.tile_cols * tile);
    const int c = blockIdx.y;
    if (c >= cols) return;
    const int pos = kv4_pos(a.pos_dev, a.pos, seq, a.rows, a.c.cap);
    const int nb = pos < 0 ? 0 : (pos + (a.tile_cols * tile + cols - 1) / group) / kKv4Block + 1;
    const int active = min(a.nsplit, nb);
    if (active == 1) return;  // written by the split itself
    const int row = (a.tile_cols * tile + c) / group, h = (a.tile_cols * tile + c) % group;
    const size_t base = (((size_t)seq * ntile + tile) * a.c.nkv + g) * a.nsplit * a.part_cols + c;
    for (int d = threadIdx.x; d < a.c.hd; d += kBlock) {
        float M = -INFINITY, L = 0.f, O = 0.f;
        for (int s = 0; s < active; s++) M = fmaxf(M, a.part_ml[(base + (size_t)s * a.part_cols) * 2]);
        for (int s = 0; s < active; s++) {
            const size_t p = base + (size_t)s * a.part_cols;
            const float m = a.part_ml[p * 2], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
            L = fmaf(a.part_ml[p * 2 + 1], f, L);
            O = fmaf(a.part[p * a.c.hd + d], f, O);
        }
        kv4_store(a, seq, row, (g * group + h) * a.c.hd + d, L == 0.f ? 0.f : O / L);
    }
}

}  // namespace

Kv4Plan plan_kv4_attn(const Kv4Cache &c, int rows, int nq, uint32_t ctx) {
    Kv4Plan p{};
    const int64_t ncol = (int64_t)rows * (nq / c.nkv);
    p.tile_cols = 16;
    p.part_cols = (int)std::min<int64_t>(p.tile_cols, ncol);
    p.tiles = (ncol + p.tile_cols - 1) / p.tile_cols * c.nkv * c.n_seq;
    const int64_t nb = ((int64_t)ctx + kKv4Block - 1) / kKv4Block;
    p.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({nb, (kKv4Workgroups + p.tiles - 1) / p.tiles, kKv4MaxSplits}));
    return p;
}

size_t kv4_attn_part_floats(const Kv4Cache &c, int rows, int nq) {
    // the number of splits does not fall as the context grows
    const Kv4Plan p = plan_kv4_attn(c, rows, nq, c.cap);
    return p.nsplit == 1 ? 0 : (size_t)p.tiles * p.nsplit * p.part_cols * (c.hd + 2);
}

hipError_t launch_kv4_attn(Kv4AttnArgs a, float *ws, hipStream_t s) {
    const uint32_t ctx = a.pos_dev ? a.c.cap : (uint32_t)(a.pos + a.rows);
    const Kv4Plan p = plan_kv4_attn(a.c, a.rows, a.nq, ctx);
    if (p.tiles * p.nsplit > 0x7fffffff || (p.nsplit > 1 && !ws)) return hipErrorInvalidValue;
    a.nsplit = p.nsplit;
    a.tile_cols = p.tile_cols;
    a.part_cols = p.part_cols;
    a.part = ws;
    a.part_ml = ws + (size_t)p.tiles * p.nsplit * p.part_cols * a.c.hd;
    const dim3 grid((unsigned)(p.tiles * p.nsplit));
    switch (a.c.hd) {
        case 16: hipLaunchKernelGGL((kv4_attn_rows_kernel<16>), grid, dim3(kBlock), 0, s, a); break;
        case 32: hipLaunchKernelGGL((kv4_attn_rows_kernel<32>), grid, dim3(kBlock), 0, s, a); break;
        case 64: hipLaunchKernelGGL((kv4_attn_rows_kernel<64>), grid, dim3(kBlock), 0, s, a); break;
        case 128: hipLaunchKernelGGL((kv4_attn_rows_kernel<128>), grid, dim3(kBlock), 0, s, a); break;
        case 256: hipLaunchKernelGGL((kv4_attn_rows_kernel<256>), grid, dim3(kBlock), 0, s, a); break;
        default: return hipErrorInvalidValue;
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.nsplit == 1) return e;
    hipLaunchKernelGGL(kv4_combine_kernel, dim3((unsigned)p.tiles, p.part_cols), dim3(kBlock), 0, s, a);
    return hipGetLastError();
}
}  // namespace tmg
