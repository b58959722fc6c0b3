// Causal GQA attention over the 4-bit KV cache (the format: kv4.cuh).
//
//   S = q K^T / sqrt(hd),  P = softmax of S over positions 0 .. the row's own,
//   O = P V
//
// Scores.  The cache's codes and scale bytes are what
// v_mfma_scale_f32_16x16x128_f8f6f4 takes, so keys go from memory into the
// matrix instruction as they are.  The query, scaled to log2 units, is the
// sum of six 6-bit floats (e2m3) a dimension, of which the multiples of 1/8
// up to 15/8 are used: digits of the fixed-point number that the largest of 32
// dimensions scales to (-15 .. 15, then -8 .. 8 at each sixteenth of the
// scale), so 2^-24 of the largest dimension is left out, as f32 itself would.
// A 4-bit and a 6-bit operand run at four times the bf16 rate: six parts cost
// half of three bf16 ones.
//
// Values.  A value's scale belongs to a (position, 32 dimensions), which the
// instruction cannot take along its contracted axis, so values are widened to
// bf16 (exact) and multiplied on the bf16 MFMA with P as three bf16 parts
// (exact).
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
// sequence is row c / group, head c % group.  Decode steps have two or four
// columns, not the 16 of a matrix instruction; its other columns then take the
// parts of the same ones, side by side (Kv4Lanes): one instruction does the
// scores of 16 keys for two columns instead of six, and one the values'
// instead of three.
#include <algorithm>

#include "coh.cuh"
#include "kv4.cuh"

namespace tmg {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x6 __attribute__((ext_vector_type(6)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x32 __attribute__((ext_vector_type(32)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kQParts = 6, kPParts = 3;  // of a query and of a weight

// A barrier for LDS alone: loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The 16 columns of a matrix operand as C columns of 16 / C parts each: lane r
// has column r / PARTS of part r % PARTS; what does not fit goes into further
// sets.  Sums over a column's parts are then sums over PARTS neighbouring
// lanes.
template <int C>
struct Kv4Lanes {
    static constexpr int PARTS = 16 / C;
    static constexpr int QSETS = (kQParts + PARTS - 1) / PARTS, PSETS = (kPParts + PARTS - 1) / PARTS;
    // Every lane gets the sum of its column's parts, and the same bits: a
    // butterfly adds the same pairs in both of their lanes.  (The half mirror
    // is the other quad's lane here, all of whose lanes hold its sum.)
    static __device__ __forceinline__ float sum(float v) {
        static_assert(PARTS == 1 || PARTS == 4 || PARTS == 8, "one, four or eight lanes a column");
        if constexpr (PARTS >= 4) v += dpp_mov<kDppXor1>(v);
        if constexpr (PARTS >= 4) v += dpp_mov<kDppXor2>(v);
        if constexpr (PARTS >= 8) v += dpp_mov<kDppHalfMirror>(v);
        return v;
    }
};

// A column's query in a lane: 128-dimension halves, sets of parts, scale
// bytes.
template <int HD, int C>
struct Kv4Query {
    static constexpr int KH = (HD + 127) / 128, SETS = Kv4Lanes<C>::QSETS, PARTS = Kv4Lanes<C>::PARTS;
    f32x16 ev[KH], od[KH];  // the lane's even and odd dimensions, until split
    int first[KH];          // the first part's scale byte, 255 for what is not finite
    float mul[KH];          // what ev and od are still to be scaled by
    u32x6 part[KH][SETS];
    uint32_t scale[KH][(SETS + 3) / 4];  // set s's byte: byte s & 3 of word s >> 2

    // src: the column's HD floats.  Lanes past the head's dimensions repeat
    // the first ones; ready() takes them as zeros.  (No branch: a loaded value
    // that meets a constant is waited for on the spot.)
    __device__ __forceinline__ void fetch(const float *src, int lg) {
#pragma unroll
        for (int h = 0; h < KH; h++) {
            const float *p = src + (128 * h + 32 * lg < HD ? 128 * h + 32 * lg : 0);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (4 * i < HD) {
                    const f32x4 v = *reinterpret_cast<const f32x4 *>(p + 4 * i);
                    ev[h][2 * i] = v.x;
                    od[h][2 * i] = v.y;
                    ev[h][2 * i + 1] = v.z;
                    od[h][2 * i + 1] = v.w;
                } else {
                    ev[h][2 * i] = ev[h][2 * i + 1] = od[h][2 * i] = od[h][2 * i + 1] = 0.f;
                }
            }
        }
    }

    // The first parts' scales of what was fetched, times f.
    __device__ __forceinline__ void ready(float f, int lg) {
#pragma unroll
        for (int h = 0; h < KH; h++) {
            // (a NaN or an infinity times the zero marks a column that is NaN anyway)
            mul[h] = 128 * h + 32 * lg < HD ? f : 0.f;
            float m = 0.f;  // NaN where one is
#pragma unroll
            for (int i = 0; i < 16; i++)
                m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(m, fabsf(ev[h][i])), fabsf(od[h][i]));
            const uint32_t bits = __float_as_uint(m * fabsf(mul[h]));
            // the largest magnitude is at most 15/8 of the first part's scale;
            // 2^126 and more count as infinite
            first[h] = bits >= 0x7E800000u ? 255 : max((int)(bits >> 23) + ((bits & 0x7FFFFFu) > 0x700000u), 27);
        }
    }
    __device__ __forceinline__ void scales(int pr) {
#pragma unroll
        for (int h = 0; h < KH; h++) {
#pragma unroll
            for (int w = 0; w < (SETS + 3) / 4; w++) scale[h][w] = 0;
#pragma unroll
            for (int set = 0; set < SETS; set++) {
                const int n = set * PARTS + pr;
                const int byte = first[h] == 255 || n >= kQParts ? first[h] : first[h] - 4 * n;
                scale[h][set >> 2] |= (uint32_t)byte << (8 * (set & 3));
            }
        }
    }

    // Part n of half h (zeros past the last): with x = q / (2 s) in units of
    // 16^-n, what the nearest integer to it leaves, to the nearest sixteenth
    // (the conversion's rounding); for the first part x itself.  So any part is
    // made by itself, and lanes or wavefronts make one each: a conversion
    // takes some 125 clocks.
    __device__ __forceinline__ u32x6 digit(int h, int n) const {
        // x * mul is rounded as if alone: the rest is a power of two
        const float g = n < kQParts ? mul[h] * __uint_as_float((uint32_t)(253 - first[h] + 4 * n) << 23) : 0.f;
        const float whole = n == 0 ? 0.f : -1.f;
        f32x16 a, b;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float x = ev[h][i] * g, y = od[h][i] * g;
            a[i] = fmaf(whole, rintf(x), x);
            b[i] = fmaf(whole, rintf(y), y);
        }
        return __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(a, b, 0.5f);
    }
};

// The parts of a tile's columns in LDS.
template <int HD>
struct Kv4SharedQuery {
    static constexpr int KH = (HD + 127) / 128;
    uint2 w[KH][kQParts][3][4][16];
    __device__ __forceinline__ void put(const u32x6 &p, int h, int n, int r, int lg) {
#pragma unroll
        for (int i = 0; i < 3; i++) w[h][n][i][lg][r] = make_uint2(p[2 * i], p[2 * i + 1]);
    }
    __device__ __forceinline__ void get(Kv4Query<HD, 16> &q, int r, int lg) const {
#pragma unroll
        for (int h = 0; h < KH; h++)
#pragma unroll
            for (int n = 0; n < kQParts; n++)
#pragma unroll
                for (int i = 0; i < 3; i++) {
                    const uint2 x = w[h][n][i][lg][r];
                    q.part[h][n][2 * i] = x.x;
                    q.part[h][n][2 * i + 1] = x.y;
                }
    }
};

template <int HD>
struct Kv4Key {
    static constexpr int KH = (HD + 127) / 128;
    u32x4 code[KH];
    uint32_t scale[KH];

    // Codes and scales at the row `row` of their planes.  Lanes past the
    // head's dimensions repeat the first ones, against zeros of the query.
    __device__ __forceinline__ void load(const uint8_t *kc, const uint8_t *ks, unsigned row, int lg) {
#pragma unroll
        for (int h = 0; h < KH; h++) {
            const unsigned at = 128 * h + 32 * lg < HD ? 4 * h + lg : 0;
            if constexpr (HD == 16) {
                const uint2 c = *reinterpret_cast<const uint2 *>(kc + row * (HD / 2));
                code[h] = u32x4{c.x, c.y, 0, 0};
            } else {
                code[h] = *reinterpret_cast<const u32x4 *>(kc + (row * (HD / 2) + 16 * at));
            }
            scale[h] = ks[row * kv4_groups(HD) + at];
        }
    }
};

// Set S's products of TILES tiles of 16 keys with the columns.
template <int S, int HD, int C, int TILES>
__device__ __forceinline__ void score_set(const Kv4Key<HD> (&k)[TILES], const Kv4Query<HD, C> &q, int h, f32x4 (&s)[TILES]) {
    const u32x6 p = q.part[h][S];
    const i32x8 b = {(int)p[0], (int)p[1], (int)p[2], (int)p[3], (int)p[4], (int)p[5], 0, 0};
#pragma unroll
    for (int i = 0; i < TILES; i++) {
        const u32x4 c = k[i].code[h];
        const i32x8 a = {(int)c.x, (int)c.y, (int)c.z, (int)c.w, 0, 0, 0, 0};
        s[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, s[i], 4 /* fp4 */, 2 /* fp6 e2m3 */, 0,
                                                                (int)k[i].scale[h], S & 3, (int)q.scale[h][S >> 2]);
    }
}

template <int S, int HD, int C, int TILES>
__device__ __forceinline__ void score_sets(const Kv4Key<HD> (&k)[TILES], const Kv4Query<HD, C> &q, f32x4 (&s)[TILES]) {
    if constexpr (S < Kv4Lanes<C>::QSETS) {
#pragma unroll
        for (int h = 0; h < Kv4Key<HD>::KH; h++) score_set<S>(k, q, h, s);
        score_sets<S + 1>(k, q, s);
    }
}

// Scores in log2 units, less `ref`: the sums start from -ref and the largest
// part, so that what follows is added to numbers as small as the differences.
// pr: the lane's part.
template <int HD, int C, int TILES>
__device__ __forceinline__ void kv4_scores(const Kv4Key<HD> (&k)[TILES], const Kv4Query<HD, C> &q, float ref, int pr,
                                           f32x4 (&s)[TILES]) {
    const float from = pr == 0 ? -ref : 0.f;
#pragma unroll
    for (int i = 0; i < TILES; i++) s[i] = f32x4{from, from, from, from};
    score_sets<0>(k, q, s);
#pragma unroll
    for (int i = 0; i < TILES; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[i][e] = Kv4Lanes<C>::sum(s[i][e]);
}

// Whether a lane of the wavefront has a scale byte past the largest; those are
// replaced then, and *bits tells the lane's.
__device__ __forceinline__ bool take_marks(uint32_t (&scale)[8], uint32_t *bits) {
    uint32_t most = scale[0];
#pragma unroll
    for (int j = 1; j < 8; j++) most = max(most, scale[j]);
    *bits = 0;
    if (__builtin_amdgcn_ballot_w64(most > kKv4MaxScale) == 0) return false;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const bool marked = scale[j] > kKv4MaxScale;
        *bits |= marked ? 1u << j : 0u;
        scale[j] = marked ? 127u : scale[j];
    }
    return true;
}

// A lane's HD / 16 dimensions of its eight keys of a unit of 32.
template <int HD>
struct Kv4Values {
    static constexpr int DPL = HD / 16;                // dimensions, tiles
    static constexpr int W = HD == 256 ? 2 : 1;        // words of codes a key
    uint32_t code[8][W];
    uint32_t scale[8];

    // Rows 0 .. 31 of the planes; unless WHOLE, rows past d repeat row d.
    template <bool WHOLE>
    __device__ __forceinline__ void load(const uint8_t *vc, const uint8_t *vs, int d, int r, int lg) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const unsigned at = 16 * (j >> 2) + 4 * lg + (j & 3), row = WHOLE ? at : min(at, (unsigned)d);
            const uint8_t *p = vc + row * (HD / 2);
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
                code[j][0] = p[r >> 1];
            }
            scale[j] = vs[row * kv4_groups(HD) + r * DPL / 32];
        }
    }

    // Whether some group of this lane's keys is marked as not finite; its
    // values are then taken as finite ones (a masked key's weight of zero
    // must not meet a NaN), and nan_values puts the NaN where it belongs.  So
    // do the scales past the largest, which only rows never written can hold.
    __device__ __forceinline__ bool take_bad(uint32_t *bits) { return take_marks(scale, bits); }

    // The bf16 operands of two neighbouring tiles: dimensions 2 i and 2 i + 1
    // of the lane's, eight keys each.
    template <int I>
    __device__ __forceinline__ void widen(u32x4 &even, u32x4 &odd) const {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            w[j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(
                                                    code[j][I / 4], kv4_scale(scale[j]), I & 3));
        // a lane's one dimension of 16 is half of the byte it read
        const uint32_t pick = HD == 16 && (threadIdx.x & 1) ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            even[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], pick);
            odd[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x07060302u);
        }
    }
};

// Eight weights as bf16 parts, their upper, middle and lower eight significant
// bits: exact.  Set by set, the lane's part of each.
template <int C>
__device__ __forceinline__ void split_p(const float *p, int pr, bf16x8 (&out)[Kv4Lanes<C>::PSETS]) {
    static_assert(C == 16 || Kv4Lanes<C>::PSETS == 1, "the parts of a column in one set, or a set each");
    if constexpr (C == 16) {
        uint32_t x[kPParts][8];  // the parts are the upper halves
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float m = p[j] - __uint_as_float(__float_as_uint(p[j]) & 0xFFFF0000u);
            x[0][j] = __float_as_uint(p[j]);
            x[1][j] = __float_as_uint(m);
            x[2][j] = __float_as_uint(m - __uint_as_float(__float_as_uint(m) & 0xFFFF0000u));
        }
#pragma unroll
        for (int n = 0; n < kPParts; n++) {
            u32x4 a;
#pragma unroll
            for (int j = 0; j < 4; j++) a[j] = __builtin_amdgcn_perm(x[n][2 * j + 1], x[n][2 * j], 0x07060302u);
            out[n] = __builtin_bit_cast(bf16x8, a);
        }
    } else {
        // the lane's part by masks (selects become branches here); lanes past
        // the last part take zeros by the byte selector
        const uint32_t m1 = pr >= 1 ? 0xFFFF0000u : 0u, m2 = pr >= 2 ? 0xFFFF0000u : 0u;
        const uint32_t pick = pr < kPParts ? 0x07060302u : 0x0C0C0C0Cu;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j] = p[j] - __uint_as_float(__float_as_uint(p[j]) & m1);
            x[j] -= __uint_as_float(__float_as_uint(x[j]) & m2);
        }
        u32x4 a;
#pragma unroll
        for (int j = 0; j < 4; j++) a[j] = __builtin_amdgcn_perm(__float_as_uint(x[2 * j + 1]), __float_as_uint(x[2 * j]), pick);
        out[0] = __builtin_bit_cast(bf16x8, a);
    }
}

template <int SETS>
__device__ __forceinline__ f32x4 mfma_pv(const u32x4 &v, const bf16x8 (&p)[SETS], f32x4 o) {
#pragma unroll
    for (int n = SETS - 1; n >= 0; n--)
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
// of the lanes (4 lg + i, any) of marked(j), the lanes whose key j is marked.
template <int HD, class F>
__device__ __forceinline__ void nan_values(F marked, int key0, int qpos, int lg, f32x4 (&o)[HD / 16]) {
#pragma unroll 1
    for (int j = 0; j < 8; j++) {
        const unsigned long long lanes = marked(j);
#pragma unroll 1
        for (int kl = 0; kl < 4; kl++) {
            if (key0 + 16 * (j >> 2) + 4 * kl + (j & 3) > qpos) continue;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if ((lanes >> (16 * kl + 4 * lg + i)) & 1)
#pragma unroll
                    for (int t = 0; t < HD / 16; t++) o[t][i] = __builtin_nanf("");
        }
    }
}

// Running softmax state of a lane's column over the keys its wavefront took.
template <int HD>
struct Kv4State {
    float ref = 0.f;   // what the weights are relative to
    bool any = false;  // ref is a score's; before that, no score was above -inf
    float l = 0.f;
    f32x4 o[HD / 16];
    __device__ Kv4State() {
#pragma unroll
        for (int t = 0; t < HD / 16; t++) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // The reference of a merge: -inf where no score was above it.
    __device__ __forceinline__ float max_ref() const { return any ? ref : -INFINITY; }

    // The scores of some key tiles, less ref, become weights.  The reference
    // is raised in steps of at least 2^8 only: weights up to 2^8 cost no
    // precision in f32, and most blocks then leave the sums as they are.
    template <int TILES>
    __device__ __forceinline__ void weights(f32x4 (&s)[TILES], float (&p)[4 * TILES]) {
        float mx = s[0][0];
#pragma unroll
        for (int j = 1; j < 4 * TILES; j++) mx = fmaxf(mx, s[j >> 2][j & 3]);
        mx = max_xor16_32(mx);
        const bool raise = any ? mx > 8.0f : mx > -INFINITY;
        if (__builtin_amdgcn_ballot_w64(raise)) {
            const float up = raise ? mx : 0.0f, corr = raise ? (any ? __builtin_amdgcn_exp2f(-mx) : 0.0f) : 1.0f;
            ref += up;
            any |= raise;
            l *= corr;
#pragma unroll
            for (int t = 0; t < HD / 16; t++) o[t] *= corr;
#pragma unroll
            for (int j = 0; j < 4 * TILES; j++) s[j >> 2][j & 3] -= up;
        }
#pragma unroll
        for (int j = 0; j < 4 * TILES; j++) {
            p[j] = __builtin_amdgcn_exp2f(s[j >> 2][j & 3]);
            l += p[j];
        }
    }
};

// A new row of one head, quantized by a wavefront, in LDS in the cache's layout.
template <int HD>
struct Kv4NewRow {
    static constexpr int NG = kv4_groups(HD), LPR = HD / 8, W = Kv4Values<HD>::W;
    union {
        uint32_t code[2][LPR];
        u32x4 key16[2 * LPR / 4 ? 2 * LPR / 4 : 1];
    };
    uint8_t scale[2][8];

    // Lanes [0, LPR) take the key, the next LPR the value; x: the lane's
    // eight floats.  Also written to the cache's row.
    __device__ __forceinline__ void put(const float (&x)[8], int lane, const Kv4Planes<HD> &pl, size_t row) {
        const int i = lane / LPR, at = lane % LPR;
        uint32_t byte;
        const uint32_t c = kv4_quantize8<LPR / NG>(x, &byte);
        if (i < 2) {
            code[i][at] = c;
            *reinterpret_cast<uint32_t *>((i ? pl.vc : pl.kc) + row * (HD / 2) + at * 4) = c;
            if (at % (LPR / NG) == 0) {
                scale[i][at / (LPR / NG)] = (uint8_t)byte;
                (i ? pl.vs : pl.ks)[row * NG + at / (LPR / NG)] = (uint8_t)byte;
            }
        }
    }
    // The row in the place of row `at` of a unit that was loaded.
    __device__ __forceinline__ void patch(Kv4Key<HD> (&k)[2], Kv4Values<HD> &v, int at, int r, int lg) const {
        if (r == (at & 15)) {
#pragma unroll
            for (int h = 0; h < Kv4Key<HD>::KH; h++) {
                const int w = 128 * h + 32 * lg < HD ? 4 * h + lg : 0;
                const u32x4 c = HD == 16 ? u32x4{code[0][0], code[0][1], 0, 0} : key16[w];
                const uint32_t sc = scale[0][w];
                if (at < 16) {
                    k[0].code[h] = c;
                    k[0].scale[h] = sc;
                } else {
                    k[1].code[h] = c;
                    k[1].scale[h] = sc;
                }
            }
        }
        const uint8_t *p = reinterpret_cast<const uint8_t *>(code[1]);
        uint32_t c[W];
        if constexpr (HD == 256) {
            c[0] = code[1][2 * r];
            c[1] = code[1][2 * r + 1];
        } else if constexpr (HD == 128) {
            c[0] = code[1][r];
        } else if constexpr (HD == 64) {
            c[0] = reinterpret_cast<const uint16_t *>(p)[r];
        } else {
            c[0] = p[HD == 32 ? r : r >> 1];
        }
        const uint32_t sc = scale[1][r * Kv4Values<HD>::DPL / 32];
        const bool mine = lg == ((at >> 2) & 3);
        const int slot = (at >> 4) * 4 + (at & 3);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const bool here = mine && j == slot;
#pragma unroll
            for (int w = 0; w < W; w++) v.code[j][w] = here ? c[w] : v.code[j][w];
            v.scale[j] = here ? sc : v.scale[j];
        }
    }
};

// x / group for x below 2^21, by the reciprocal the host gives.
__device__ __forceinline__ int div_group(const Kv4AttnArgs &a, int x) { return (int)(((float)x + 0.5f) * a.inv_group); }

// An item is a tile of 16 columns of one sequence: the sequence's columns
// 16 tile .. + cols - 1, the first of them head h0 of query row t0.
struct Kv4Item {
    int seq, tile, cols, t0, h0;
    int pos;   // the sequence's first row position, or -1
    int last;  // the tile's last position
    int nb;    // blocks of keys up to it
};

// p: the sequence's position as given.
template <int BLOCK>
__device__ __forceinline__ Kv4Item kv4_item(const Kv4AttnArgs &a, int i, int p) {
    Kv4Item it;
    it.seq = a.ntile == 1 ? i : i / a.ntile;
    it.tile = i - it.seq * a.ntile;
    it.cols = min(16, a.rows * a.group - 16 * it.tile);
    it.t0 = a.ntile == 1 ? 0 : 16 * it.tile / a.group;
    it.h0 = 16 * it.tile - it.t0 * a.group;
    it.pos = kv4_pos(p, a.rows, a.c.cap);
    it.last = it.pos + it.t0 + div_group(a, it.h0 + it.cols - 1);
    it.nb = it.pos < 0 ? 0 : it.last / BLOCK + 1;
    return it;
}
template <int BLOCK>
__device__ __forceinline__ Kv4Item kv4_item(const Kv4AttnArgs &a, int i) {
    return kv4_item<BLOCK>(a, i, a.pos_dev ? a.pos_dev[a.ntile == 1 ? i : i / a.ntile] : a.pos);
}

__device__ __forceinline__ float uniform(float v) {
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
}

// Shares a.runs workgroups of a KV head out to the items: an item of n blocks
// gets ceil(n / each) of them, with the smallest `each` (to a 32nd of where it
// can be) for which there are enough, so every workgroup has one item and most
// have as many blocks.  Every wavefront finds its workgroup's share by itself;
// all of them come to the same numbers.  False where workgroup `run` has none.
// blocks: kKv4DealItems floats in LDS, to which all wavefronts write the same.
template <int BLOCK>
__device__ __forceinline__ bool kv4_deal(const Kv4AttnArgs &a, int run, int lane, float *blocks, int *item, int *part, int *parts) {
    float total = 0.f, most = 1.f;  // (integers below 2^24)
#pragma unroll 1
    for (int i = lane; i < a.items; i += 64) {
        const float n = (float)max(1, kv4_item<BLOCK>(a, i).nb);
        blocks[i] = n;
        total += n;
        most = fmaxf(most, n);
    }
    // a lane reads what it wrote itself
    const float n0 = lane < a.items ? blocks[lane] : 0.f;
    total = uniform(wave_sum(total));
    most = uniform(wave_max(most));
    float inv = 0.f;  // 1 / each
    auto share = [&](float n) { return n > 0.f ? min((int)((n - 0.5f) * inv) + 1, kKv4MaxRuns) : 0; };
    int lo = max((int)ceilf(total / (float)a.runs), max((int)most / kKv4MaxRuns, kKv4WholeKeys / BLOCK)), hi = max(lo, (int)most);
    // one an item, and one more for every `each` blocks past the first
    if (a.runs > a.items) hi = min(hi, max(lo, (int)((total - (float)a.items) / (float)(a.runs - a.items)) + 1));
#pragma unroll 1
    for (int turn = 0; turn < 5 && lo < hi; turn++) {
        const int mid = (lo + hi) >> 1;
        inv = __builtin_amdgcn_rcpf((float)mid);
        int sum = share(n0);
#pragma unroll 1
        for (int i = lane + 64; i < a.items; i += 64) sum += share(blocks[i]);
        if ((int)uniform(wave_sum((float)sum)) <= a.runs) hi = mid;
        else lo = mid + 1;
    }
    inv = __builtin_amdgcn_rcpf((float)hi);
    int before = 0;
#pragma unroll 1
    for (int i = 0; i < a.items; i += 64) {
        const int mine = share(i == 0 ? n0 : i + lane < a.items ? blocks[i + lane] : 0.f);
        int upto = mine;  // over the lanes up to this one
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(upto, off, 64);
            upto += lane >= off ? o : 0;
        }
        const int first = before + upto - mine;
        const unsigned long long here = __builtin_amdgcn_ballot_w64(run >= first && run < first + mine);
        if (here) {
            const int l = __builtin_ctzll(here);
            *item = i + l;
            *part = run - __builtin_amdgcn_readlane(first, l);
            *parts = __builtin_amdgcn_readlane(mine, l);
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// Output elements d, d + 1 of the item's column c.
template <int HD>
__device__ __forceinline__ void kv4_put(const Kv4AttnArgs &a, const Kv4Item &it, int g, int c, int d, float2 O, float L) {
    const int dt = div_group(a, it.h0 + c), h = it.h0 + c - dt * a.group;
    const size_t i = ((size_t)it.seq * a.rows + it.t0 + dt) * a.out_stride + (size_t)(g * a.group + h) * HD + d;
    const float f = L == 0.f ? 0.f : __builtin_amdgcn_rcpf(L);  // (within an ulp)
    const float x = O.x * f, y = O.y * f;
    if (a.out) *reinterpret_cast<float2 *>(a.out + i) = make_float2(x, y);
    if (a.out_hi) {
        split_bf16(x, a.out_hi + i, a.out_lo + i);
        split_bf16(y, a.out_hi + i + 1, a.out_lo + i + 1);
    }
}

// Wavefronts of a workgroup; a wavefront takes 32 keys of a block.  One item
// alone is spread over eight (fewer workgroups to merge: at 8300 positions 11.2
// us against 12.4 with four, at 200 5.7 against 5.3); of several, two workgroups
// of four share a CU, so that one's loads, query and merge run beside the
// other's products (64 sequences of 2001 positions 26.7 us against 29.0 with
// one of eight, 500 tokens 11.1 against 15.4; 32 of 2001 20.5 against 16.2).
// At head dim 256 the registers leave room for one wavefront a SIMD.
template <int HD, bool ONE>
constexpr int kv4_waves() {
    return ONE && HD < 256 ? 8 : 4;
}

// A workgroup owns one KV head and blocks of an item (32 keys a wavefront), each
// wavefront with a softmax state of its own; the wavefronts are merged through
// LDS.  Where several workgroups share an item they take its blocks in turn,
// and the last of them to arrive merges their states, in the order of the
// parts, so that the result does not depend on who is last: one launch in all.
//
// - ONE item: a workgroup's first block does not hang on the position, so its
//   keys are loaded before the position, which may live on the device, is
//   known.
// - Up to kKv4DealItems items (a.deal): kv4_deal shares the workgroups out.
//   (The same number of them for every item left sequences of 65 to 131070
//   positions at 100 us, 1.9 times the time of their mean.)
// - More items: a workgroup each.
//
// With a.k_new (one row a sequence) the wavefront that owns the new position
// quantizes the row, stores it and takes it from LDS; no other needs it.
//
// Bound by the latency of its loads and of the merge for one sequence (16 heads
// over 8 of 128: 6.0 us at 320 positions, 11 at 8300) or a few (14 of up to 1003
// positions 11 us); by VALU issue (78%: a value takes a conversion and half a
// permute) and the cache's bytes for many: four sequences, 271 thousand
// positions, 56.6 us, 5.2 TB/s.
template <int HD, bool ONE, int C>
__global__ __launch_bounds__((64 * kv4_waves<HD, ONE>()), (HD == 256 ? 1 : 2)) void kv4_attn_rows_kernel(const Kv4AttnArgs a) {
    constexpr int DPL = HD / 16, PITCH = HD + 4, NW = kv4_waves<HD, ONE>(), NT = 64 * NW, BLOCK = 32 * NW;
    // the wavefronts' sums [NW][16][PITCH], then the runs' weights [16][kKv4MaxRuns]
    constexpr int SUMS = NW * 16 * PITCH, WEIGHTS = 16 * kKv4MaxRuns;
    __shared__ __attribute__((aligned(16))) float s_o[SUMS > WEIGHTS ? SUMS : WEIGHTS];
    __shared__ float s_m[16][NW], s_l[16][NW];
    __shared__ Kv4SharedQuery<C == 16 ? HD : 16> s_q;
    __shared__ Kv4NewRow<HD> s_new;
    __shared__ unsigned s_arrived;
    __shared__ float s_blocks[ONE ? 1 : kKv4DealItems];
    __shared__ float2 s_red[NT];
    const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, r = lane & 15, lg = lane >> 4;
    // (run, KV head): one item's runs read different keys; several items' tiles
    // share a head's, whose workgroups are nkv apart, so on one XCD for eight
    const int g = ONE ? (int)blockIdx.y : (int)(blockIdx.x % (unsigned)a.c.nkv);
    const int run = ONE ? (int)blockIdx.x : (int)(blockIdx.x / (unsigned)a.c.nkv);
    const size_t row0 = (size_t)g * a.c.cap;
    const bool append = a.k_new != nullptr;

    Kv4Key<HD> k[2];
    Kv4Values<HD> v;
    Kv4Query<HD, C> q;
    float xn[8];
    // the lane's column and part
    constexpr int PARTS = Kv4Lanes<C>::PARTS;
    const int rc = r / PARTS, pr = r % PARTS;
    // keys key0 .. +31 of the head; those past lim repeat it
    auto load = [&](const Kv4Planes<HD> &pl, int key0, int lim) {
        const int at = min(key0, lim), d = lim - at;
        const size_t row = row0 + at;
        const uint8_t *const kc = pl.kc + row * (HD / 2), *const ks = pl.ks + row * kv4_groups(HD);
        const uint8_t *const vc = pl.vc + row * (HD / 2), *const vs = pl.vs + row * kv4_groups(HD);
        if (d >= 31) {  // constant offsets: a third of the unit's address arithmetic
            k[0].load(kc, ks, (unsigned)r, lg);
            k[1].load(kc, ks, (unsigned)(16 + r), lg);
            v.template load<true>(vc, vs, d, r, lg);
        } else {
            k[0].load(kc, ks, (unsigned)min(r, d), lg);
            k[1].load(kc, ks, (unsigned)min(16 + r, d), lg);
            v.template load<false>(vc, vs, d, r, lg);
        }
    };
    auto fetch = [&](int seq, int t0, int h0, int cols) {
        const int c = h0 + min(rc, cols - 1), dt = div_group(a, c), h = c - dt * a.group;
        q.fetch(a.q + ((size_t)seq * a.rows + t0 + dt) * a.q_stride + (size_t)(g * a.group + h) * HD, lg);
        if (append) {
            const int l = lane % (HD / 4);
            const float *src = (l < HD / 8 ? a.k_new : a.v_new) + (size_t)seq * a.new_stride + (size_t)g * HD + l % (HD / 8) * 8;
            *reinterpret_cast<f32x4 *>(xn) = *reinterpret_cast<const f32x4 *>(src);
            *reinterpret_cast<f32x4 *>(xn + 4) = *reinterpret_cast<const f32x4 *>(src + 4);
        }
    };

    // the query's parts, from what was fetched
    auto split = [&](int cols) {
        q.ready(a.scale * 1.4426950408889634f, lg);
        q.scales(pr);
#pragma unroll
        for (int h = 0; h < Kv4Query<HD, C>::KH; h++) {
            if constexpr (C < 16) {  // a lane makes its own
#pragma unroll
                for (int set = 0; set < Kv4Lanes<C>::QSETS; set++) q.part[h][set] = q.digit(h, set * PARTS + pr);
            } else {  // the wavefronts make them together
                for (int n = wave; n < kQParts; n += NW) {
                    const u32x6 d = q.digit(h, n);
                    if (r < cols) s_q.put(d, h, n, r, lg);
                }
            }
        }
        if constexpr (C == 16) {
            lds_barrier();  // the keys may still be on their way
            s_q.get(q, min(r, cols - 1), lg);
        }
    };

    int pos0 = a.pos;
    int item = 0, part = 0, parts = 1;  // this workgroup's, and those that share the item
    const bool deal = !ONE && a.deal;
    if constexpr (ONE) {
        // the query first: it is split while the first keys are on their way
        fetch(0, 0, 0, min(16, a.rows * a.group));
        load(Kv4Planes<HD>(a.c, 0), run * BLOCK + 32 * wave, (int)a.c.cap - 1);
        asm volatile("" ::: "memory");  // not behind the position's read
        if (a.pos_dev) pos0 = *a.pos_dev;
        split(min(16, a.rows * a.group));
        if constexpr (C < 16)  // made here, while the position is on its way
#pragma unroll
            for (int h = 0; h < Kv4Query<HD, C>::KH; h++)
#pragma unroll
                for (int set = 0; set < Kv4Lanes<C>::QSETS; set++) asm volatile("" : "+v"(q.part[h][set]));
    } else if (deal) {
        if (!kv4_deal<BLOCK>(a, run, lane, s_blocks, &item, &part, &parts)) return;
    } else {
        item = a.items - 1 - run;  // the latest rows, with the most keys, first
    }
    const Kv4Item it = ONE ? kv4_item<BLOCK>(a, 0, pos0) : kv4_item<BLOCK>(a, item);
    const Kv4Planes<HD> pl(a.c, it.seq);
    if constexpr (ONE) {
        if (it.nb > kKv4WholeKeys / BLOCK) {
            const unsigned each = ((unsigned)it.nb + a.runs - 1) / (unsigned)a.runs;
            parts = (int)(((unsigned)it.nb + each - 1) / each);
        }
        if (run >= parts) return;
        part = run;
    }
    const int cols = it.cols, pos = it.pos;
    Kv4State<HD> st;
    if (pos >= 0) {
        // (lanes past the columns repeat the last one)
        const int qpos = pos + it.t0 + div_group(a, it.h0 + min(rc, cols - 1));
        const int first_pos = pos + it.t0;
        const int step = parts * BLOCK;
        int key0 = part * BLOCK + 32 * wave;
        if constexpr (!ONE) {
            fetch(it.seq, it.t0, it.h0, cols);
            load(pl, key0, it.last);
            split(cols);
        }
        for (; key0 <= it.last; key0 += step) {
            if (append && key0 + 31 >= pos) {
                s_new.put(xn, lane, pl, row0 + pos);
                // the wavefront's own LDS writes, in order
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                s_new.patch(k, v, pos - key0, r, lg);
            }
            f32x4 s[2];
            kv4_scores(k, q, st.ref, pr, s);
            Kv4Values<HD> vn = v;
            if (key0 + step <= it.last) load(pl, key0 + step, it.last);
            if (key0 + 31 > first_pos) {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (key0 + 16 * (j >> 2) + 4 * lg + (j & 3) > qpos) s[j >> 2][j & 3] = -INFINITY;
            }
            float p[8];
            st.weights(s, p);
            bf16x8 pp[Kv4Lanes<C>::PSETS];
            split_p<C>(p, pr, pp);
            uint32_t bad;
            const bool any_bad = vn.take_bad(&bad);
            kv4_values(vn, pp, st.o);
            if (any_bad)
                nan_values<HD>([&](int j) { return __builtin_amdgcn_ballot_w64((bad >> j) & 1); }, key0, qpos, lg, st.o);
        }
    }
    // the wavefronts' states
    st.l = add_xor32(add_xor16(st.l));
    constexpr int OPARTS = C < 16 ? kPParts : 1;  // lanes with parts of a column's sums
    if (rc < cols && pr < OPARTS) {
        float *const dst = s_o + (wave * 16 + r) * PITCH + 4 * lg * DPL;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int d = 0; d < DPL; d++) dst[i * DPL + d] = st.o[d][i];
        if (lg == 0 && pr == 0) {
            s_m[rc][wave] = st.max_ref();
            s_l[rc][wave] = st.l;
        }
    }
    lds_barrier();  // (an appended row's stores may still be on their way)
    const size_t slot0 = (size_t)g * a.runs + run - part, slot = slot0 + part;  // of partial states
    for (int idx = t; idx < cols * (HD / 2); idx += NT) {
        const int c = idx / (HD / 2), d = idx % (HD / 2) * 2;
        float M = s_m[c][0];
#pragma unroll
        for (int w = 1; w < NW; w++) M = fmaxf(M, s_m[c][w]);
        float L = 0.f;
        float2 O = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            // a wavefront without a finite maximum still brings its sums:
            // they are zeros, or NaN
            const float f = s_m[c][w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[c][w] - M);
            L = fmaf(s_l[c][w], f, L);
            float2 sum = *reinterpret_cast<const float2 *>(s_o + (w * 16 + c * PARTS) * PITCH + d);
#pragma unroll
            for (int e = 1; e < OPARTS; e++) {
                const float2 x = *reinterpret_cast<const float2 *>(s_o + (w * 16 + c * PARTS + e) * PITCH + d);
                sum = make_float2(sum.x + x.x, sum.y + x.y);
            }
            O = make_float2(fmaf(sum.x, f, O.x), fmaf(sum.y, f, O.y));
        }
        if (parts == 1) {
            kv4_put<HD>(a, it, g, c, d, O, L);
        } else {
            st_dev2(a.part + (slot * a.part_cols + c) * HD + d, O.x, O.y);
            if (d == 0) st_dev2(a.part_ml + (slot * a.part_cols + c) * 2, M, L);
        }
    }
    if (parts > 1) {
        // a workgroup's partial state is complete before it counts itself in
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        unsigned *const count = a.arrived + slot0;
        if (t == 0) s_arrived = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (s_arrived == (unsigned)parts - 1) {
            if (t == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            auto at = [&](int i) { return (slot0 + i) * a.part_cols; };
            // SUB threads a pair of elements, each with the parts sub, sub +
            // SUB, ..; its first parts are on their way while the columns'
            // weights and sums are made
            constexpr int FAR = kKv4MaxRuns / 64, AHEAD = C == 16 ? 8 : 16;
            const int pairs = cols * (HD / 2), SUB = max(1, NT / pairs);
            const int e0 = SUB == 1 ? t : t % pairs, sub = SUB == 1 ? 0 : t / pairs;
            float2 ahead[AHEAD];
            auto grab = [&](int e, int i) {
                const float *src = a.part + (size_t)(e / (HD / 2)) * HD + e % (HD / 2) * 2;
#pragma unroll
                for (int u = 0; u < AHEAD; u++)
                    if (i + u * SUB < parts) ahead[u] = ld_dev2(src + at(i + u * SUB) * HD);
            };
            const bool busy = sub < SUB && e0 < pairs;
            if (busy) grab(e0, sub);
            for (int c = wave; c < cols; c += NW) {
                float M = -INFINITY, L = 0.f, m[FAR], l[FAR];
#pragma unroll
                for (int i = 0; i < FAR; i++) {
                    m[i] = -INFINITY;
                    l[i] = 0.f;
                    if (64 * i >= parts) continue;
                    const float2 ml = ld_dev2(a.part_ml + (at(min(lane + 64 * i, parts - 1)) + c) * 2);
                    m[i] = ml.x;
                    l[i] = ml.y;
                }
#pragma unroll
                for (int i = 0; i < FAR; i++) M = fmaxf(M, m[i]);
                M = wave_max(M);
#pragma unroll
                for (int i = 0; i < FAR; i++) {
                    if (64 * i >= parts) continue;
                    const bool there = lane + 64 * i < parts;
                    const float f = m[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[i] - M);
                    L = there ? fmaf(l[i], f, L) : L;
                    if (there) s_o[c * kKv4MaxRuns + lane + 64 * i] = f;
                }
                L = wave_sum(L);
                if (lane == 0) s_l[c][0] = L;
            }
            __syncthreads();
            bool fresh = true;
            for (int e = e0; busy && e < pairs; e += NT) {
                const int c = e / (HD / 2);
                float2 O = make_float2(0.f, 0.f);
                for (int i = sub; i < parts; i += AHEAD * SUB) {
                    if (!fresh) grab(e, i);
                    fresh = false;
#pragma unroll
                    for (int u = 0; u < AHEAD; u++)
                        if (i + u * SUB < parts) {
                            const float f = s_o[c * kKv4MaxRuns + i + u * SUB];
                            O = make_float2(fmaf(ahead[u].x, f, O.x), fmaf(ahead[u].y, f, O.y));
                        }
                }
                if (SUB == 1)
                    kv4_put<HD>(a, it, g, c, e % (HD / 2) * 2, O, s_l[c][0]);
                else
                    s_red[sub * pairs + e] = O;
            }
            if (SUB > 1) {
                __syncthreads();
                if (t < pairs) {
                    float2 O = s_red[t];
                    for (int i = 1; i < SUB; i++) O = make_float2(O.x + s_red[i * pairs + t].x, O.y + s_red[i * pairs + t].y);
                    kv4_put<HD>(a, it, g, t / (HD / 2), t % (HD / 2) * 2, O, s_l[t / (HD / 2)][0]);
                }
            }
        }
    }
}

// ---- many columns -----------------------------------------------------------

// Column tiles of 16 of a wavefront; a workgroup is four wavefronts.  With one,
// three wavefronts fit a SIMD: 8192 tokens 548 us, against 703 with two tiles
// and two wavefronts.
constexpr int kColTiles = 1;
constexpr int kTileKeys = 64;  // keys of a block

// A wavefront's share of widening a block's values: a unit of 32 keys, and
// half of a lane's dimensions (all of them where a lane has one or two; then
// only the even wavefronts have a share).
template <int HD>
struct Kv4Stage {
    static constexpr int DPL = HD / 16, TILES = DPL < 4 ? DPL : DPL / 2;
    uint32_t code[8], scale[8];

    template <bool WHOLE>
    __device__ __forceinline__ void load(const uint8_t *vc, const uint8_t *vs, int d, int half, int r, int lg) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const unsigned at = 16 * (j >> 2) + 4 * lg + (j & 3), row = WHOLE ? at : min(at, (unsigned)d);
            const uint8_t *p = vc + row * (HD / 2);
            if constexpr (HD == 256)
                code[j] = *reinterpret_cast<const uint32_t *>(p + 8 * r + 4 * half);
            else if constexpr (HD == 128)
                code[j] = *reinterpret_cast<const uint16_t *>(p + 4 * r + 2 * half);
            else if constexpr (HD == 64)
                code[j] = p[2 * r + half];
            else
                code[j] = p[HD == 32 ? r : r >> 1];
            scale[j] = vs[row * kv4_groups(HD) + r * DPL / 32];
        }
    }

    // The tiles' bf16 operands to dst[tile][64 lanes]; the marked lanes of
    // each key to mark, and whether there are any to *any (by half 0).
    __device__ __forceinline__ void store(u32x4 (*dst)[64], unsigned long long *mark, int *any, int half, int lane) {
        uint32_t bad;
        const bool some = take_marks(scale, &bad);
        if (half == 0) {
            if (some) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const unsigned long long lanes = __builtin_amdgcn_ballot_w64((bad >> j) & 1);
                    if (lane == 0) mark[j] = lanes;
                }
            }
            if (lane == 0) *any = some;
        }
        put<0>(dst + (DPL < 4 ? 0 : half * TILES), lane);
    }

  private:
    template <int I>
    __device__ __forceinline__ void put(u32x4 (*dst)[64], int lane) const {
        if constexpr (2 * I < TILES) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
                w[j] = __builtin_bit_cast(
                    uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code[j], kv4_scale(scale[j]), I));
            const uint32_t pick = HD == 16 && (lane & 1) ? 0x07060302u : 0x05040100u;
            u32x4 even, odd;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                even[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], pick);
                odd[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x07060302u);
            }
            dst[2 * I][lane] = even;
            if constexpr (2 * I + 1 < TILES) dst[2 * I + 1][lane] = odd;
            put<I + 1>(dst, lane);
        }
    }
};

// Long prompts: a workgroup owns a tile of 64 kColTiles columns, 16 kColTiles
// a wavefront, and goes through their blocks of 64 keys.  The
// wavefronts read the block's keys straight into matrix operands; the values
// are widened once for all of them, a share each, into LDS in operand order (a
// lane's operand is 16 bytes at 16 lane: no bank conflicts), a block ahead.
//
// Workgroups of the latest positions come first: they have the most keys.
// Bound by the issue of its three wavefronts a SIMD (MFMA busy 49%, VALU 66%):
// 8192 tokens, 16 heads over 8 of 128, 546-567 us, 485-503 TFLOP/s of the
// causal products' 275 GFLOP.  With the parts of Q and P that is 618 GFLOP in
// bf16 products' time: 1.09-1.13 PFLOP/s, where a plain bf16 product of 8192^3
// reaches 1.19.  (Wave priorities around the products or the softmax: 567-571.)
template <int HD>
__global__ __launch_bounds__(kBlock, HD == 256 ? 2 : 3) void kv4_attn_tile_kernel(const Kv4AttnArgs a) {
    constexpr int DPL = HD / 16, CT = kColTiles, TC = 64 * CT;
    // the wavefronts' query parts at first, then the values of two blocks
    constexpr size_t PARTS = 4 * sizeof(Kv4SharedQuery<HD>), VALUES = 4 * DPL * 64 * sizeof(u32x4);
    __shared__ __attribute__((aligned(16))) char s_buf[PARTS > VALUES ? PARTS : VALUES];
    Kv4SharedQuery<HD> *const s_q = reinterpret_cast<Kv4SharedQuery<HD> *>(s_buf);
    u32x4 (*const s_v)[2][DPL][64] = reinterpret_cast<u32x4 (*)[2][DPL][64]>(s_buf);
    __shared__ unsigned long long s_mark[2][2][8];
    __shared__ int s_any[2][2];
    const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, r = lane & 15, lg = lane >> 4;
    const int g = (int)(blockIdx.x % (unsigned)a.c.nkv);
    const unsigned rest = blockIdx.x / (unsigned)a.c.nkv;
    const int seq = (int)(rest % (unsigned)a.c.n_seq), tile = a.ntile - 1 - (int)(rest / (unsigned)a.c.n_seq);
    const int ncol = a.rows * a.group, cols = min(TC, ncol - TC * tile);
    const int pos = kv4_pos(a.pos_dev, a.pos, seq, a.rows, a.c.cap);
    const int t0 = TC * tile / a.group, h0 = TC * tile - t0 * a.group;
    const int last = pos + t0 + div_group(a, h0 + cols - 1);
    const int nb = pos < 0 ? 0 : last / kTileKeys + 1;
    const Kv4Planes<HD> pl(a.c, seq);
    const size_t row0 = (size_t)g * a.c.cap;

    int col[CT], qpos[CT];  // in the tile; lanes past the columns repeat the last one
    Kv4Query<HD, 16> q[CT];
    Kv4State<HD> st[CT];
    const bool mine = 16 * CT * wave < cols;
#pragma unroll
    for (int c = 0; c < CT; c++) {
        col[c] = 16 * (CT * wave + c) + r;
        const int dt = div_group(a, h0 + min(col[c], cols - 1)), h = h0 + min(col[c], cols - 1) - dt * a.group;
        qpos[c] = pos + t0 + dt;
        q[c].fetch(a.q + ((size_t)seq * a.rows + t0 + dt) * a.q_stride + (size_t)(g * a.group + h) * HD, lg);
    }
    const int wave_first = pos + t0 + div_group(a, h0 + min(16 * CT * wave, cols - 1));
    const int wave_last = pos + t0 + div_group(a, h0 + min(16 * CT * (wave + 1), cols) - 1);
    const int unit = wave >> 1, half = wave & 1;
    const bool stages = DPL >= 4 || half == 0;

    Kv4Key<HD> k[4];
    Kv4Stage<HD> v;
    auto load_keys = [&](int key0) {
        const int at = min(key0, last), d = last - at;
        const size_t row = row0 + at;
        const uint8_t *const kc = pl.kc + row * (HD / 2), *const ks = pl.ks + row * kv4_groups(HD);
        if (d >= kTileKeys - 1) {
#pragma unroll
            for (int i = 0; i < 4; i++) k[i].load(kc, ks, (unsigned)(16 * i + r), lg);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) k[i].load(kc, ks, (unsigned)min(16 * i + r, d), lg);
        }
    };
    auto load_values = [&](int key0) {
        const int at = min(key0 + 32 * unit, last);
        const size_t row = row0 + at;
        const uint8_t *const vc = pl.vc + row * (HD / 2), *const vs = pl.vs + row * kv4_groups(HD);
        if (last - at >= 31)
            v.template load<true>(vc, vs, 31, half, r, lg);
        else
            v.template load<false>(vc, vs, last - at, half, r, lg);
    };
    if (nb) {
        load_keys(0);
        if (stages) load_values(0);
    }
#pragma unroll
    for (int c = 0; c < CT; c++) {
        q[c].ready(a.scale * 1.4426950408889634f, lg);
        q[c].scales(0);
        // through LDS, so that the parts are made in a loop: unrolled they
        // are most of the kernel's code
#pragma unroll
        for (int h = 0; h < Kv4Query<HD, 16>::KH; h++)
#pragma unroll 1
            for (int n = 0; n < kQParts; n++) s_q[wave].put(q[c].digit(h, n), h, n, r, lg);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        s_q[wave].get(q[c], r, lg);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    lds_barrier();  // the values take the parts' place
    if (nb && stages) {
        v.store(s_v[0][unit], s_mark[0][unit], &s_any[0][unit], half, lane);
        load_values(kTileKeys);
    }
    lds_barrier();
    for (int b = 0; b < nb; b++) {
        const int key0 = b * kTileKeys, buf = b & 1;
        const bool work = mine && key0 <= wave_last;
        bf16x8 p[CT][2][3];
        if (work) {
            f32x4 s[CT][4];
#pragma unroll
            for (int c = 0; c < CT; c++) kv4_scores(k, q[c], st[c].ref, 0, s[c]);
            load_keys(key0 + kTileKeys);
#pragma unroll
            for (int c = 0; c < CT; c++) {
                if (key0 + kTileKeys - 1 > wave_first) {
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        if (key0 + 16 * (j >> 2) + 4 * lg + (j & 3) > qpos[c]) s[c][j >> 2][j & 3] = -INFINITY;
                }
                float w[16];
                st[c].weights(s[c], w);
                split_p<16>(w, 0, p[c][0]);
                split_p<16>(w + 8, 0, p[c][1]);
            }
        }
        // the next block's values, while this one's are multiplied
        if (b + 1 < nb && stages) {
            v.store(s_v[buf ^ 1][unit], s_mark[buf ^ 1][unit], &s_any[buf ^ 1][unit], half, lane);
            load_values(key0 + 2 * kTileKeys);
        }
        if (work) {
#pragma unroll
            for (int d = 0; d < DPL; d++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const u32x4 x = s_v[buf][u][d][lane];
#pragma unroll
                    for (int c = 0; c < CT; c++) st[c].o[d] = mfma_pv(x, p[c][u], st[c].o[d]);
                }
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (s_any[buf][u])
#pragma unroll
                    for (int c = 0; c < CT; c++)
                        nan_values<HD>([&](int j) { return s_mark[buf][u][j]; }, key0 + 32 * u, qpos[c], lg, st[c].o);
        }
        lds_barrier();
    }
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const float l = add_xor32(add_xor16(st[c].l)), f = l == 0.f ? 0.f : 1.0f / l;
        if (col[c] >= cols) continue;
        const int dt = div_group(a, h0 + col[c]), h = h0 + col[c] - dt * a.group;
        const size_t to = ((size_t)seq * a.rows + t0 + dt) * a.out_stride + (size_t)(g * a.group + h) * HD;
        constexpr int VEC = DPL < 4 ? DPL : 4;
        typedef float vec __attribute__((ext_vector_type(VEC)));
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int d = 0; d < DPL; d += VEC) {
                const size_t at = to + (4 * lg + i) * DPL + d;
                vec y;
#pragma unroll
                for (int e = 0; e < VEC; e++) y[e] = st[c].o[d + e][i] * f;
                if (a.out) *reinterpret_cast<vec *>(a.out + at) = y;
                if (a.out_hi)
#pragma unroll
                    for (int e = 0; e < VEC; e++) split_bf16(y[e], a.out_hi + at + e, a.out_lo + at + e);
            }
    }
}

}  // namespace

Kv4Plan plan_kv4_attn(const Kv4Cache &c, int rows, int nq) {
    Kv4Plan p{};
    const int64_t ncol = (int64_t)rows * (nq / c.nkv);
    const int tc = 64 * kColTiles;
    p.ntile = (int)((ncol + tc - 1) / tc);
    p.items = (int64_t)p.ntile * c.n_seq;
    p.runs = 1;  // (of the tile kernel)
    p.tile = ncol > kKv4RowCols && p.items * c.nkv >= kKv4TileWorkgroups;
    if (p.tile) return p;
    p.part_cols = (int)std::min<int64_t>(16, ncol);
    p.ntile = (int)((ncol + 15) / 16);
    p.items = (int64_t)p.ntile * c.n_seq;
    const bool one = p.items == 1;
    const int block = one && c.hd < 256 ? 32 * kv4_waves<128, true>() : 32 * kv4_waves<128, false>();
    const int64_t nb = ((int64_t)c.cap + block - 1) / block;
    const int groups = one && c.hd < 256 ? kKv4Workgroups / 2 : kKv4Workgroups;
    const int64_t most = std::min<int64_t>(p.items * nb, std::max(1, groups / c.nkv));
    // (kv4_deal counts up to 2^21 blocks)
    const bool share = c.cap > kKv4WholeKeys && most > 1;
    p.deal = share && !one && p.items * c.nkv <= kKv4Workgroups && nb <= 1 << 20;
    p.split = share && (one || p.deal);
    p.runs = (int)(!p.split ? p.items : one ? std::min<int64_t>(most, kKv4MaxRuns) : most);
    return p;
}

// Partial states of a launch.
static size_t kv4_part_states(const Kv4Plan &p, int nkv) { return p.split ? (size_t)nkv * p.runs * p.part_cols : 0; }

size_t kv4_attn_ws_bytes(const Kv4Cache &c, int rows, int nq) {
    const size_t n = kv4_part_states(plan_kv4_attn(c, rows, nq), c.nkv);
    return n ? kKv4CounterBytes + n * (c.hd + 2) * 4 : 0;
}

namespace {

// Columns of an item in as few lanes as hold them: two or four with their
// parts beside them, or 16.
template <int HD, bool ONE>
void launch_rows(const Kv4AttnArgs &a, unsigned grid, hipStream_t s) {
    const dim3 block(64 * kv4_waves<HD, ONE>()), wgs = ONE ? dim3(a.runs, a.c.nkv) : dim3(grid);
    if (a.part_cols <= 2)
        hipLaunchKernelGGL((kv4_attn_rows_kernel<HD, ONE, 2>), wgs, block, 0, s, a);
    else if (a.part_cols <= 4)
        hipLaunchKernelGGL((kv4_attn_rows_kernel<HD, ONE, 4>), wgs, block, 0, s, a);
    else
        hipLaunchKernelGGL((kv4_attn_rows_kernel<HD, ONE, 16>), wgs, block, 0, s, a);
}

template <int HD>
void launch_attn_hd(const Kv4AttnArgs &a, bool tile, unsigned grid, hipStream_t s) {
    if (tile)
        hipLaunchKernelGGL((kv4_attn_tile_kernel<HD>), dim3(grid), dim3(kBlock), 0, s, a);
    else if (a.items == 1)
        launch_rows<HD, true>(a, grid, s);
    else
        launch_rows<HD, false>(a, grid, s);
}

}  // namespace

hipError_t launch_kv4_attn(Kv4AttnArgs a, void *ws, hipStream_t s) {
    const Kv4Plan p = plan_kv4_attn(a.c, a.rows, a.nq);
    const int64_t grid = (p.tile ? p.items : 1) * p.runs * a.c.nkv;
    if (grid > 0x7fffffff || (p.split && !ws)) return hipErrorInvalidValue;
    if (a.k_new && a.rows > 1) {
        const Kv4WriteArgs w{a.c, a.k_new, a.v_new, a.new_stride, a.rows, a.pos_dev, a.pos};
        const hipError_t e = launch_kv4_write(w, s);
        if (e != hipSuccess) return e;
        a.k_new = a.v_new = nullptr;
    }
    a.group = a.nq / a.c.nkv;
    a.inv_group = 1.0f / (float)a.group;
    a.ntile = p.ntile;
    a.items = (int)p.items;
    a.deal = p.deal;
    a.runs = p.runs;
    a.part_cols = p.part_cols;
    a.arrived = (unsigned *)ws;
    a.part = (float *)((char *)ws + kKv4CounterBytes);
    a.part_ml = a.part + kv4_part_states(p, a.c.nkv) * a.c.hd;
    switch (a.c.hd) {
        case 16: launch_attn_hd<16>(a, p.tile, (unsigned)grid, s); break;
        case 32: launch_attn_hd<32>(a, p.tile, (unsigned)grid, s); break;
        case 64: launch_attn_hd<64>(a, p.tile, (unsigned)grid, s); break;
        case 128: launch_attn_hd<128>(a, p.tile, (unsigned)grid, s); break;
        case 256: launch_attn_hd<256>(a, p.tile, (unsigned)grid, s); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace tmg
