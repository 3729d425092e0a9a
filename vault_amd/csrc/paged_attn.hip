// Attention over the paged 8-bit K/V cache (include/vault_amd.h: vgx_paged_attn).
//
// For a sequence's queries r = (token t, head of the kv group) against keys j of its pages,
//   s_rj = scale q_r . c_j ks(page of j),   o_r = sum_j exp(s_rj - m_r) vs(page of j) d_j / sum_j exp(s_rj - m_r)
// with c, d the code values of K and V, which are exact in fp16.
//
// The products run on mfma_f32_16x16x32_f16 as S^T = C Q^T and O^T = D P^T, 16 query rows and 64 tokens at a time.
// Row m of the t-th 16-token S tile is token 16 (m / 4) + 4 t + m % 4 of the 64, so a lane (column = query row lane & 15,
// rows 4 (lane >> 4) .. + 3 of each tile) ends up with the scores of the 16 consecutive tokens 16 (lane >> 4) ..,
// which is the B operand of the second product when V is stored with tokens contiguous: one 16-byte load per lane is 16
// tokens of one dim, and no probability leaves its lane.
//
// Queries are scaled by a power of two per row (largest magnitude in [2^14, 2^15)) and held as one (bf16 rows, exact
// down to 2^-31 of the largest) or two fp16 pieces (fp32 rows: 22 bits, 2^-39 of the largest).  V's page scale, split
// into mantissa and exponent vs = a 2^e, joins the probability before its rounding: with m' >= max(log2-scores + e), an
// integer, p' = 2^(s + e - m' + 15) a lies in (0, 2^15], again one or two fp16 pieces, so what is rounded away is small
// against the largest contribution to the sum and not against the largest probability.  The integer reference makes
// every rescaling a power of two.  The softmax's sum adds 2^(s + e - m' + 15) 2^-e in fp32.
#include "paged.h"

using namespace vgx;

namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kTile = 64;                    // tokens of a tile
constexpr float kNeg = -3.0e38f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPre = 15;                     // probabilities lie below 2^15

struct AttnArgs {
    PagedLayer c;
    const void *q;
    void *out;
    int64_t ldq, ldo, ldt;
    const int32_t *table, *lens, *q_start;
    float *part;
    float scale;
    int N, B, H, R, cols, window, n_sink, splits, min_tiles;
};

// 16 query rows r0 .. of sequence b: row r is token r / R, head r % R of the group.
struct RowTile {
    int b, r0, rows, lo, n, len;
};

VGX_DEV int tiles_of(int n, int R) { return (int)(((int64_t)n * R + 15) >> 4); }

VGX_DEV RowTile row_tile(const AttnArgs &A, int64_t x) {
    RowTile t;
    int64_t place;
    if (A.q_start == nullptr) {
        const int per = tiles_of(1, A.R);
        t.b = x < (int64_t)A.B * per ? (int)(x / per) : -1;
        if (t.b < 0) return t;
        place = x - (int64_t)t.b * per;
    } else {
        t.b = find_unit(x, A.B, [&](int b) {
            const SeqRows r = seq_rows(A.q_start, b, A.N);
            return tiles_of(r.hi - r.lo, A.R);
        }, place);
        if (t.b < 0) return t;
    }
    const SeqRows r = seq_rows(A.q_start, t.b, A.N);
    t.lo = r.lo;
    t.n = r.hi - r.lo;
    t.r0 = (int)(place * 16);
    t.rows = (int)min((int64_t)16, (int64_t)t.n * A.R - t.r0);
    t.len = A.lens[t.b];
    return t;
}

// The 64-token tiles that some row of positions p_min .. p_max sees: `sinks` tiles from 0, then those from `lo` on.
struct Tiles {
    int sinks, lo, count, last;              // last: no token after it is visible
};
VGX_DEV Tiles visible_tiles(const AttnArgs &A, int p_min, int p_max) {
    Tiles t{0, 0, 0, 0};
    t.last = (int)min((int64_t)p_max, ((int64_t)A.cols << A.c.log_page) - 1);
    if (t.last < 0) return t;
    if (A.window > 0) {
        const int64_t lo = max((int64_t)0, (int64_t)p_min - A.window + 1);
        t.lo = (int)(lo / kTile);
        t.sinks = min((int)(((int64_t)A.n_sink + kTile - 1) / kTile), t.lo);
    }
    t.sinks = min(t.sinks, t.last / kTile + 1);
    t.count = t.sinks + max(0, t.last / kTile - t.lo + 1);
    return t;
}

// Eight code bytes to fp16.
template <int FMT>
VGX_DEV f16x8_t codes8(uint32_t a, uint32_t b) {
    union {
        vgx_f16x2_t h[4];
        f16x8_t v;
    } u;
    if constexpr (FMT == VGX_I8) {
        // 0x64uu is 1024 + u
        const vgx_f16x2_t off = {(_Float16)1152.0f, (_Float16)1152.0f};
        const auto two = [&](uint32_t w, uint32_t sel) {
            return __builtin_bit_cast(vgx_f16x2_t, __builtin_amdgcn_perm(0x64646464u, w, sel)) - off;
        };
        u.h[0] = two(a, 0x04010400u);
        u.h[1] = two(a, 0x04030402u);
        u.h[2] = two(b, 0x04010400u);
        u.h[3] = two(b, 0x04030402u);
    } else {
        u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
        u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
        u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false);
        u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
    }
    return u.v;
}

// Eight floats as PIECES fp16 vectors, the first rounded to nearest, the second holding what it left.
template <int PIECES>
VGX_DEV void pieces8(const float (&x)[8], f16x8_t (&o)[PIECES]) {
    union {
        uint32_t w[4];
        f16x8_t v;
    } hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        hi.w[i] = pack_f16x2(x[2 * i], x[2 * i + 1]);
        if constexpr (PIECES == 2) {
            const auto h = __builtin_bit_cast(vgx_f16x2_t, hi.w[i]);
            lo.w[i] = pack_f16x2(x[2 * i] - (float)h[0], x[2 * i + 1] - (float)h[1]);
        }
    }
    o[0] = hi.v;
    if constexpr (PIECES == 2) o[1] = lo.v;
}

template <bool BF16>
VGX_DEV void load8(const void *p, int64_t at, float (&x)[8]) {
    if constexpr (BF16) {
        const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + at);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = bf16_bits_to_float(u[i]);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        }
    } else {
        const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
        const float4 b = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
}

// Where a lane's 16-token groups of a tile lie: byte offset of the group's page (for this head), or no page.
struct Group {
    int64_t at;                  // page * G + head
    int off;                     // token within the page
    bool have;
};
VGX_DEV Group group_of(const AttnArgs &A, const int32_t *__restrict__ row, int g, int tok) {
    Group r;
    const int col = tok >> A.c.log_page;
    const int page = col < A.cols ? row[col] : -1;
    r.have = page >= 0 && page < A.c.n_pages;
    r.at = (int64_t)(r.have ? page : 0) * A.c.G + g;
    r.off = tok & ((1 << A.c.log_page) - 1);
    return r;
}

// One workgroup: a row tile, a kv head and a range of its key tiles, dealt to the waves in turn.
template <int FMT, int D, bool BF16>
__global__ __launch_bounds__(kThreads) void rows_kernel(const AttnArgs A) {
    constexpr int PIECES = BF16 ? 1 : 2, KS = D / 32, DT = D / 16, LD = D / 64;
    __shared__ float sm_m[kWaves][16], sm_l[kWaves][16], sm_o[kWaves][16][D + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, grp = lane >> 4;
    const int64_t x = blockIdx.x / (unsigned)A.c.G;
    const int g = (int)(blockIdx.x % (unsigned)A.c.G), split = blockIdx.y;
    const RowTile rt = row_tile(A, x);
    if (rt.b < 0) return;
    const int p0 = rt.len - rt.n;                                       // the position of the sequence's first query
    const int p_min = p0 + rt.r0 / A.R, p_max = p0 + (rt.r0 + rt.rows - 1) / A.R;
    const Tiles T = visible_tiles(A, p_min, p_max);
    const int per = max(A.min_tiles, (T.count + A.splits - 1) / A.splits), used = max(1, (T.count + per - 1) / per);
    if (split >= used) return;
    const int t_end = min(T.count, (split + 1) * per);
    const int r = rt.r0 + col;
    const bool live = col < rt.rows;
    const int p_row = live ? min(p0 + r / A.R, T.last) : -1;           // last visible token of this lane's row
    const int p_from = A.window > 0 && live ? p0 + r / A.R - A.window : -1;   // tokens after it, or below n_sink

    // the row's query, scaled by a power of two, as the lane's slices of the B operands
    f16x8_t qf[KS][PIECES];
    float q_unit;                                                        // what a unit of the product is worth
    {
        float y[KS][8], most = 0.0f;
        const int64_t at = (int64_t)(rt.lo + (live ? r / A.R : 0)) * A.ldq + (int64_t)(g * A.R + (live ? r % A.R : 0)) * D;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            load8<BF16>(A.q, at + (i >> 1) * 64 + grp * 16 + (i & 1) * 8, y[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(y[i][e]));
        }
        most = xor32_max(xor16_max(most));
        const int ex = __builtin_amdgcn_frexp_expf(most);               // most in [2^(ex - 1), 2^ex)
        const float sign = most == INFINITY ? NAN : A.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[i][e] = live ? ldexpf(y[i][e] * sign, kPre - ex) : 0.0f;
            pieces8<PIECES>(y[i], qf[i]);
        }
        q_unit = ldexpf(fabsf(A.scale) * kLog2e, ex - kPre);
    }

    const int32_t *__restrict__ row = A.table + (int64_t)rt.b * A.ldt;
    f32x4_t acc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[i] = f32x4_t{0, 0, 0, 0};
    float m = kNeg, l = 0.0f;

    for (int ti = split * per + wave; ti < t_end; ti += kWaves) {
        const int tok0 = (ti < T.sinks ? ti : T.lo + ti - T.sinks) * kTile;
        const Group kg = group_of(A, row, g, tok0 + (col >> 2) * 16), vg = group_of(A, row, g, tok0 + grp * 16);
        const float ks = A.c.ks[vg.at], vs = A.c.vs[vg.at];
        uint4 kw[4][LD], vw[DT];
        const uint8_t *kp = A.c.k + kg.at * A.c.head_bytes + (int64_t)(kg.off + (col & 3)) * D + grp * 16;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int h = 0; h < LD; ++h) kw[t][h] = *reinterpret_cast<const uint4 *>(kp + t * 4 * D + h * 64);
        const uint8_t *vp = A.c.v + vg.at * A.c.head_bytes + vg.off + ((int64_t)col << A.c.log_page);
#pragma unroll
        for (int i = 0; i < DT; ++i) vw[i] = *reinterpret_cast<const uint4 *>(vp + ((int64_t)(i * 16) << A.c.log_page));

        f32x4_t s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = f32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const uint4 w = kw[t][i >> 1];
                const f16x8_t a = (i & 1) ? codes8<FMT>(w.z, w.w) : codes8<FMT>(w.x, w.y);
#pragma unroll
                for (int p = PIECES - 1; p >= 0; --p)
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[i][p], s[t], 0, 0, 0);
            }
        }

        // which of the lane's 16 tokens its row sees: all, unless the tile lies on a border
        uint32_t vis = 0xFFFFu;
        const bool whole = tok0 + kTile - 1 <= min(p_min, T.last) &&
                           (A.window <= 0 || tok0 > p_max - A.window || tok0 + kTile <= A.n_sink) && __all(vg.have);
        if (!whole) {
            vis = 0;
            uint32_t any = 0;                                           // tokens that some row of the tile sees
            const int any_from = A.window > 0 ? p_min - A.window : -1;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int tok = tok0 + grp * 16 + i;
                if (vg.have && tok <= p_row && (tok > p_from || tok < A.n_sink)) vis |= 1u << i;
                if (vg.have && tok <= T.last && (tok > any_from || tok < A.n_sink)) any |= 1u << i;
            }
            // bytes of unseen tokens may hold anything, the NaN code among it, whose product with 0 is not 0
            uint32_t keep[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t n = any >> (4 * w);
                keep[w] = (n & 1 ? 0xFFu : 0) | (n & 2 ? 0xFF00u : 0) | (n & 4 ? 0xFF0000u : 0) | (n & 8 ? 0xFF000000u : 0);
            }
#pragma unroll
            for (int i = 0; i < DT; ++i) {
                vw[i].x &= keep[0];
                vw[i].y &= keep[1];
                vw[i].z &= keep[2];
                vw[i].w &= keep[3];
            }
        }
        // scales of a group that the row does not see may hold anything
        const float c = vis ? ks * q_unit : 0.0f, a = vis ? __builtin_amdgcn_frexp_mantf(vs) : 0.0f;
        const int e = vis ? __builtin_amdgcn_frexp_expf(vs) : 0;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (whole || (vis >> i & 1)) top = fmaxf(top, s[i >> 2][i & 3] * c);
        top += (float)e;
        if (__any(top > m)) {
            const float now = fmaxf(m, ceilf(xor32_max(xor16_max(top))));
            const float f = __builtin_amdgcn_exp2f(m - now);
            m = now;
            l *= f;
#pragma unroll
            for (int i = 0; i < DT; ++i) acc[i] *= f;
        }
        const float b = (float)kPre - (m - (float)e);
        float sum = 0.0f, pr[2][8];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float v = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], c, b));
            if (!whole) v = (vis >> i & 1) ? v : 0.0f;
            sum += v;
            pr[i >> 3][i & 7] = v * a;
        }
        l += ldexpf(sum, -e);
        f16x8_t pf[2][PIECES];
        pieces8<PIECES>(pr[0], pf[0]);
        pieces8<PIECES>(pr[1], pf[1]);
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            const f16x8_t v0 = codes8<FMT>(vw[i].x, vw[i].y), v1 = codes8<FMT>(vw[i].z, vw[i].w);
#pragma unroll
            for (int p = PIECES - 1; p >= 0; --p) {
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[0][p], acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[1][p], acc[i], 0, 0, 0);
            }
        }
    }

    // the waves' states joined in order
    l = xor32_sum(xor16_sum(l));
    if (grp == 0) {
        sm_m[wave][col] = m;
        sm_l[wave][col] = l;
    }
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sm_o[wave][col][i * 16 + grp * 4 + j] = acc[i][j];
    __syncthreads();
    for (int u = tid; u < 16 * (D / 4); u += kThreads) {
        const int rr = u / (D / 4), d = (u - rr * (D / 4)) * 4;
        if (rr >= rt.rows) continue;
        float M = kNeg, L = 0.0f, o[4] = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, sm_m[w][rr]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(sm_m[w][rr] - M);
            L = fmaf(f, sm_l[w][rr], L);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = fmaf(f, sm_o[w][rr][d + j], o[j]);
        }
        if (used > 1) {
            float *pp = A.part + (((x * A.c.G + g) * A.splits + split) * 16 + rr) * (D + 4);
            *reinterpret_cast<float4 *>(pp + d) = make_float4(o[0], o[1], o[2], o[3]);
            if (d == 0) {
                pp[D] = M;
                pp[D + 1] = L;
            }
            continue;
        }
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        const int rq = rt.r0 + rr;
        const int64_t at = (int64_t)(rt.lo + rq / A.R) * A.ldo + (int64_t)(g * A.R + rq % A.R) * D + d;
        if constexpr (BF16)
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(A.out) + at) =
                make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
        else
            *reinterpret_cast<float4 *>(static_cast<float *>(A.out) + at) =
                make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    }
}

// The splits of a row tile and head joined in order.
template <int D, bool BF16>
__global__ __launch_bounds__(kThreads) void merge_kernel(const AttnArgs A) {
    const int64_t x = blockIdx.x / (unsigned)A.c.G;
    const int g = (int)(blockIdx.x % (unsigned)A.c.G);
    const RowTile rt = row_tile(A, x);
    if (rt.b < 0) return;
    const int p0 = rt.len - rt.n;
    const Tiles T = visible_tiles(A, p0 + rt.r0 / A.R, p0 + (rt.r0 + rt.rows - 1) / A.R);
    const int per = max(A.min_tiles, (T.count + A.splits - 1) / A.splits), used = max(1, (T.count + per - 1) / per);
    if (used <= 1) return;
    const float *pp = A.part + (x * A.c.G + g) * A.splits * 16 * (D + 4);
    for (int u = threadIdx.x; u < rt.rows * D; u += kThreads) {
        const int rr = u / D, d = u - rr * D;
        float M = kNeg, L = 0.0f, o = 0.0f;
        for (int s = 0; s < used; ++s) M = fmaxf(M, pp[(s * 16 + rr) * (D + 4) + D]);
        for (int s = 0; s < used; ++s) {
            const float *q = pp + (s * 16 + rr) * (D + 4);
            const float f = __builtin_amdgcn_exp2f(q[D] - M);
            L = fmaf(f, q[D + 1], L);
            o = fmaf(f, q[d], o);
        }
        o *= L == 0.0f ? 0.0f : 1.0f / L;
        const int rq = rt.r0 + rr;
        const int64_t at = (int64_t)(rt.lo + rq / A.R) * A.ldo + (int64_t)(g * A.R + rq % A.R) * D + d;
        if constexpr (BF16) static_cast<uint16_t *>(A.out)[at] = (uint16_t)float_to_bf16_bits(o);
        else static_cast<float *>(A.out)[at] = o;
    }
}

// Workgroups of row tiles and heads, and into how many ranges each one's keys are split: enough workgroups to fill the
// GPU, each with a tile for every wave at least.
struct Plan {
    int64_t tiles, splits, bytes;
};
constexpr int64_t kMaxTokens = 1 << 30;      // positions, rows and windows fit 32 bits with room for their differences
constexpr int kTargetGroups = 1024, kMaxSplits = 64;
Plan plan_of(int64_t N, int64_t B, int64_t H, int64_t G, int64_t D, int64_t max_keys, int64_t window, int64_t n_sink) {
    Plan p;
    const int64_t R = H / G;
    p.tiles = N * R / 16 + B;                // a sequence's n rows make at most n R / 16 + 1 tiles
    int64_t keys = max_keys;
    if (window > 0) keys = std::min(keys, window + n_sink + 2 * kTile);
    const int64_t most = std::max<int64_t>(1, (keys / kTile + 1) / kWaves);
    p.splits = std::max<int64_t>(1, std::min({(kTargetGroups + p.tiles * G - 1) / (p.tiles * G), most, (int64_t)kMaxSplits}));
    p.bytes = p.splits > 1 ? p.tiles * G * p.splits * 16 * (D + 4) * 4 : 0;
    return p;
}

}  // namespace

extern "C" {

int64_t vgx_paged_attn_workspace_bytes(int64_t N, int64_t B, int64_t H, int64_t G, int64_t D, int64_t max_new,
                                       int64_t max_keys, int64_t window, int64_t n_sink) {
    if (N < 0 || B < 0 || H <= 0 || G <= 0 || max_new < 0 || max_keys < 0 || window < 0 || n_sink < 0) return VGX_E_SIZE;
    if (H % G || (D != 64 && D != 128)) return VGX_E_SHAPE;
    if (N > kMaxTokens || B > kMaxTokens || H > 65535 || max_keys > kMaxTokens) return VGX_E_LIMIT;
    return N == 0 || B == 0 ? 0 : plan_of(N, B, H, G, D, max_keys, window, n_sink).bytes;
}

int vgx_paged_attn(const vgx_paged_kv *kv, int64_t layer, int dtype, const void *q, int64_t ldq, void *out, int64_t ldo,
                   int64_t N, int64_t H, const int32_t *table, int64_t ldt, int64_t table_cols, const int32_t *lens,
                   const int32_t *q_start, int64_t B, int64_t max_new, int64_t max_keys, int64_t window, int64_t n_sink,
                   float scale, void *workspace, int64_t workspace_bytes, void *stream) {
    if (const int rc = check_paged(kv, layer)) return rc;
    if (dtype != VGX_F32 && dtype != VGX_BF16) return VGX_E_DTYPE;
    if (!q_start && N != B) return VGX_E_SIZE;
    const int64_t need = vgx_paged_attn_workspace_bytes(N, B, H, kv->G, kv->D, max_new, max_keys, window, n_sink);
    if (need < 0) return (int)need;
    if (N == 0 || B == 0) return VGX_OK;
    if (const int rc = check_table(table, ldt, table_cols)) return rc;
    if (table_cols * kv->page >= kMaxTokens) return VGX_E_LIMIT;
    if (!q || !out || !lens) return VGX_E_ARG;
    if (ldq < H * kv->D || ldo < H * kv->D) return VGX_E_SIZE;
    const int64_t es = dtype == VGX_F32 ? 4 : 2;
    if (((uintptr_t)q | (uintptr_t)out) % 16 || ldq * es % 16 || ldo * es % 16) return VGX_E_ALIGN;
    if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) return VGX_E_ARENA;
    const Plan p = plan_of(N, B, H, kv->G, kv->D, max_keys, window, n_sink);
    if (p.tiles * kv->G > 0x7FFFFFFF) return VGX_E_LIMIT;
    // no position reaches kMaxTokens: a window of that many tokens is none
    const int win = window >= kMaxTokens ? 0 : (int)window, sink = (int)std::min(n_sink, kMaxTokens);
    const AttnArgs A{paged_layer(kv, layer), q, out, ldq, ldo, ldt, table, lens, q_start, static_cast<float *>(workspace),
                     scale, (int)N, (int)B, (int)H, (int)(H / kv->G), (int)table_cols, win, sink,
                     (int)p.splits, kWaves};
    const int64_t tiles = q_start ? p.tiles : B * ((H / kv->G + 15) / 16);
    const dim3 grid((unsigned)(tiles * kv->G), (unsigned)p.splits);
    const auto launch = [&](auto fm, auto dm, auto bf) -> int {
        hipLaunchKernelGGL((rows_kernel<fm.value, dm.value, bf.value>), grid, dim3(kThreads), 0, (hipStream_t)stream, A);
        VGX_CHECK_LAUNCH();
        if (p.splits > 1) {
            hipLaunchKernelGGL((merge_kernel<dm.value, bf.value>), dim3(grid.x), dim3(kThreads), 0, (hipStream_t)stream, A);
            VGX_CHECK_LAUNCH();
        }
        return VGX_OK;
    };
    return with_format(kv->fmt, kv->D, dtype == VGX_BF16, launch);
}

}  // extern "C"
