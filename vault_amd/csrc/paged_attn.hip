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
    int32_t *tickets;            // one per row tile and head, zero between calls; NULL: a launch of its own merges
    int N, B, H, R, cols, window, n_sink, splits, per;
};

// RT query rows r0 .. of sequence b: row r is token r / R, head r % R of the group.
struct RowTile {
    int b, r0, rows, lo, n, len;
};

template <int RT>
VGX_DEV int tiles_of(int n, int R) { return (int)(((int64_t)n * R + RT - 1) / RT); }

template <int RT>
VGX_DEV RowTile row_tile(const AttnArgs &A, int64_t x) {
    RowTile t;
    int64_t place;
    if (A.q_start == nullptr) {
        const int per = tiles_of<RT>(1, A.R);
        t.b = x < (int64_t)A.B * per ? (int)(x / per) : -1;
        if (t.b < 0) return t;
        place = x - (int64_t)t.b * per;
    } else {
        t.b = find_unit(x, A.B, [&](int b) {
            const SeqRows r = seq_rows(A.q_start, b, A.N);
            return tiles_of<RT>(r.hi - r.lo, A.R);
        }, place);
        t.b = __builtin_amdgcn_readfirstlane(t.b);
        if (t.b < 0) return t;
    }
    const SeqRows r = seq_rows(A.q_start, t.b, A.N);
    t.lo = r.lo;
    t.n = r.hi - r.lo;
    t.r0 = __builtin_amdgcn_readfirstlane((int)place) * RT;
    t.rows = (int)min((int64_t)RT, (int64_t)t.n * A.R - t.r0);
    t.len = max(A.lens[t.b], 0);            // so that positions, which are len - n and on, fit 32 bits
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

// Eight K codes to fp16 for the scores of bf16 queries: I8 bytes as they are, which are the fp16 numbers u 2^-24 (below
// the normal range, exact), so that -128 2^-24 times the sum of its query belongs to every score.  Half the instructions
// of codes8; the offset costs 2^-24 128 sum |q|, far below what a bf16 result shows.
template <int FMT>
VGX_DEV f16x8_t codes8_offset(uint32_t a, uint32_t b) {
    if constexpr (FMT != VGX_I8) return codes8<FMT>(a, b);
    union {
        uint32_t w[4];
        f16x8_t v;
    } u;
    u.w[0] = __builtin_amdgcn_perm(0u, a, 0x0C010C00u);
    u.w[1] = __builtin_amdgcn_perm(0u, a, 0x0C030C02u);
    u.w[2] = __builtin_amdgcn_perm(0u, b, 0x0C010C00u);
    u.w[3] = __builtin_amdgcn_perm(0u, b, 0x0C030C02u);
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

// The pages of a tile's tokens, as a lane needs them: of the 16-token group whose K rows it loads (lane & 15) / 4, and of
// the group whose scores and V bytes it holds (lane / 16).  ONE: pages of 64 tokens or more, so that both are the tile's
// one page, the same for the whole wave (scalar registers, scalar loads).  `have` is whether there is a page.
template <bool ONE>
struct Pages {
    int k, v;
    bool have;
};
// A zero that the compiler takes for a lane's own value.  Added to the address of a wave-uniform load it makes that a
// vector load: scalar loads share a counter with LDS operations and return out of order with them, so every wait for
// either would wait for both.
VGX_DEV int lane_zero() {
    int z;
    asm("v_mov_b32 %0, 0" : "=v"(z));
    return z;
}
VGX_DEV float load_lane(const float *p) {
    return *reinterpret_cast<const float *>(reinterpret_cast<const char *>(p) + (uint32_t)lane_zero());
}

// A copy that stays one: without it the loop keeps a loaded value in two registers and moves it at the end of the
// iteration that requested it, which waits for every load under way.
VGX_DEV float taken(float x) {
    float y;
    asm volatile("v_mov_b32 %0, %1" : "=v"(y) : "v"(x));
    return y;
}

// The table entries themselves, whose loads are issued a tile before anything looks at them.
struct Entries {
    int k, v;
};
template <bool ONE>
VGX_DEV Entries entries_of(const AttnArgs &A, const int32_t *__restrict__ row, int tok0) {
    // past the table: its last entry, for tokens that no row sees
    const auto entry = [&](int tok) { return row[min((int)((uint32_t)tok >> A.c.log_page), A.cols - 1)]; };
    if constexpr (ONE) {
        const int e = entry(tok0 + lane_zero());
        return {e, e};
    } else {
        return {entry(tok0 + ((threadIdx.x & 15) >> 2) * 16), entry(tok0 + ((threadIdx.x & 63) >> 4) * 16)};
    }
}
template <bool ONE>
VGX_DEV Pages<ONE> pages_of(const AttnArgs &A, const Entries &e) {
    Pages<ONE> p;
    if constexpr (ONE) {
        const int id = __builtin_amdgcn_readfirstlane(e.v);
        p.have = id >= 0 && id < A.c.n_pages;
        p.k = p.v = p.have ? id : 0;
    } else {
        p.have = e.v >= 0 && e.v < A.c.n_pages;
        p.v = p.have ? e.v : 0;
        p.k = e.k >= 0 && e.k < A.c.n_pages ? e.k : 0;
    }
    return p;
}
template <bool ONE>
VGX_DEV bool all_have(const Pages<ONE> &p) {
    if constexpr (ONE) return p.have;
    else return __all(p.have);
}

// Where the lane's K rows (token 4 t + lane % 4 of its group, from its 16 bytes on) and V rows (dim lane % 16) begin.
template <bool ONE, int D>
VGX_DEV const uint8_t *k_rows(const AttnArgs &A, const Pages<ONE> &p, int g, int tok0, int t) {
    const int lane = threadIdx.x & 63, col = lane & 15, in = (1 << A.c.log_page) - 1;
    const int group = (col >> 2) * 16, rest = (t * 4 + (col & 3)) * D + (lane >> 4) * 16;
    const uint8_t *base = A.c.k + ((int64_t)p.k * A.c.G + g) * A.c.head_bytes;
    if constexpr (ONE) return base + (tok0 & in) * D + (uint32_t)(group * D + rest);
    else return base + ((tok0 + group) & in) * D + rest;
}
template <bool ONE>
VGX_DEV const uint8_t *v_rows(const AttnArgs &A, const Pages<ONE> &p, int g, int tok0, int dim0) {
    const int lane = threadIdx.x & 63, in = (1 << A.c.log_page) - 1;
    const int group = (lane >> 4) * 16, rest = (dim0 + (lane & 15)) << A.c.log_page;
    const uint8_t *base = A.c.v + ((int64_t)p.v * A.c.G + g) * A.c.head_bytes;
    if constexpr (ONE) return base + (tok0 & in) + (uint32_t)(group + rest);
    else return base + ((tok0 + group) & in) + rest;
}

// Rows of one 16-column tile, as a lane sees them: its row's last visible token, the token that its window starts after,
// and its query as the lane's slices of the B operands, scaled by a power of two; `unit`: what a unit of the product is
// worth in the exponent.
template <int D, int PIECES>
struct Query {
    f16x8_t f[D / 32][PIECES];
    float unit;
    int last, from;
};
template <int D, bool BF16>
VGX_DEV void load_query(const AttnArgs &A, const RowTile &rt, int g, int r, Query<D, BF16 ? 1 : 2> &q) {
    constexpr int KS = D / 32;
    const int grp = (threadIdx.x & 63) >> 4;
    const bool live = r < rt.r0 + rt.rows;
    float y[KS][8], most = 0.0f;
    const int64_t at = (int64_t)(rt.lo + (live ? r / A.R : 0)) * A.ldq + (int64_t)(g * A.R + (live ? r % A.R : 0)) * D;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
        load8<BF16>(A.q, at + (i >> 1) * 64 + grp * 16 + (i & 1) * 8, y[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(y[i][e]));
    }
    most = xor32_max(xor16_max(most));
    const int ex = __builtin_amdgcn_frexp_expf(most);                   // most in [2^(ex - 1), 2^ex)
    const float sign = most == INFINITY ? NAN : A.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = live ? ldexpf(y[i][e] * sign, kPre - ex) : 0.0f;
        pieces8<BF16 ? 1 : 2>(y[i], q.f[i]);
    }
    q.unit = ldexpf(fabsf(A.scale) * kLog2e, ex - kPre);
}
template <int D, int PIECES>
VGX_DEV void see(const AttnArgs &A, const RowTile &rt, int r, int last, Query<D, PIECES> &q) {
    const bool live = r < rt.r0 + rt.rows;
    const int p = rt.len - rt.n + r / A.R;
    q.last = live ? min(p, last) : -1;
    q.from = A.window > 0 && live ? p - A.window : -1;
}

// Which of the 16 tokens from tok a row sees that sees those up to `last` after `from` and those below n_sink.
VGX_DEV uint32_t seen16(int tok, int last, int from, int n_sink) {
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (tok + i <= last && (tok + i > from || tok + i < n_sink)) v |= 1u << i;
    return v;
}

// Bytes of unseen tokens may hold anything, the NaN code among it, whose product with 0 is not 0.
VGX_DEV void keep_bytes(uint32_t any, uint32_t (&keep)[4]) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const uint32_t n = any >> (4 * w);
        keep[w] = (n & 1 ? 0xFFu : 0) | (n & 2 ? 0xFF00u : 0) | (n & 4 ? 0xFF0000u : 0) | (n & 8 ? 0xFF000000u : 0);
    }
}

// One step of a row's softmax, in two halves: new_maximum() moves the row's reference m on to the products s of the lane's
// 16 tokens, and returns (for the wave) whether sums so far have to be multiplied by `f`; probabilities() makes the
// products the B operands pf of the second product and adds to the row's sum l.  `shift` belongs to every product.  `vis`: tokens that the row sees, all 16
// where WHOLE.  The page's V scale a 2^e: with two pieces a multiplies the exponential, with one its logarithm is added to
// the exponent (2^-17 of a probability that is then rounded to 2^-12); WHOLE with one piece takes positive scales only.
// FULL (one piece, one page for all lanes): l is the row's sum, the same in all of its four lanes, added up by the matrix
// unit from the rounded probabilities; otherwise each lane's own part.  Scales of a group that the row does not see may
// hold anything.
template <bool WHOLE>
VGX_DEV bool new_maximum(const f32x4_t (&s)[4], uint32_t vis, float ks, float vs, float unit, float shift, float &m, float &l,
                         float &f) {
    const bool some = WHOLE || vis != 0;
    const float c = some ? ks * unit : 0.0f;
    const int e = some ? __builtin_amdgcn_frexp_expf(vs) : 0;
    float top = -INFINITY;                                    // c is not negative: the largest product has the largest score
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, WHOLE || (vis >> i & 1) ? s[i >> 2][i & 3] : -INFINITY);
    top = fmaf(top + shift, c, (float)e);                     // NaN where the row sees nothing: no new maximum
    if (!__any(top > m)) return false;
    const float now = fmaxf(m, ceilf(xor32_max(xor16_max(top))));
    f = __builtin_amdgcn_exp2f(m - now);
    m = now;
    l *= f;
    return true;
}
template <bool WHOLE, bool FULL, int PIECES>
VGX_DEV void probabilities(const f32x4_t (&s)[4], uint32_t vis, float ks, float vs, float unit, float shift, float m,
                           float &l, f16x8_t (&pf)[2][PIECES]) {
    const bool some = WHOLE || vis != 0;
    const float c = some ? ks * unit : 0.0f, a = some ? __builtin_amdgcn_frexp_mantf(vs) : 0.0f;
    const int e = some ? __builtin_amdgcn_frexp_expf(vs) : 0;
    float b = fmaf(shift, c, (float)kPre - (m - (float)e)), back = 1.0f;
    if (PIECES == 1 && (WHOLE || a > 0.0f)) {
        b += __builtin_amdgcn_logf(a);                        // log2
        back = __builtin_amdgcn_rcpf(a);
    }
    float sum = 0.0f, pr[2][8];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float v = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], c, b));
        if (!WHOLE) v = (vis >> i & 1) ? v : 0.0f;
        if (!(WHOLE && FULL)) sum += v;
        pr[i >> 3][i & 7] = PIECES == 1 ? v : v * a;
    }
    if (PIECES == 1 && !WHOLE && __any(!(a > 0.0f))) {        // a scale of 0, or NaN
        const float w = a > 0.0f ? 1.0f : a;
#pragma unroll
        for (int i = 0; i < 16; ++i) pr[i >> 3][i & 7] *= w;
    }
    pieces8<PIECES>(pr[0], pf[0]);
    pieces8<PIECES>(pr[1], pf[1]);
    if constexpr (WHOLE && FULL) {
        const f16x8_t one = {1, 1, 1, 1, 1, 1, 1, 1};
        f32x4_t t = {0, 0, 0, 0};
        t = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, pf[0][0], t, 0, 0, 0);
        t = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, pf[1][0], t, 0, 0, 0);
        l += ldexpf(t[0] * back, -e);
    } else {
        sum = ldexpf(sum * back, -e);
        l += FULL ? xor32_sum(xor16_sum(sum)) : sum;
    }
}

// The key tiles of a split, `per` of them, whatever the sequence's length, so that the first one is known before the length
// is (the last split takes what a hint too small leaves); and how many splits have any (one at least).
struct Range {
    int first, end, used;
};
VGX_DEV Range range_of(const AttnArgs &A, int count, int split) {
    const int used = min(A.splits, max(1, (count + A.per - 1) / A.per));
    return {split * A.per, split == A.splits - 1 ? count : min(count, (split + 1) * A.per), used};
}

template <bool BF16>
VGX_DEV void store_out4(void *out, int64_t at, const float (&o)[4], float inv) {
    if constexpr (BF16)
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(out) + at) =
            make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
    else
        *reinterpret_cast<float4 *>(static_cast<float *>(out) + at) =
            make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
}
VGX_DEV float inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
VGX_DEV int64_t out_at(const AttnArgs &A, const RowTile &rt, int g, int row, int D) {
    const int r = rt.r0 + row;
    return (int64_t)(rt.lo + r / A.R) * A.ldo + (int64_t)(g * A.R + r % A.R) * D;
}

// Two floats of a partial state, written to and read from the level that all dies of the GPU share: a workgroup on one of
// them joins what others wrote, within one launch (ordered by the ticket; a fence would write back a whole cache).
VGX_DEV void put2(float *p, float a, float b) {
    const uint64_t v = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <bool SHARED>
VGX_DEV float2 get2(const float *p) {
    if constexpr (!SHARED) return *reinterpret_cast<const float2 *>(p);
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// Row rr of a tile of RT rows from its splits' partial states, by the 16 threads that ask for it: all loads of eight
// splits at once.
template <int RT, int D, bool BF16, bool SHARED>
VGX_DEV void join_rows(const AttnArgs &A, const RowTile &rt, int64_t x, int g, int used, int rr) {
    constexpr int V = D / 32;                        // pairs of floats of a thread
    const int d = (threadIdx.x & 15) * 2;
    if (rr >= rt.rows) return;
    const int64_t step = (int64_t)RT * (D + 4);
    const float *pp = A.part + (x * A.c.G + g) * A.splits * step + (int64_t)rr * (D + 4);
    float M = kNeg, L = 0.0f, o[V][2] = {};
    for (int s0 = 0; s0 < used; s0 += 8) {
        float2 ml[8], v[8][V];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            ml[u] = make_float2(kNeg, 0.0f);
#pragma unroll
            for (int j = 0; j < V; ++j) v[u][j] = make_float2(0.0f, 0.0f);
            if (s0 + u >= used) continue;
            const float *w = pp + (s0 + u) * step;
            ml[u] = get2<SHARED>(w + D);
#pragma unroll
            for (int j = 0; j < V; ++j) v[u][j] = get2<SHARED>(w + j * 32 + d);
        }
        float now = M;
#pragma unroll
        for (int u = 0; u < 8; ++u) now = fmaxf(now, ml[u].x);
        const float f0 = __builtin_amdgcn_exp2f(M - now);
        M = now;
        L *= f0;
#pragma unroll
        for (int j = 0; j < V; ++j) o[j][0] *= f0, o[j][1] *= f0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float f = s0 + u < used ? __builtin_amdgcn_exp2f(ml[u].x - M) : 0.0f;
            L = fmaf(f, ml[u].y, L);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                o[j][0] = fmaf(f, v[u][j].x, o[j][0]);
                o[j][1] = fmaf(f, v[u][j].y, o[j][1]);
            }
        }
    }
    const int64_t at = out_at(A, rt, g, rr, D) + d;
    const float inv = inverse(L);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if constexpr (BF16)
            *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(A.out) + at + j * 32) = pack_bf16x2(o[j][0] * inv, o[j][1] * inv);
        else
            *reinterpret_cast<float2 *>(static_cast<float *>(A.out) + at + j * 32) = make_float2(o[j][0] * inv, o[j][1] * inv);
    }
}

// One workgroup: a tile of 16 rows, a kv head and a range of its key tiles, dealt to the waves in turn.  For few query
// rows per sequence: codes go from memory to registers of the one wave that multiplies them.
template <int FMT, int D, bool BF16, bool ONE>
__global__ __launch_bounds__(kThreads) void rows_kernel(const AttnArgs A) {
    constexpr int PIECES = BF16 ? 1 : 2, KS = D / 32, DT = D / 16, LD = D / 64;
    __shared__ float sm_m[kWaves][16], sm_l[kWaves][16], sm_o[kWaves][16][D + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15,
              grp = lane >> 4;
    const int64_t x = blockIdx.x / (unsigned)A.c.G;
    const int g = (int)(blockIdx.x % (unsigned)A.c.G), split = blockIdx.y;
    const RowTile rt = row_tile<16>(A, x);
    if (rt.b < 0) return;
    const int32_t *__restrict__ row = A.table + (int64_t)rt.b * A.ldt;
    // what does not wait for the sequence's length: without a window the first tile's table entries, and the query
    Entries ids{-1, -1};
    if (A.window <= 0) ids = entries_of<ONE>(A, row, (split * A.per + wave) * kTile);
    Query<D, PIECES> q;
    load_query<D, BF16>(A, rt, g, rt.r0 + col, q);
    const int p0 = rt.len - rt.n;                                       // the position of the sequence's first query
    const int p_min = p0 + rt.r0 / A.R, p_max = p0 + (rt.r0 + rt.rows - 1) / A.R;
    const Tiles T = visible_tiles(A, p_min, p_max);
    const Range R = range_of(A, T.count, split);
    if (split >= R.used) return;
    see(A, rt, rt.r0 + col, T.last, q);
    const auto token_of = [&](int ti) { return (ti < T.sinks ? ti : T.lo + ti - T.sinks) * kTile; };
    if (A.window > 0 && R.first + wave < R.end) ids = entries_of<ONE>(A, row, token_of(R.first + wave));

    f32x4_t acc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[i] = f32x4_t{0, 0, 0, 0};
    float m = kNeg, l = 0.0f;

    // K of the next tile is requested as soon as this one's scores are there (64 ragged sequences of up to 16384 tokens:
    // 250 us without, 245 with)
    uint4 kw[4][LD];
    Pages<ONE> pg{0, 0, false};
    float ks_in = 0.0f, vs_in = 0.0f;
    const auto request = [&](int ti) {
        pg = pages_of<ONE>(A, ids);
        const uint8_t *kp = k_rows<ONE, D>(A, pg, g, token_of(ti), 0);
        ks_in = load_lane(A.c.ks + ((int64_t)pg.v * A.c.G + g));
        vs_in = load_lane(A.c.vs + ((int64_t)pg.v * A.c.G + g));
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int h = 0; h < LD; ++h) kw[t][h] = *reinterpret_cast<const uint4 *>(kp + t * 4 * D + h * 64);
        if (ti + kWaves < R.end) ids = entries_of<ONE>(A, row, token_of(ti + kWaves));
    };
    if (R.first + wave < R.end) request(R.first + wave);
    for (int ti = R.first + wave; ti < R.end; ti += kWaves) {
        const int tok0 = token_of(ti);
        uint4 vw[DT];
        const uint8_t *vp = v_rows<ONE>(A, pg, g, tok0, 0);
#pragma unroll
        for (int i = 0; i < DT; ++i) vw[i] = *reinterpret_cast<const uint4 *>(vp + ((i * 16) << A.c.log_page));
        const float ks = taken(ks_in), vs = taken(vs_in);
        const bool have = pg.have, all = all_have(pg);

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
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q.f[i][p], s[t], 0, 0, 0);
            }
        }
        if (ti + kWaves < R.end) request(ti + kWaves);

        const bool whole = tok0 + kTile - 1 <= min(p_min, T.last) &&
                           (A.window <= 0 || tok0 > p_max - A.window || tok0 + kTile <= A.n_sink) && all &&
                           (PIECES == 2 || __all(vs > 0.0f));
        float f;
        f16x8_t pf[2][PIECES];
        bool moved;
        if (whole) {
            moved = new_maximum<true>(s, 0, ks, vs, q.unit, 0.0f, m, l, f);
            probabilities<true, false>(s, 0, ks, vs, q.unit, 0.0f, m, l, pf);
        } else {
            const uint32_t vis = have ? seen16(tok0 + grp * 16, q.last, q.from, A.n_sink) : 0;
            uint32_t keep[4];
            keep_bytes(have ? seen16(tok0 + grp * 16, T.last, A.window > 0 ? p_min - A.window : -1, A.n_sink) : 0, keep);
#pragma unroll
            for (int i = 0; i < DT; ++i) {
                vw[i].x &= keep[0];
                vw[i].y &= keep[1];
                vw[i].z &= keep[2];
                vw[i].w &= keep[3];
            }
            moved = new_maximum<false>(s, vis, ks, vs, q.unit, 0.0f, m, l, f);
            probabilities<false, false>(s, vis, ks, vs, q.unit, 0.0f, m, l, pf);
        }
        if (moved) {
#pragma unroll
            for (int i = 0; i < DT; ++i) acc[i] *= f;
        }
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
        if (R.used > 1) {
            float *pp = A.part + (((x * A.c.G + g) * A.splits + split) * 16 + rr) * (D + 4);
            if (A.tickets != nullptr) {
                put2(pp + d, o[0], o[1]);
                put2(pp + d + 2, o[2], o[3]);
                if (d == 0) put2(pp + D, M, L);
            } else {
                *reinterpret_cast<float4 *>(pp + d) = make_float4(o[0], o[1], o[2], o[3]);
                if (d == 0) *reinterpret_cast<float2 *>(pp + D) = make_float2(M, L);
            }
            continue;
        }
        store_out4<BF16>(A.out, out_at(A, rt, g, rr, D) + d, o, inverse(L));
    }
    if (R.used == 1 || A.tickets == nullptr) return;
    // the workgroup that finishes a row tile and head last joins its splits and leaves the ticket at zero
    __shared__ int last;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                    // this thread's partials have arrived
    __syncthreads();
    int32_t *ticket = A.tickets + x * A.c.G + g;
    if (tid == 0) last = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == R.used - 1;
    __syncthreads();
    if (!last) return;
    if (tid == 0) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    join_rows<16, D, BF16, true>(A, rt, x, g, R.used, tid / 16);
}

// One workgroup: a tile of 128 rows (64 of fp32), 32 (16) to a wave, a kv head and a range of its key tiles.  For many
// query rows.  K codes go to the registers of every wave that multiplies them (the waves' loads meet in the vector cache);
// V is converted once, a quarter by each wave, and passes through shared memory in fp16, in the order in which the waves'
// operands read it (16 bytes a lane, lane after lane).  With K in shared memory too the matrix unit waited for it: a wave
// of 32 rows takes 1 KB of it for every two matrix instructions, 32 cycles, and shared memory gives 64 bytes a cycle to
// all four SIMDs (1024 queries on 9216 keys, 12 / 2 heads: 89 us).
template <bool BF16>
constexpr int kBlockRows = BF16 ? 128 : 64;
template <int FMT, int D, bool BF16, bool ONE>
__global__ __launch_bounds__(kThreads, 2) void block_kernel(const AttnArgs A) {
    constexpr int PIECES = BF16 ? 1 : 2, KS = D / 32, DT = D / 16, LD = D / 64, QT = BF16 ? 2 : 1, VT = DT / kWaves;
    constexpr bool FULL = ONE && PIECES == 1, OFFSET = FMT == VGX_I8 && BF16;
    __shared__ f16x8_t vf[2][2 * DT][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15,
              grp = lane >> 4;
    const int64_t x = blockIdx.x / (unsigned)A.c.G;
    const int g = (int)(blockIdx.x % (unsigned)A.c.G), split = blockIdx.y;
    const RowTile rt = row_tile<kBlockRows<BF16>>(A, x);
    if (rt.b < 0) return;
    const int p0 = rt.len - rt.n;
    const int p_min = p0 + rt.r0 / A.R, p_max = p0 + (rt.r0 + rt.rows - 1) / A.R;
    const Tiles T = visible_tiles(A, p_min, p_max);
    const Range R = range_of(A, T.count, split);
    if (split >= R.used) return;
    // this wave's rows and their positions
    const int w0 = rt.r0 + wave * 16 * QT, w_end = min(w0 + 16 * QT, rt.r0 + rt.rows);
    const bool idle = w0 >= w_end;
    const int w_min = p0 + w0 / A.R, w_max = idle ? -1 : p0 + (w_end - 1) / A.R;
    const int32_t *__restrict__ row = A.table + (int64_t)rt.b * A.ldt;
    const int n = max(0, R.end - R.first);
    const auto token_of = [&](int i) {                 // of the i-th tile of this range
        const int ti = R.first + min(i, n - 1);
        return (ti < T.sinks ? ti : T.lo + ti - T.sinks) * kTile;
    };

    // What is on its way: the table entries of the tile after next (`ids`), K codes of the next one (this wave's operands,
    // all of them), V codes of the next one (its quarter) and that tile's scales.
    Entries ids;
    vgx_u32x4_t kc[4][LD], vc[VT];
    float ks_next = 0.0f, vs_next = 0.0f;
    bool have_next = false, all_next = false;
    Pages<ONE> pg;
    const auto fetch_k = [&](int i, auto half) {
        const uint8_t *kp = k_rows<ONE, D>(A, pg, g, token_of(i), 0);
#pragma unroll
        for (int t = 2 * half.value; t < 2 * half.value + 2; ++t)
#pragma unroll
            for (int h = 0; h < LD; ++h) kc[t][h] = *reinterpret_cast<const vgx_u32x4_t *>(kp + t * 4 * D + h * 64);
    };
    const auto fetch_v = [&](int i) {
        const uint8_t *vp = v_rows<ONE>(A, pg, g, token_of(i), wave * VT * 16);
#pragma unroll
        for (int j = 0; j < VT; ++j) vc[j] = *reinterpret_cast<const vgx_u32x4_t *>(vp + ((j * 16) << A.c.log_page));
        const int64_t at = (int64_t)pg.v * A.c.G + g;
        ks_next = load_lane(A.c.ks + at);
        vs_next = load_lane(A.c.vs + at);
        have_next = pg.have;
        all_next = all_have(pg);
    };
    // the pages of tile i, and the request for the entries of the one after it
    const auto turn = [&](int i) {
        pg = pages_of<ONE>(A, ids);
        ids = entries_of<ONE>(A, row, token_of(i + 1));
    };
    const auto stage = [&](int buf) {
#pragma unroll
        for (int j = 0; j < VT; ++j) {
            vf[buf][(wave * VT + j) * 2][lane] = codes8<FMT>(vc[j][0], vc[j][1]);
            vf[buf][(wave * VT + j) * 2 + 1][lane] = codes8<FMT>(vc[j][2], vc[j][3]);
        }
    };
    // Codes of tokens that no row of the workgroup sees become 0.
    const auto drop_unseen = [&](int tok0) {
        const bool inside = tok0 + kTile - 1 <= T.last && all_next &&
                            (A.window <= 0 || tok0 > p_min - A.window || tok0 + kTile <= A.n_sink);
        if (inside) return;
        uint32_t keep[4];
        keep_bytes(have_next ? seen16(tok0 + grp * 16, T.last, A.window > 0 ? p_min - A.window : -1, A.n_sink) : 0, keep);
#pragma unroll
        for (int j = 0; j < VT; ++j)
#pragma unroll
            for (int w = 0; w < 4; ++w) vc[j][w] &= keep[w];
    };
    Query<D, PIECES> q[QT];
    float shift[QT], m[QT], l[QT];
    f32x4_t acc[QT][DT];
    const auto scores = [&](f32x4_t (&s)[QT][4]) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int c = 0; c < QT; ++c) s[c][t] = f32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const uint32_t a = kc[t][i >> 1][(i & 1) * 2], b = kc[t][i >> 1][(i & 1) * 2 + 1];
                const f16x8_t k = OFFSET ? codes8_offset<FMT>(a, b) : codes8<FMT>(a, b);
#pragma unroll
                for (int p = PIECES - 1; p >= 0; --p)
#pragma unroll
                    for (int c = 0; c < QT; ++c)
                        s[c][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[c].f[i][p], s[c][t], 0, 0, 0);
            }
        }
    };
    const auto rescale = [&](int c, float f) {
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[c][i] *= f;
    };
    const auto values = [&](int buf, const f16x8_t (&pf)[QT][2][PIECES]) {
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            const f16x8_t v0 = vf[buf][i * 2][lane], v1 = vf[buf][i * 2 + 1][lane];
#pragma unroll
            for (int p = PIECES - 1; p >= 0; --p)
#pragma unroll
                for (int c = 0; c < QT; ++c) {
                    acc[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[c][0][p], acc[c][i], 0, 0, 0);
                    acc[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[c][1][p], acc[c][i], 0, 0, 0);
                }
        }
    };

    if (n > 0) {
        ids = entries_of<ONE>(A, row, token_of(0));
        turn(0);
        fetch_v(0);
        fetch_k(0, std::integral_constant<int, 0>{});
        fetch_k(0, std::integral_constant<int, 1>{});
    }
#pragma unroll
    for (int c = 0; c < QT; ++c) {
        load_query<D, BF16>(A, rt, g, w0 + c * 16 + col, q[c]);
        see(A, rt, w0 + c * 16 + col, T.last, q[c]);
        shift[c] = 0.0f;
        if constexpr (OFFSET) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += (float)q[c].f[i][0][e];
            shift[c] = xor32_sum(xor16_sum(sum)) * (-128.0f * 0x1p-24f);
            q[c].unit *= 0x1p24f;
        }
        m[c] = kNeg;
        l[c] = 0.0f;
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[c][i] = f32x4_t{0, 0, 0, 0};
    }
    float ks = 0.0f, vs = 0.0f;                        // of the tile in hand
    bool have = false;
    if (n > 0) {
        drop_unseen(token_of(0));
        stage(0);
        ks = taken(ks_next), vs = taken(vs_next), have = have_next;
        turn(1);
        fetch_v(1);
    }
    __syncthreads();
    // Step i: V of tile i is in buffer i % 2, its K in registers; V of tile i + 1 is on its way, pg are its pages.  (Past
    // the last tile the last one is requested again and not used.)
    for (int i = 0; i < n; ++i) {
        const int buf = i & 1, tok0 = token_of(i);
        // all rows of the wave see all of the tile in hand
        const bool plain = tok0 + kTile - 1 <= min(w_min, T.last) &&
                           (A.window <= 0 || tok0 > w_max - A.window || tok0 + kTile <= A.n_sink) &&
                           (ONE ? have : (bool)__all(have)) && (PIECES == 2 || __all(vs > 0.0f));
        f32x4_t s[QT][4];
        f16x8_t pf[QT][2][PIECES];
        scores(s);
        // the softmax before another wave's matrix instructions, which run on without being issued (1024 queries on 36864
        // keys: 273 us, 279 at equal priorities, 276 with the products first)
        __builtin_amdgcn_s_setprio(1);
        __builtin_amdgcn_sched_barrier(0);
        fetch_k(i + 1, std::integral_constant<int, 0>{});
        bool moved = false;
        float f[QT];
        uint32_t vis[QT];
#pragma unroll
        for (int c = 0; c < QT; ++c) f[c] = 1.0f, vis[c] = 0;
        if (plain) {
#pragma unroll
            for (int c = 0; c < QT; ++c)
                moved |= new_maximum<true>(s[c], 0, ks, vs, q[c].unit, shift[c], m[c], l[c], f[c]);
        } else {
#pragma unroll
            for (int c = 0; c < QT; ++c) {
                vis[c] = have ? seen16(tok0 + grp * 16, q[c].last, q[c].from, A.n_sink) : 0u;
                moved |= new_maximum<false>(s[c], vis[c], ks, vs, q[c].unit, shift[c], m[c], l[c], f[c]);
            }
        }
        if (moved) {
#pragma unroll
            for (int c = 0; c < QT; ++c) rescale(c, f[c]);
        }
        if (plain) {
#pragma unroll
            for (int c = 0; c < QT; ++c)
                probabilities<true, FULL>(s[c], 0, ks, vs, q[c].unit, shift[c], m[c], l[c], pf[c]);
        } else {
#pragma unroll
            for (int c = 0; c < QT; ++c)
                probabilities<false, FULL>(s[c], vis[c], ks, vs, q[c].unit, shift[c], m[c], l[c], pf[c]);
        }
        __builtin_amdgcn_sched_barrier(0);             // the registers of s are free from here on
        fetch_k(i + 1, std::integral_constant<int, 1>{});
        __builtin_amdgcn_s_setprio(0);
        values(buf, pf);
        drop_unseen(token_of(i + 1));
        stage(buf ^ 1);
        ks = taken(ks_next), vs = taken(vs_next), have = have_next;
        turn(i + 2);
        fetch_v(i + 2);
        __syncthreads();
    }
#pragma unroll
    for (int c = 0; c < QT; ++c) {
        const float L = FULL ? l[c] : xor32_sum(xor16_sum(l[c]));
        const int rr = wave * 16 * QT + c * 16 + col;
        if (rr >= rt.rows) continue;
        if (R.used > 1) {
            float *pp = A.part + (((x * A.c.G + g) * A.splits + split) * kBlockRows<BF16> + rr) * (D + 4);
#pragma unroll
            for (int i = 0; i < DT; ++i)
                *reinterpret_cast<float4 *>(pp + i * 16 + grp * 4) = make_float4(acc[c][i][0], acc[c][i][1], acc[c][i][2], acc[c][i][3]);
            if (grp == 0) *reinterpret_cast<float2 *>(pp + D) = make_float2(m[c], L);
            continue;
        }
        const int64_t at = out_at(A, rt, g, rr, D) + grp * 4;
        const float inv = inverse(L);
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            const float o[4] = {acc[c][i][0], acc[c][i][1], acc[c][i][2], acc[c][i][3]};
            store_out4<BF16>(A.out, at + i * 16, o, inv);
        }
    }
}

// The splits of 16 rows of a row tile and head joined in order, a launch of its own.
template <int RT, int D, bool BF16>
__global__ __launch_bounds__(kThreads) void merge_kernel(const AttnArgs A) {
    const int64_t x = blockIdx.x / (unsigned)A.c.G;
    const int g = (int)(blockIdx.x % (unsigned)A.c.G);
    const RowTile rt = row_tile<RT>(A, x);
    if (rt.b < 0) return;
    const int p0 = rt.len - rt.n;
    const Tiles T = visible_tiles(A, p0 + rt.r0 / A.R, p0 + (rt.r0 + rt.rows - 1) / A.R);
    const int used = range_of(A, T.count, 0).used;
    if (used > 1) join_rows<RT, D, BF16, false>(A, rt, x, g, used, blockIdx.y * 16 + threadIdx.x / 16);
}

// How a call is split: row tiles of 16 or 128 (64 of fp32) rows, and each one's keys into ranges of `per` tiles, so that the
// workgroups fill the GPU.
struct Plan {
    int64_t tiles, splits, bytes;
    int rows, per;
};
constexpr int64_t kMaxTokens = 1 << 30;      // positions, rows and windows fit 32 bits with room for their differences
constexpr int kMaxSplits = 64;
Plan plan_of(int64_t N, int64_t B, int64_t H, int64_t G, bool bf16, int64_t max_new, int64_t max_keys, int64_t D,
             int64_t window, int64_t n_sink) {
    Plan p;
    const int64_t R = H / G;
    max_new = std::min(max_new, N);
    // tiles of 16 rows read K and V for each of them, large ones pass V through shared memory and are partly empty for few
    // rows (96 rows, bf16: 32 sequences of 4096 tokens and 2 kv heads 31 us in small tiles, 37 in large ones; 384 rows, 4
    // sequences of 9216 tokens and 8 kv heads: 125 and 84; 96 rows, 16 of those: 105 and 101, fp32 110 and 180)
    p.rows = max_new * R <= 96 ? 16 : bf16 ? kBlockRows<true> : kBlockRows<false>;
    p.tiles = N * R / p.rows + B;            // a sequence's n rows make at most n R / rows + 1 tiles
    int64_t keys = max_keys;
    if (window > 0 && window < kMaxTokens) keys = std::min(keys, window + std::min(n_sink, kMaxTokens) + max_new + 2 * kTile);
    const int64_t most = std::max<int64_t>(1, (keys + kTile - 1) / kTile);
    // as many tiles as the hint allows, of which p.tiles is the bound without it
    const int64_t groups = G * std::min(p.tiles, B * ((std::max<int64_t>(max_new, 1) * R + p.rows - 1) / p.rows));
    // 512 workgroups fill the GPU, two to a CU; where the sequences alone are as many, four times that for an even end
    // (32 windowed sequences of 2 kv heads: 384 workgroups 20.7 us, 512 20.0, 768 25.9; 64 of 8 kv heads and up to 16384
    // tokens: 1024 249 us, 2048 235, 4096 235)
    const int64_t want = std::max<int64_t>(1, (p.rows == 16 && groups >= 512 ? 2048 : 512) / groups);
    p.per = (int)std::max<int64_t>(kWaves, (most + std::min<int64_t>(want, kMaxSplits) - 1) / std::min<int64_t>(want, kMaxSplits));
    p.splits = (most + p.per - 1) / p.per;
    p.bytes = p.splits > 1 ? p.tiles * G * p.splits * p.rows * (D + 4) * 4 : 0;
    return p;
}

}  // namespace

extern "C" {

int64_t vgx_paged_attn_workspace_bytes(int64_t N, int64_t B, int64_t H, int64_t G, int64_t D, int64_t max_new,
                                       int64_t max_keys, int64_t window, int64_t n_sink) {
    if (N < 0 || B < 0 || H <= 0 || G <= 0 || max_new < 0 || max_keys < 0 || window < 0 || n_sink < 0) return VGX_E_SIZE;
    if (H % G || (D != 64 && D != 128)) return VGX_E_SHAPE;
    if (N > kMaxTokens || B > kMaxTokens || H > 65535 || max_keys > kMaxTokens || N * (H / G) > kMaxTokens) return VGX_E_LIMIT;
    if (N == 0 || B == 0) return 0;
    return std::max(plan_of(N, B, H, G, false, max_new, max_keys, D, window, n_sink).bytes,
                    plan_of(N, B, H, G, true, max_new, max_keys, D, window, n_sink).bytes);
}

int vgx_paged_attn(const vgx_paged_kv *kv, int64_t layer, int dtype, const void *q, int64_t ldq, void *out, int64_t ldo,
                   int64_t N, int64_t H, const int32_t *table, int64_t ldt, int64_t table_cols, const int32_t *lens,
                   const int32_t *q_start, int64_t B, int64_t max_new, int64_t max_keys, int64_t window, int64_t n_sink,
                   float scale, void *workspace, int64_t workspace_bytes, void *stream) {
    return vgx_paged_attn_tickets(kv, layer, dtype, q, ldq, out, ldo, N, H, table, ldt, table_cols, lens, q_start, B, max_new,
                                  max_keys, window, n_sink, scale, workspace, workspace_bytes, nullptr, 0, stream);
}

int vgx_paged_attn_tickets(const vgx_paged_kv *kv, int64_t layer, int dtype, const void *q, int64_t ldq, void *out,
                           int64_t ldo, int64_t N, int64_t H, const int32_t *table, int64_t ldt, int64_t table_cols,
                           const int32_t *lens, const int32_t *q_start, int64_t B, int64_t max_new, int64_t max_keys,
                           int64_t window, int64_t n_sink, float scale, void *workspace, int64_t workspace_bytes,
                           int32_t *tickets, int64_t n_tickets, void *stream) {
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
    const Plan p = plan_of(N, B, H, kv->G, dtype == VGX_BF16, max_new, max_keys, kv->D, window, n_sink);
    if (p.tiles * kv->G > kMaxGroups) return VGX_E_LIMIT;
    if (n_tickets < 0) return VGX_E_SIZE;
    if ((uintptr_t)tickets % 4) return VGX_E_ALIGN;
    // few rows a tile: a launch saved (one sequence of 2112 tokens 10.6 us, 14.0 with a launch that joins; 32 windowed ones
    // 19.1 and 21.6); more, and their states are too many for the one workgroup that would join them
    int32_t *mine = p.rows == 16 && n_tickets >= p.tiles * kv->G ? tickets : nullptr;
    // no position reaches kMaxTokens: a window of that many tokens is none
    const int win = window >= kMaxTokens ? 0 : (int)window, sink = (int)std::min(n_sink, kMaxTokens);
    const AttnArgs A{paged_layer(kv, layer), q, out, ldq, ldo, ldt, table, lens, q_start, static_cast<float *>(workspace),
                     scale, mine, (int)N, (int)B, (int)H, (int)(H / kv->G), (int)table_cols, win, sink, (int)p.splits, p.per};
    const int64_t tiles = q_start ? p.tiles : B * ((H / kv->G + p.rows - 1) / p.rows);
    const dim3 grid((unsigned)(tiles * kv->G), (unsigned)p.splits);
    const auto launch = [&](auto fm, auto dm, auto bf) -> int {
        const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, (hipStream_t)stream, A); };
        const bool one = kv->page >= kTile;
        if (p.rows == 16) one ? run(rows_kernel<fm.value, dm.value, bf.value, true>) : run(rows_kernel<fm.value, dm.value, bf.value, false>);
        else one ? run(block_kernel<fm.value, dm.value, bf.value, true>) : run(block_kernel<fm.value, dm.value, bf.value, false>);
        VGX_CHECK_LAUNCH();
        if (p.splits == 1 || mine) return VGX_OK;
        if (p.rows == 16)
            hipLaunchKernelGGL((merge_kernel<16, dm.value, bf.value>), dim3(grid.x, 1), dim3(kThreads), 0,
                               (hipStream_t)stream, A);
        else
            hipLaunchKernelGGL((merge_kernel<kBlockRows<bf.value>, dm.value, bf.value>), dim3(grid.x, p.rows / 16), dim3(kThreads),
                               0, (hipStream_t)stream, A);
        VGX_CHECK_LAUNCH();
        return VGX_OK;
    };
    return with_format(kv->fmt, kv->D, dtype == VGX_BF16, launch);
}

}  // extern "C"
