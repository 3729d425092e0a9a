// Writing, reading and reordering the paged 8-bit K/V cache (include/vault_amd.h: vgx_paged_append, vgx_paged_read,
// vgx_paged_reorder).
#include "paged.h"

using namespace vgx;

namespace {

constexpr int kThreads = 256;

template <bool BF16>
VGX_DEV void load4(const void *p, int64_t at, float (&x)[4]) {
    if constexpr (BF16) {
        const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + at);
        x[0] = bf16_bits_to_float(w.x);
        x[1] = __uint_as_float(w.x & 0xFFFF0000u);
        x[2] = bf16_bits_to_float(w.y);
        x[3] = __uint_as_float(w.y & 0xFFFF0000u);
    } else {
        const float4 f = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
        x[0] = f.x;
        x[1] = f.y;
        x[2] = f.z;
        x[3] = f.w;
    }
}

template <bool BF16>
VGX_DEV void store4(void *p, int64_t at, const float (&x)[4]) {
    if constexpr (BF16)
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + at) =
            make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
    else
        *reinterpret_cast<float4 *>(static_cast<float *>(p) + at) = make_float4(x[0], x[1], x[2], x[3]);
}

struct AppendArgs {
    PagedLayer c;
    const void *k, *v, *q;
    void *q_out;
    int64_t ldk, ldv, ldq, ldqo;
    const int32_t *table, *start, *q_start;
    int64_t ldt;
    const float *rope;
    int64_t rope_ld, rope_rows;
    int N, B, H, cols;
    int64_t kv_groups;          // workgroups that store K / V; the rest rotate q
};

// Tokens [a, z) of a page, the first of them row `row`, at position pos0 + a.
struct PageRun {
    int a, z;
    int64_t row, pos0;
};

// Four dims of a K row from d and four from d + D / 2, rotated: products and sum in fp64, rounded once, so that the
// codes are those of the definition and not of an order of fp32 operations.  (Queries are not rounded to codes: fp32.)
template <bool BF16, int D>
VGX_DEV void rotated8(const AppendArgs &A, int64_t row, int64_t pos, int g, int d, float (&lo)[4], float (&hi)[4]) {
    float a[4], b[4];
    load4<BF16>(A.k, row * A.ldk + (int64_t)g * D + d, a);
    load4<BF16>(A.k, row * A.ldk + (int64_t)g * D + D / 2 + d, b);
    if (A.rope == nullptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i) lo[i] = a[i], hi[i] = b[i];
        return;
    }
    const bool known = pos < A.rope_rows;
    float c[4] = {NAN, NAN, NAN, NAN}, s[4] = {NAN, NAN, NAN, NAN};
    if (known) {
        load4<false>(A.rope, pos * A.rope_ld + d, c);
        load4<false>(A.rope, pos * A.rope_ld + D / 2 + d, s);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo[i] = (float)((double)a[i] * (double)c[i] - (double)b[i] * (double)s[i]);
        hi[i] = (float)((double)b[i] * (double)c[i] + (double)a[i] * (double)s[i]);
    }
}

VGX_DEV uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// The largest of a workgroup's values, in every thread.
VGX_DEV uint32_t block_max(uint32_t v, uint32_t *red) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off, kWave));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = max(max(red[0], red[1]), max(red[2], red[3]));
    __syncthreads();
    return v;
}

struct Scale {
    float now, old;
    bool grown;                 // older codes have to be rounded again
};
// The scale of a page and head whose new tokens have the largest magnitude `bits`.
template <int FMT>
VGX_DEV Scale new_scale(uint32_t bits, float was, bool older) {
    Scale s{__fdiv_rn(__uint_as_float(bits), FMT == VGX_I8 ? kQMaxI8 : kQMaxE4M3), was, false};
    if (bits >= 0x7F800000u || (older && was != was)) {
        s.now = NAN;
    } else if (older) {
        s.grown = s.now > was;
        s.now = fmaxf(s.now, was);
    }
    return s;
}

// fp32(x / scale) of four values; zeros for the scales that no value can be divided by.  1 / scale in fp64 makes the
// product differ from the quotient by 2^-52 at most, which the rounding to fp32 takes away.
VGX_DEV void quotients(float (&x)[4], double inv) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = inv == 0.0 ? 0.0f : (float)((double)x[i] * inv);
}

template <int FMT>
VGX_DEV uint32_t again4(uint32_t w, const Scale &s) {
    float c[4];
    code_values4<FMT>(w, c);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = (float)((double)c[i] * (double)s.old / (double)s.now);
    return to_codes4<FMT>(c);
}

// w[t] holds byte d of token t in its byte d; afterwards w[d] holds byte d of token t in its byte t.
VGX_DEV void transpose_bytes(uint32_t (&w)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// Queries: a wave takes one row; a lane has 8 dims of the lower half of a head and their partners of the upper one, and
// goes through the heads with its piece of the rotation in registers.
template <int D, bool BF16>
VGX_DEV void rotate_query(const AppendArgs &A, int64_t row) {
    constexpr int T = D / 16, HEADS = 64 / T;
    const int lane = threadIdx.x & 63, d = (lane % T) * 8;
    int b = (int)row;
    int64_t pos = 0;
    if (A.q_start != nullptr) {
        if (row < A.q_start[0] || row >= A.q_start[A.B]) return;
        int lo = 0, hi = A.B;                    // the last b with q_start[b] <= row
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (A.q_start[mid] <= row) lo = mid;
            else hi = mid;
        }
        b = lo;
        pos = row - A.q_start[b];
    }
    pos += A.start[b];
    if (pos < 0) return;
    float cs[2][4], sn[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cs[j][i] = A.rope == nullptr ? 1.0f : NAN;
            sn[j][i] = A.rope == nullptr ? 0.0f : NAN;
        }
    if (A.rope != nullptr && pos < A.rope_rows) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            load4<false>(A.rope, pos * A.rope_ld + d + 4 * j, cs[j]);
            load4<false>(A.rope, pos * A.rope_ld + D / 2 + d + 4 * j, sn[j]);
        }
    }
#pragma unroll 2
    for (int h = lane / T; h < A.H; h += HEADS) {
        const int64_t at = row * A.ldq + (int64_t)h * D + d, to = row * A.ldqo + (int64_t)h * D + d;
        float a[2][4], c[2][4], x[2][4], y[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            load4<BF16>(A.q, at + 4 * j, a[j]);
            load4<BF16>(A.q, at + D / 2 + 4 * j, c[j]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[j][i] = A.rope == nullptr ? a[j][i] : fmaf(a[j][i], cs[j][i], -(c[j][i] * sn[j][i]));
                y[j][i] = A.rope == nullptr ? c[j][i] : fmaf(c[j][i], cs[j][i], a[j][i] * sn[j][i]);
            }
            store4<BF16>(A.q_out, to + 4 * j, x[j]);
            store4<BF16>(A.q_out, to + D / 2 + 4 * j, y[j]);
        }
    }
}

// A workgroup stores the new tokens of one page and head: a thread has four tokens and, of each, four dims of the lower
// half and their partners of the upper one.  ONCE: the page's tokens fit the workgroup's registers (64 of 128 dims), which
// then hold them between the search for the largest magnitude and the rounding; otherwise they are read again.  V's codes
// are turned from tokens to dims in registers, four by four, and pass through shared memory (rows of page + 4 bytes, so
// that the dims of a wave's words lie in different banks) on their way to whole 16-byte pieces.  What bounds it is the
// rotated queries' traffic: 13057 tokens of 32 / 8 heads in bf16 37 us; 63 when every thread took two loads of its rotation
// for 8 values of q and the tokens were read twice.
template <int FMT, int D, bool BF16, bool ONCE>
__global__ __launch_bounds__(kThreads) void append_kernel(const AppendArgs A) {
    __shared__ uint32_t red[4];
    extern __shared__ uint8_t tile[];
    const int tid = threadIdx.x;
    if ((int64_t)blockIdx.x >= A.kv_groups) {
        const int64_t row = ((int64_t)blockIdx.x - A.kv_groups) * (kThreads / 64) + (tid >> 6);
        if (row < A.N) rotate_query<D, BF16>(A, row);
        return;
    }
    const int g = (int)(blockIdx.x % (unsigned)A.c.G), P = 1 << A.c.log_page, S = P + 4;
    int64_t j = 0;
    const auto first_of = [&](int b, int &n) -> int64_t {      // first position at or above 0 and the tokens from it on
        const SeqRows r = seq_rows(A.q_start, b, A.N);
        const int64_t st = A.start[b];
        n = (int)max((int64_t)0, (int64_t)(r.hi - r.lo) - max((int64_t)0, -st));
        return max(st, (int64_t)0);
    };
    int b = (int)(blockIdx.x / (unsigned)A.c.G);
    if (A.q_start != nullptr) {
        b = find_unit(b, A.B, [&](int i) {
            int n;
            const int64_t p = first_of(i, n);
            return n <= 0 ? 0 : (int)(((p + n - 1) >> A.c.log_page) - (p >> A.c.log_page) + 1);
        }, j);
        b = __builtin_amdgcn_readfirstlane(b);
        if (b < 0) return;
    }
    int n;
    const int64_t p0 = first_of(b, n);
    if (n <= 0) return;
    const int64_t col = (p0 >> A.c.log_page) + __builtin_amdgcn_readfirstlane((int)j);
    if (col >= A.cols) return;
    const int page = A.table[(int64_t)b * A.ldt + col];
    if (page < 0 || page >= A.c.n_pages) return;
    PageRun R;
    R.pos0 = col << A.c.log_page;
    R.a = (int)max((int64_t)0, p0 - R.pos0);
    R.z = (int)min((int64_t)P, p0 + n - R.pos0);
    R.row = seq_rows(A.q_start, b, A.N).lo + (R.pos0 + R.a - A.start[b]);
    const int64_t at = (int64_t)page * A.c.G + g, bytes = at * A.c.head_bytes;
    uint8_t *kp = A.c.k + bytes, *vp = A.c.v + bytes;
    const bool older = R.a > 0;
    const float was_k = A.c.ks[at], was_v = A.c.vs[at];
    constexpr int T = D / 8, PER = 4 * kThreads / T;           // threads of a token, tokens of the workgroup
    const int t4 = (tid / T) * 4, d = (tid % T) * 4;

    float kx[4][2][4], vx[4][2][4];
    const auto load = [&](int base) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int i = base + t4 + t;
#pragma unroll
            for (int e = 0; e < 4; ++e) kx[t][0][e] = kx[t][1][e] = vx[t][0][e] = vx[t][1][e] = 0.0f;
            if (i < R.a || i >= R.z) continue;
            const int64_t row = R.row + (i - R.a);
            rotated8<BF16, D>(A, row, R.pos0 + i, g, d, kx[t][0], kx[t][1]);
            load4<BF16>(A.v, row * A.ldv + (int64_t)g * D + d, vx[t][0]);
            load4<BF16>(A.v, row * A.ldv + (int64_t)g * D + D / 2 + d, vx[t][1]);
        }
    };
    uint32_t kmax = 0, vmax = 0;
    for (int base = R.a & ~3; base < R.z; base += PER) {
        load(base);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    kmax = max(kmax, abs_bits(kx[t][h][e]));
                    vmax = max(vmax, abs_bits(vx[t][h][e]));
                }
    }
    kmax = block_max(kmax, red);
    vmax = block_max(vmax, red);
    const Scale sk = new_scale<FMT>(kmax, was_k, older), sv = new_scale<FMT>(vmax, was_v, older);
    if (tid == 0) {
        A.c.ks[at] = sk.now;
        A.c.vs[at] = sv.now;
    }
    const double ik = sk.now > 0.0f ? 1.0 / (double)sk.now : 0.0, iv = sv.now > 0.0f ? 1.0 / (double)sv.now : 0.0;
    for (int base = R.a & ~3; base < R.z; base += PER) {
        if (!ONCE) load(base);
        if (base + t4 >= R.z) continue;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t w[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int i = base + t4 + t;
                quotients(kx[t][h], ik);
                if (i >= R.a && i < R.z)
                    *reinterpret_cast<uint32_t *>(kp + (int64_t)i * D + h * (D / 2) + d) = to_codes4<FMT>(kx[t][h]);
                quotients(vx[t][h], iv);
                w[t] = to_codes4<FMT>(vx[t][h]);
            }
            transpose_bytes(w);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<uint32_t *>(tile + (h * (D / 2) + d + e) * S + base + t4) = w[e];
        }
    }
    __syncthreads();
    // V rows are dims: whole 16-byte pieces of new tokens at once, the ends of the run byte by byte
    const int c0 = R.a / 16, cn = (R.z + 15) / 16 - c0;        // the 16-token pieces that the run touches
    for (int u = tid; u < D * cn; u += kThreads) {
        const int dim = u / cn, i0 = (c0 + u - dim * cn) * 16;
        const uint8_t *src = tile + dim * S + i0;
        uint8_t *dst = vp + dim * P + i0;
        if (i0 >= R.a && i0 + 16 <= R.z) {
            const uint32_t *w = reinterpret_cast<const uint32_t *>(src);
            *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            for (int i = max(i0, R.a) - i0; i < min(i0 + 16, R.z) - i0; ++i) dst[i] = src[i];
        }
    }
    if (sk.grown)
        for (int u = tid; u < R.a * D / 4; u += kThreads) {
            uint32_t *w = reinterpret_cast<uint32_t *>(kp) + u;
            *w = again4<FMT>(*w, sk);
        }
    if (sv.grown)
        for (int u = tid; u < D * R.a; u += kThreads) {
            uint8_t *c = vp + (u / R.a) * P + u % R.a;
            *c = (uint8_t)again4<FMT>(*c, sv);
        }
}

// One page of one (layer, sequence, head).  A thread has four tokens of four dims: K's words lie that way, V's are words
// of four tokens and pass through shared memory (rows of page + 4 bytes, so that the dims of a wave lie in different
// banks).  The grid has a page more than a run of whole pages needs, and workgroups go to the dies and
// their engines in turn: with the pages turned by a hash, those without work do not all meet on the same ones (one page of
// 128 tokens of 128 sequences, 2 heads and 28 layers in fp32, 1.2 GB: 244 us, 368 without, 337 turned every four heads).
template <int FMT, int D, bool BF16>
__global__ __launch_bounds__(kThreads) void read_kernel(const vgx_paged_kv kv, int log_page, const int32_t *table,
                                                        int64_t ldt, int cols, const int32_t *first,
                                                        const int32_t *lens, int n, void *k_out, void *v_out) {
    extern __shared__ uint8_t tile[];
    const int tid = threadIdx.x, P = 1 << log_page, S = P + 4, G = (int)kv.G;
    const int g = (int)(blockIdx.y % (unsigned)G), b = (int)(blockIdx.y / (unsigned)G), layer = blockIdx.z;
    const unsigned turned = (blockIdx.x + (((blockIdx.y + blockIdx.z * gridDim.y) * 0x9E3779B1u) >> 16)) % gridDim.x;
    const int64_t f = first[b], len = lens[b], col = (f >> log_page) + turned, p0 = col << log_page;
    const int lo = (int)max((int64_t)0, f - p0), hi = (int)min((int64_t)P, f + n - p0);   // the page's tokens to write
    if (hi <= lo) return;
    const int page = col >= 0 && col < cols ? table[(int64_t)b * ldt + col] : -1;
    const bool have = page >= 0 && page < kv.n_pages;
    const int end = have ? (int)max((int64_t)0, min((int64_t)hi, len - p0)) : 0;                            // tokens below it exist
    const int64_t at = (int64_t)max(page, 0) * G + g, bytes = layer * kv.layer_stride + at * (P * D);
    const int64_t row0 = (((int64_t)layer * (gridDim.y / (unsigned)G) + b) * G + g) * n + (p0 - f);
    float ks = 0.0f, vs = 0.0f;
    if (end > lo) {
        ks = kv.k_scale[layer * kv.scale_layer_stride + at];
        vs = kv.v_scale[layer * kv.scale_layer_stride + at];
        const int c0 = lo / 16, cn = (end + 15) / 16 - c0;     // the 16-token pieces asked for
        for (int u = tid; u < D * cn; u += kThreads) {
            const int dim = u / cn, i0 = (c0 + u - dim * cn) * 16;
            const uint4 w = *reinterpret_cast<const uint4 *>(kv.v + bytes + dim * P + i0);
            uint32_t *t = reinterpret_cast<uint32_t *>(tile + dim * S + i0);
            t[0] = w.x, t[1] = w.y, t[2] = w.z, t[3] = w.w;
        }
    }
    __syncthreads();
    constexpr int T = D / 4;
    const int d = (tid % T) * 4;
    for (int i0 = (lo & ~3) + tid / T * 4; i0 < hi; i0 += kThreads / T * 4) {
        uint32_t kw[4], vw[4];
#pragma unroll
        for (int t = 0; t < 4; ++t)                            // the page's tokens, whether asked for or not
            kw[t] = i0 < end ? *reinterpret_cast<const uint32_t *>(kv.k + bytes + (int64_t)(i0 + t) * D + d) : 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) vw[e] = i0 < end ? *reinterpret_cast<const uint32_t *>(tile + (d + e) * S + i0) : 0u;
        transpose_bytes(vw);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int i = i0 + t;
            if (i < lo || i >= hi) continue;
            float x[4] = {0, 0, 0, 0}, y[4] = {0, 0, 0, 0};
            if (i < end) {
                code_values4<FMT>(kw[t], x);
                code_values4<FMT>(vw[t], y);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] *= ks, y[e] *= vs;
            }
            store4<BF16>(k_out, (row0 + i) * D + d, x);
            store4<BF16>(v_out, (row0 + i) * D + d, y);
        }
    }
}

// Workgroup (beam, layer, slice of the page); those of one extra layer write the tables.  Every wave works out the group's
// heirs from the parents: lane i is beam i.  Beams turn with the layer: the first beams of a group seldom copy, and a beam
// of all layers would go to one die (16 groups of 8 beams, 28 layers, pages of 128 tokens: 40 us, 55 without).
__global__ __launch_bounds__(kThreads) void reorder_kernel(const vgx_paged_kv kv, int log_page, const int32_t *table,
                                                           int64_t ldt, int cols, const int32_t *lens,
                                                           const int32_t *parents, int K, int32_t *table_out,
                                                           int64_t ldt_out, int32_t *lens_out) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t base = (int64_t)(blockIdx.x / (unsigned)K) * K;
    const int me = (int)((blockIdx.x + blockIdx.y) % (unsigned)K);
    int par = lane < K ? parents[base + lane] : -1;
    if (lane < K && (par < 0 || par >= K)) par = lane;
    // heirs: the first child of each parent; dead: beams without children
    uint64_t heirs = 0, seen = 0;
    for (int i = 0; i < K; ++i) {
        const int p = __shfl(par, i, kWave);
        if (!(seen >> p & 1)) heirs |= 1ull << i;
        seen |= 1ull << p;
    }
    const uint64_t all = K == 64 ? ~0ull : (1ull << K) - 1, dead = all & ~seen;
    const int p = __shfl(par, me, kWave);
    int giver = p;
    if (!(heirs >> me & 1)) {
        int rank = __popcll(all & ~heirs & ((1ull << me) - 1));
        uint64_t m = dead;
        while (rank-- > 0) m &= m - 1;
        giver = __ffsll((unsigned long long)m) - 1;
    }
    const int64_t row = base + me, prow = base + p, grow = base + giver;
    const int len = max(lens[prow], 0);
    const int64_t at = (int64_t)len >> log_page, give_at = (int64_t)max(lens[grow], 0) >> log_page;
    const int dst = give_at < cols ? table[grow * ldt + give_at] : -1;
    if (blockIdx.y == kv.n_layers) {
        if (blockIdx.z != 0) return;
        const int64_t mine = (int64_t)max(lens[row], 0) >> log_page;
        for (int64_t j = tid; j < cols; j += kThreads)
            table_out[row * ldt_out + j] = j < at ? table[prow * ldt + j]
                                           : j == at ? dst
                                           : j > mine ? table[row * ldt + j] : -1;
        if (tid == 0) lens_out[row] = lens[prow];
        return;
    }
    if (giver == p) return;
    const int src = at < cols ? table[prow * ldt + at] : -1;
    if (src < 0 || src >= kv.n_pages || dst < 0 || dst >= kv.n_pages || (len & ((1 << log_page) - 1)) == 0) return;
    const int64_t page_bytes = kv.G * kv.page * kv.D, lo = (int64_t)blockIdx.y * kv.layer_stride;
    const int64_t s0 = (int64_t)blockIdx.y * kv.scale_layer_stride;
    const auto *ks = reinterpret_cast<const uint4 *>(kv.k + lo + src * page_bytes);
    const auto *vs = reinterpret_cast<const uint4 *>(kv.v + lo + src * page_bytes);
    auto *kd = reinterpret_cast<uint4 *>(kv.k + lo + dst * page_bytes);
    auto *vd = reinterpret_cast<uint4 *>(kv.v + lo + dst * page_bytes);
    const int64_t pieces = page_bytes / 16, per = (pieces + gridDim.z - 1) / gridDim.z;
    const int64_t u1 = min(pieces, (blockIdx.z + 1) * per);
#pragma unroll 2
    for (int64_t u = blockIdx.z * per + tid; u < u1; u += kThreads) {
        const uint4 a = ks[u], c = vs[u];
        kd[u] = a;
        vd[u] = c;
    }
    if (blockIdx.z != 0) return;
    for (int64_t g = tid; g < kv.G; g += kThreads) {
        kv.k_scale[s0 + dst * kv.G + g] = kv.k_scale[s0 + src * kv.G + g];
        kv.v_scale[s0 + dst * kv.G + g] = kv.v_scale[s0 + src * kv.G + g];
    }
}

int check_rows(const void *p, int64_t ld, int64_t need, int64_t es) {
    if (!p) return VGX_E_ARG;
    if (ld < need) return VGX_E_SIZE;
    if ((uintptr_t)p % 16 || ld * es % 16) return VGX_E_ALIGN;
    return VGX_OK;
}

}  // namespace

extern "C" {

int vgx_paged_append(const vgx_paged_kv *kv, int64_t layer, int dtype, const void *k, int64_t ldk, const void *v,
                     int64_t ldv, int64_t N, const int32_t *table, int64_t ldt, int64_t table_cols, const int32_t *start,
                     const int32_t *q_start, int64_t B, const float *rope, int64_t rope_ld, int64_t rope_rows,
                     const void *q, int64_t ldq, void *q_out, int64_t ldqo, int64_t H, void *stream) {
    if (const int rc = check_paged(kv, layer)) return rc;
    if (dtype != VGX_F32 && dtype != VGX_BF16) return VGX_E_DTYPE;
    if (N < 0 || B < 0 || (!q_start && N != B)) return VGX_E_SIZE;
    if (N == 0 || B == 0) return VGX_OK;
    if (N > 0x7FFFFFFF || B >= 0x7FFFFFFF) return VGX_E_LIMIT;
    if (const int rc = check_table(table, ldt, table_cols)) return rc;
    if (!start) return VGX_E_ARG;
    const int64_t es = dtype == VGX_F32 ? 4 : 2;
    if (const int rc = check_rows(k, ldk, kv->G * kv->D, es)) return rc;
    if (const int rc = check_rows(v, ldv, kv->G * kv->D, es)) return rc;
    if (rope && (rope_ld < kv->D || rope_rows < 0)) return VGX_E_SIZE;
    if (rope && ((uintptr_t)rope % 16 || rope_ld % 4)) return VGX_E_ALIGN;
    if (q) {
        if (H <= 0) return VGX_E_SIZE;
        if (H > 65535) return VGX_E_LIMIT;
        if (const int rc = check_rows(q, ldq, H * kv->D, es)) return rc;
        if (const int rc = check_rows(q_out, ldqo, H * kv->D, es)) return rc;
    }
    AppendArgs A{paged_layer(kv, layer), k, v, q, q_out, ldk, ldv, ldq, ldqo, table, start, q_start, ldt, rope, rope_ld,
                 rope_rows, (int)N, (int)B, (int)H, (int)table_cols, 0};
    // a sequence's n rows touch at most n / page + 2 pages, and no more than n
    const int64_t slots = q_start ? std::min(N, N / kv->page + 2 * B) : B;
    A.kv_groups = slots * kv->G;
    const int64_t groups = A.kv_groups + (q ? (N + 3) / 4 : 0);
    if (groups > kMaxGroups) return VGX_E_LIMIT;
    return with_format(kv->fmt, kv->D, dtype == VGX_BF16, [&](auto fm, auto dm, auto bf) -> int {
        const auto run = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(kThreads), (size_t)(kv->D * (kv->page + 4)),
                               (hipStream_t)stream, A);
        };
        // tokens that a workgroup holds at once (13057 tokens in pages of 64, read back: 62 us, 81 when they are read twice)
        if (kv->page <= 4 * kThreads / (dm.value / 8)) run(append_kernel<fm.value, dm.value, bf.value, true>);
        else run(append_kernel<fm.value, dm.value, bf.value, false>);
        VGX_CHECK_LAUNCH();
        return VGX_OK;
    });
}

int vgx_paged_read(const vgx_paged_kv *kv, int dtype, const int32_t *table, int64_t ldt, int64_t table_cols,
                   const int32_t *first, const int32_t *lens, int64_t B, int64_t n, void *k_out, void *v_out,
                   void *stream) {
    if (const int rc = check_paged(kv, 0)) return rc;
    if (dtype != VGX_F32 && dtype != VGX_BF16) return VGX_E_DTYPE;
    if (B < 0 || n < 0) return VGX_E_SIZE;
    if (B == 0 || n == 0) return VGX_OK;
    if (const int rc = check_table(table, ldt, table_cols)) return rc;
    if (!first || !lens || !k_out || !v_out) return VGX_E_ARG;
    if (((uintptr_t)k_out | (uintptr_t)v_out) % 16) return VGX_E_ALIGN;
    const int64_t pages = (std::min<int64_t>(n, 1 << 30) + kv->page - 2) / kv->page + 1;
    if (n > 0x3FFFFFFF || pages > kMaxGroups || B > 65535 || B * kv->G > 65535) return VGX_E_LIMIT;
    const int log_page = paged_layer(kv, 0).log_page;
    return with_format(kv->fmt, kv->D, dtype == VGX_BF16, [&](auto fm, auto dm, auto bf) -> int {
        hipLaunchKernelGGL((read_kernel<fm.value, dm.value, bf.value>),
                           dim3((unsigned)pages, (unsigned)(B * kv->G), (unsigned)kv->n_layers), dim3(kThreads),
                           (size_t)(kv->D * (kv->page + 4)), (hipStream_t)stream, *kv, log_page, table, ldt, (int)table_cols,
                           first, lens, (int)n, k_out, v_out);
        VGX_CHECK_LAUNCH();
        return VGX_OK;
    });
}

int vgx_paged_reorder(const vgx_paged_kv *kv, const int32_t *table, int64_t ldt, int64_t table_cols, const int32_t *lens,
                      const int32_t *parents, int64_t groups, int64_t K, int32_t *table_out, int64_t ldt_out,
                      int32_t *lens_out, void *stream) {
    if (const int rc = check_paged(kv, 0)) return rc;
    if (groups < 0 || K <= 0) return VGX_E_SIZE;
    if (K > 64) return VGX_E_LIMIT;
    if (groups == 0) return VGX_OK;
    if (const int rc = check_table(table, ldt, table_cols)) return rc;
    if (const int rc = check_table(table_out, ldt_out, table_cols)) return rc;
    if (!lens || !parents || !lens_out || table_out == table || lens_out == lens) return VGX_E_ARG;
    if (groups > kMaxGroups || groups * K > kMaxGroups || kv->n_layers >= 65535) return VGX_E_LIMIT;
    const int log_page = paged_layer(kv, 0).log_page;
    // 16 KB of K and of V to a workgroup (16 groups of 8 beams, read back: 256 us, 260 in one slice, 268 with 4 KB)
    const unsigned slices = (unsigned)std::min<int64_t>(16, std::max<int64_t>(1, kv->G * kv->page * kv->D / 16384));
    hipLaunchKernelGGL(reorder_kernel, dim3((unsigned)(groups * K), (unsigned)kv->n_layers + 1, slices), dim3(kThreads), 0,
                       (hipStream_t)stream, *kv, log_page, table, ldt, (int)table_cols, lens, parents, (int)K, table_out,
                       ldt_out, lens_out);
    VGX_CHECK_LAUNCH();
    return VGX_OK;
}

}  // extern "C"
