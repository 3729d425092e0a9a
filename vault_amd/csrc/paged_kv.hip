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
// codes are those of the definition and not of an order of fp32 operations.
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
    if (pos >= A.rope_rows) {
#pragma unroll
        for (int i = 0; i < 4; ++i) lo[i] = hi[i] = NAN;
        return;
    }
    float c[4], s[4];
    load4<false>(A.rope, pos * A.rope_ld + d, c);
    load4<false>(A.rope, pos * A.rope_ld + D / 2 + d, s);
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

template <int FMT, int D, bool BF16>
__global__ __launch_bounds__(kThreads) void append_kernel(const AppendArgs A) {
    __shared__ uint32_t red[4];
    extern __shared__ uint8_t tile[];            // V codes of the new tokens, [D][page]
    const int tid = threadIdx.x;
    if ((int64_t)blockIdx.x >= A.kv_groups) {
        // queries: thread = eight dims of one head of one row
        constexpr int T = D / 8;
        const int64_t u = ((int64_t)blockIdx.x - A.kv_groups) * kThreads + tid;
        const int64_t row = u / ((int64_t)A.H * T);
        if (row >= A.N) return;
        const int r = (int)(u - row * A.H * T), h = r / T, d = (r - h * T) * 4;
        int b = (int)row;
        int64_t pos = 0;
        if (A.q_start != nullptr) {
            int lo = 0, hi = A.B;                // the last b with q_start[b] <= row
            if (row < A.q_start[0] || row >= A.q_start[A.B]) return;
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
        float a[4], c[4], x[4], y[4];
        load4<BF16>(A.q, row * A.ldq + (int64_t)h * D + d, a);
        load4<BF16>(A.q, row * A.ldq + (int64_t)h * D + D / 2 + d, c);
        if (A.rope == nullptr) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = a[i], y[i] = c[i];
        } else if (pos >= A.rope_rows) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = y[i] = NAN;
        } else {
            float cs[4], sn[4];
            load4<false>(A.rope, pos * A.rope_ld + d, cs);
            load4<false>(A.rope, pos * A.rope_ld + D / 2 + d, sn);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = fmaf(a[i], cs[i], -(c[i] * sn[i]));
                y[i] = fmaf(c[i], cs[i], a[i] * sn[i]);
            }
        }
        store4<BF16>(A.q_out, row * A.ldqo + (int64_t)h * D + d, x);
        store4<BF16>(A.q_out, row * A.ldqo + (int64_t)h * D + D / 2 + d, y);
        return;
    }
    const int g = (int)(blockIdx.x % (unsigned)A.c.G), P = 1 << A.c.log_page;
    int64_t j = 0;
    const auto first_of = [&](int b, int &n) -> int64_t {      // first position at or above 0 and the tokens from it on
        const SeqRows r = seq_rows(A.q_start, b, A.N);
        const int64_t st = A.start[b];
        n = (int)max((int64_t)0, (int64_t)(r.hi - r.lo) - max((int64_t)0, -st));
        return max(st, (int64_t)0);
    };
    const int b = find_unit((int64_t)blockIdx.x / A.c.G, A.B, [&](int i) {
        int n;
        const int64_t p = first_of(i, n);
        return n <= 0 ? 0 : (int)(((p + n - 1) >> A.c.log_page) - (p >> A.c.log_page) + 1);
    }, j);
    if (b < 0) return;
    int n;
    const int64_t p0 = first_of(b, n);
    const int64_t col = (p0 >> A.c.log_page) + j;
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
    constexpr int T = D / 8;                                   // threads of one token
    const int t = tid / T, d = (tid - t * T) * 4;

    uint32_t kmax = 0, vmax = 0;
    for (int i = R.a + t; i < R.z; i += kThreads / T) {
        float x[4], y[4];
        const int64_t row = R.row + (i - R.a);
        rotated8<BF16, D>(A, row, R.pos0 + i, g, d, x, y);
#pragma unroll
        for (int e = 0; e < 4; ++e) kmax = max(kmax, max(abs_bits(x[e]), abs_bits(y[e])));
        load4<BF16>(A.v, row * A.ldv + (int64_t)g * D + d, x);
        load4<BF16>(A.v, row * A.ldv + (int64_t)g * D + D / 2 + d, y);
#pragma unroll
        for (int e = 0; e < 4; ++e) vmax = max(vmax, max(abs_bits(x[e]), abs_bits(y[e])));
    }
    const float was_k = A.c.ks[at], was_v = A.c.vs[at];
    kmax = block_max(kmax, red);
    vmax = block_max(vmax, red);
    const Scale sk = new_scale<FMT>(kmax, was_k, older), sv = new_scale<FMT>(vmax, was_v, older);
    if (tid == 0) {
        A.c.ks[at] = sk.now;
        A.c.vs[at] = sv.now;
    }
    const double ik = sk.now > 0.0f ? 1.0 / (double)sk.now : 0.0, iv = sv.now > 0.0f ? 1.0 / (double)sv.now : 0.0;
    for (int i = R.a + t; i < R.z; i += kThreads / T) {
        float x[4], y[4];
        const int64_t row = R.row + (i - R.a);
        rotated8<BF16, D>(A, row, R.pos0 + i, g, d, x, y);
        quotients(x, ik);
        quotients(y, ik);
        *reinterpret_cast<uint32_t *>(kp + (int64_t)i * D + d) = to_codes4<FMT>(x);
        *reinterpret_cast<uint32_t *>(kp + (int64_t)i * D + D / 2 + d) = to_codes4<FMT>(y);
        load4<BF16>(A.v, row * A.ldv + (int64_t)g * D + d, x);
        load4<BF16>(A.v, row * A.ldv + (int64_t)g * D + D / 2 + d, y);
        quotients(x, iv);
        quotients(y, iv);
        const uint32_t lo = to_codes4<FMT>(x), hi = to_codes4<FMT>(y);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            tile[(d + e) * P + i] = (uint8_t)(lo >> (8 * e));
            tile[(d + D / 2 + e) * P + i] = (uint8_t)(hi >> (8 * e));
        }
    }
    __syncthreads();
    // V rows are dims: whole 16-byte pieces of new tokens at once, the ends of the run byte by byte
    for (int u = tid; u < D * P / 16; u += kThreads) {
        const int dim = u / (P / 16), i0 = (u - dim * (P / 16)) * 16, o = dim * P + i0;
        if (i0 >= R.a && i0 + 16 <= R.z) {
            *reinterpret_cast<uint4 *>(vp + o) = *reinterpret_cast<const uint4 *>(tile + o);
        } else {
            for (int i = max(i0, R.a); i < min(i0 + 16, R.z); ++i) vp[dim * P + i] = tile[dim * P + i];
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

// One page of one (layer, sequence, head): K rows as they lie, V through shared memory.
template <int FMT, int D, bool BF16>
__global__ __launch_bounds__(kThreads) void read_kernel(const vgx_paged_kv kv, int log_page, const int32_t *table,
                                                        int64_t ldt, int cols, const int32_t *first,
                                                        const int32_t *lens, int n, void *k_out, void *v_out) {
    extern __shared__ uint8_t tile[];
    const int tid = threadIdx.x, P = 1 << log_page, G = (int)kv.G;
    const int g = (int)(blockIdx.y % (unsigned)G), b = (int)(blockIdx.y / (unsigned)G), layer = blockIdx.z;
    const int64_t f = first[b], col = (f >> log_page) + blockIdx.x, p0 = col << log_page;
    const int lo = (int)max((int64_t)0, f - p0), hi = (int)min((int64_t)P, f + n - p0);   // the page's tokens to write
    if (hi <= lo) return;
    const int page = col >= 0 && col < cols ? table[(int64_t)b * ldt + col] : -1;
    const bool have = page >= 0 && page < kv.n_pages;
    const int end = have ? (int)min((int64_t)hi, (int64_t)lens[b] - p0) : 0;               // tokens below it exist
    const int64_t at = (int64_t)max(page, 0) * G + g, bytes = layer * kv.layer_stride + at * (P * D);
    const int64_t row0 = (((int64_t)layer * (gridDim.y / (unsigned)G) + b) * G + g) * n + (p0 - f);
    float ks = 0.0f, vs = 0.0f;
    if (end > lo) {
        ks = kv.k_scale[layer * kv.scale_layer_stride + at];
        vs = kv.v_scale[layer * kv.scale_layer_stride + at];
        for (int u = tid; u < D * P / 16; u += kThreads)
            reinterpret_cast<uint4 *>(tile)[u] = reinterpret_cast<const uint4 *>(kv.v + bytes)[u];
    }
    __syncthreads();
    constexpr int T = D / 4;
    const int d = (tid % T) * 4;
    for (int i = lo + tid / T; i < hi; i += kThreads / T) {
        float x[4] = {0, 0, 0, 0}, y[4] = {0, 0, 0, 0};
        if (i < end) {
            code_values4<FMT>(*reinterpret_cast<const uint32_t *>(kv.k + bytes + (int64_t)i * D + d), x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] *= ks;
                y[e] = code_value<FMT>(tile[(d + e) * P + i]) * vs;
            }
        }
        store4<BF16>(k_out, (row0 + i) * D + d, x);
        store4<BF16>(v_out, (row0 + i) * D + d, y);
    }
}

// Workgroup (beam, layer); those of one extra layer write the tables.  Every wave works out the group's heirs from the
// parents: lane i is beam i.
__global__ __launch_bounds__(kThreads) void reorder_kernel(const vgx_paged_kv kv, int log_page, const int32_t *table,
                                                           int64_t ldt, int cols, const int32_t *lens,
                                                           const int32_t *parents, int K, int32_t *table_out,
                                                           int64_t ldt_out, int32_t *lens_out) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t base = (int64_t)(blockIdx.x / (unsigned)K) * K;
    const int me = (int)(blockIdx.x % (unsigned)K);
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
    for (int64_t u = tid; u < page_bytes / 16; u += kThreads) {
        kd[u] = ks[u];
        vd[u] = vs[u];
    }
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
    const int64_t q_threads = q ? N * H * (kv->D / 8) : 0;
    const int64_t groups = A.kv_groups + (q_threads + kThreads - 1) / kThreads;
    if (groups > 0x7FFFFFFF) return VGX_E_LIMIT;
    return with_format(kv->fmt, kv->D, dtype == VGX_BF16, [&](auto fm, auto dm, auto bf) -> int {
        hipLaunchKernelGGL((append_kernel<fm.value, dm.value, bf.value>), dim3((unsigned)groups), dim3(kThreads),
                           (size_t)(kv->D * kv->page), (hipStream_t)stream, A);
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
    if (n > 0x3FFFFFFF || B * kv->G > 65535) return VGX_E_LIMIT;
    const int log_page = paged_layer(kv, 0).log_page;
    const unsigned pages = (unsigned)((n + kv->page - 2) / kv->page + 1);
    return with_format(kv->fmt, kv->D, dtype == VGX_BF16, [&](auto fm, auto dm, auto bf) -> int {
        hipLaunchKernelGGL((read_kernel<fm.value, dm.value, bf.value>),
                           dim3(pages, (unsigned)(B * kv->G), (unsigned)kv->n_layers), dim3(kThreads),
                           (size_t)(kv->D * kv->page), (hipStream_t)stream, *kv, log_page, table, ldt, (int)table_cols,
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
    if (groups * K > 0x7FFFFFFF || kv->n_layers >= 65535) return VGX_E_LIMIT;
    const int log_page = paged_layer(kv, 0).log_page;
    hipLaunchKernelGGL(reorder_kernel, dim3((unsigned)(groups * K), (unsigned)kv->n_layers + 1), dim3(kThreads), 0,
                       (hipStream_t)stream, *kv, log_page, table, ldt, (int)table_cols, lens, parents, (int)K, table_out,
                       ldt_out, lens_out);
    VGX_CHECK_LAUNCH();
    return VGX_OK;
}

}  // extern "C"
