// Beam search's choice of continuations (include/vault_amd.h: vgx_beam_select).
//
// The order of a row's candidates by total = score + x - log sum exp x is their order by x, so one pass over the logits
// serves both: workgroup (row, chunk) keeps its values in registers, sums their exponentials under its own maximum and
// writes its K largest as sorted 64-bit keys (value, then the smaller index).  A second launch, one workgroup per group,
// joins the sums, turns keys into totals (fp64) and picks: of the K * chunks sorted lists only the K with the best heads
// can hold one of the K best totals, since each of those heads beats everything in the other lists.
//
// The K largest of a wave's values: the K-th largest of its 64 lanes' maxima is a bound that at least K values reach;
// whatever reaches it (about K values for small K, whatever the distribution of the values, as long as their order is not
// arranged by lane) is compacted into shared memory and ranked there.
#include "common.h"

#include <algorithm>

using namespace vgx;

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxK = 64;
constexpr int kCap = 512;                    // values that a wave compacts; more take the slow way
constexpr int64_t kMaxV = 1 << 19;         // K chunks of heads fit shared memory
constexpr int kJoinThreads = 1024;

// Order-preserving map of a logit, NaN and -inf (never candidates) to 0.
VGX_DEV uint32_t ordered(float v) {
    if (!(v > -INFINITY)) return 0u;
    const uint32_t u = v == 0.0f ? 0u : __float_as_uint(v);   // -0 ranks as +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
VGX_DEV float value_of(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o); }
VGX_DEV uint64_t key_of(uint32_t o, uint32_t i) { return o ? ((uint64_t)o << 32) | (0xFFFFFFFFu - i) : 0ull; }

VGX_DEV uint64_t wave_max64(uint64_t k) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const uint64_t o = ((uint64_t)(unsigned)__shfl_xor((int)(k >> 32), off, kWave) << 32) |
                           (uint64_t)(unsigned)__shfl_xor((int)k, off, kWave);
        k = o > k ? o : k;
    }
    return k;
}

// Shared-memory bitonic sort, n a power of two: before(i, j) says that element i belongs before j, swap(i, j) exchanges.
template <int THREADS, class Before, class Swap>
VGX_DEV void sort_shared(int n, Before before, Swap swap) {
    for (int size = 2; size <= n; size <<= 1)
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            for (int i = threadIdx.x; i < n / 2; i += THREADS) {
                const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
                const bool up = (lo & size) == 0;
                if (up ? before(hi, lo) : before(lo, hi)) swap(lo, hi);
            }
            __syncthreads();
        }
}

struct F4 {
    float v[4];
} __attribute__((packed, aligned(4)));

// VPT values per thread; lists[row][chunk][K] keys, sums[row][chunk] = (maximum, sum of exp(x - maximum)).
template <int VPT>
__global__ __launch_bounds__(kThreads) void chunk_kernel(const float *__restrict__ x, int64_t ld, int V, int K,
                                                         const uint8_t *__restrict__ done, uint64_t *__restrict__ lists,
                                                         float2 *__restrict__ sums) {
    __shared__ uint64_t keys[kWaves * kCap];
    __shared__ float red[kWaves];
    __shared__ int count[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.y;
    if (done != nullptr && done[row] != 0) return;
    const int base = (int)blockIdx.x * kThreads * VPT;
    const float *r = x + row * ld;
    float v[VPT];
#pragma unroll
    for (int j = 0; j < VPT / 4; ++j) {
        const int i = base + (j * kThreads + tid) * 4;
        if (i + 4 <= V) {
            const F4 f = *reinterpret_cast<const F4 *>(r + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * j + e] = f.v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * j + e] = i + e < V ? r[i + e] : -INFINITY;
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < VPT; ++j) top = fmaxf(top, v[j]);
    const float wtop = wave_max(top);
    if (lane == 0) red[wave] = wtop;
    __syncthreads();
    const float m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float s = 0.0f;
    if (m > -INFINITY) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) s += __expf(v[j] - m);
    } else {
#pragma unroll
        for (int j = 0; j < VPT; ++j) s += v[j] == v[j] ? 0.0f : v[j];     // a NaN among nothing else stays one
    }
    s = wave_sum(s);
    __syncthreads();
    if (lane == 0) red[wave] = s;

    // the K-th largest of the lanes' maxima, bit by bit; 15 bits of the mantissa will do (a value more may reach the bound)
    const uint32_t mine = ordered(top);
    uint32_t bound = 0;
#pragma unroll
    for (int bit = 31; bit >= 8; --bit) {
        const uint32_t t = bound | (1u << bit);
        if (__popcll(__ballot(mine >= t)) >= K) bound = t;
    }
    bound = max(bound, 1u);                                                 // -inf and NaN are no candidates
    int n = 0;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const uint32_t o = ordered(v[j]);
        const uint64_t in = __ballot(o >= bound);
        if (in == 0) continue;
        const int at = n + __popcll(in & ((1ull << lane) - 1));
        const uint32_t i = (uint32_t)(base + ((j >> 2) * kThreads + tid) * 4 + (j & 3));
        if (o >= bound && at < kCap) keys[wave * kCap + at] = key_of(o, i);
        n += __popcll(in);
    }
    if (n > kCap) {
        // many equal values, or large ones gathered in few lanes: the K largest one after the other
        uint64_t last = ~0ull;
        n = 0;
        for (; n < K; ++n) {
            uint64_t best = 0;
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const uint32_t i = (uint32_t)(base + ((j >> 2) * kThreads + tid) * 4 + (j & 3));
                const uint64_t k = key_of(ordered(v[j]), i);
                if (k < last && k > best) best = k;
            }
            best = wave_max64(best);
            if (best == 0) break;
            if (lane == 0) keys[wave * kCap + n] = best;
            last = best;
        }
    }
    if (lane == 0) count[wave] = n;
    __syncthreads();
    const int64_t chunk = row * gridDim.x + blockIdx.x;
    if (tid == 0) sums[chunk] = make_float2(m, red[0] + red[1] + red[2] + red[3]);
    uint64_t *out = lists + chunk * K;
    // the four waves' keys end to end, ranked by counting
    int total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += count[w];
    if (total <= kThreads) {
        uint64_t k = 0;
        int w = 0, at = tid;
        while (w < kWaves && at >= count[w]) at -= count[w++];
        if (w < kWaves) k = keys[w * kCap + at];
        int rank = 0;
        for (int u = 0; u < kWaves; ++u) {
            const int m = count[u];
#pragma unroll 8
            for (int i = 0; i < m; ++i) rank += keys[u * kCap + i] > k;
        }
        if (k != 0 && rank < K) out[rank] = k;
        if (tid < K && tid >= total) out[tid] = 0;
        return;
    }
    for (int i = lane; i < kCap; i += 64)
        if (i >= n) keys[wave * kCap + i] = 0;
    __syncthreads();
    sort_shared<kThreads>(kWaves * kCap, [&](int i, int j) { return keys[i] > keys[j]; },
                          [&](int i, int j) {
                              const uint64_t t = keys[i];
                              keys[i] = keys[j];
                              keys[j] = t;
                          });
    if (tid < K) out[tid] = keys[tid];
}

// Order-preserving map of a total; 0 for what is no candidate.
VGX_DEV uint64_t ordered64(double t) {
    if (!(t > -INFINITY)) return 0ull;
    const uint64_t u = t == 0.0 ? 0ull : (uint64_t)__double_as_longlong(t);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
VGX_DEV double total_of(uint64_t o) {
    return __longlong_as_double((long long)((o >> 63) ? (o & 0x7FFFFFFFFFFFFFFFull) : ~o));
}

struct JoinArgs {
    const uint64_t *lists;
    const float2 *sums;
    const float *scores;
    const uint8_t *done;
    float *scores_out;
    int32_t *parents;
    int64_t *tokens;
    uint8_t *done_out;
    int64_t eos;
    int V, K, chunks;
};

// One workgroup per group of beams.  Dynamic shared memory: `cells` totals and as many tags, at least K * chunks and K * K.
// COUNT: up to 1024 of both are ranked by counting what comes before them (152 heads of 8 beams over 19 chunks: 7.9 us for
// the launch, 11.5 with one of 256 threads to a cell); more are sorted, cells being a power of two (the same: 26 us).
template <int THREADS, bool COUNT>
__global__ __launch_bounds__(THREADS) void join_kernel(const JoinArgs A, int cells) {
    extern __shared__ __align__(16) uint64_t tot[];
    uint32_t *tag = reinterpret_cast<uint32_t *>(tot + cells);
    __shared__ double lse[kMaxK];
    __shared__ float score[kMaxK];
    __shared__ uint32_t fin[kMaxK];
    __shared__ int pick[kMaxK];
    const int tid = threadIdx.x, lane = tid & 63, K = A.K, C = A.chunks;
    const int64_t base = (int64_t)blockIdx.x * K;
    // this thread's head, requested before the sums are waited for
    const uint64_t head = COUNT && tid < K * C ? A.lists[(base * C + tid) * K] : 0ull;
    for (int k = tid >> 6; k < K; k += THREADS / 64) {
        const float2 *s = A.sums + (base + k) * C;
        const bool f = A.done != nullptr && A.done[base + k] != 0;
        const float sc = A.scores[base + k];
        float m = -INFINITY;
        double sum = 0.0;
        if (!f) {
            for (int c = lane; c < C; c += 64) m = fmaxf(m, s[c].x);
            m = wave_max(m);
            for (int c = lane; c < C; c += 64) {
                const float2 v = s[c];
                sum += v.x == -INFINITY ? (double)v.y : (double)v.y * (double)__expf(v.x - m);
            }
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, kWave);
        }
        if (lane == 0) {
            lse[k] = (double)m + log(sum);
            score[k] = sc;
            fin[k] = f ? 1u : 0u;
        }
    }
    if (tid < K) pick[tid] = -1;
    __syncthreads();
    const auto total = [&](int k, uint64_t key) -> uint64_t {
        return key == 0 ? 0ull : ordered64((double)score[k] + ((double)value_of((uint32_t)(key >> 32)) - lse[k]));
    };
    // heads of the K * C lists, tag = list; equal totals of one row's lists are ordered by index, as chunks are, and
    // those of different rows by row
    const auto head_of = [&](int i, uint64_t key) -> uint64_t {
        const int k = i / C;
        return !fin[k] ? total(k, key) : i % C == 0 ? ordered64((double)score[k]) : 0ull;
    };
    // entry i of the best lists, tag = k * V + token
    const auto entry_of = [&](int i, uint32_t &f) -> uint64_t {
        const int list = i < K * K ? pick[i / K] : -1;
        f = 0xFFFFFFFFu;
        if (list < 0) return 0;
        const int k = list / C;
        if (!fin[k]) {
            const uint64_t key = A.lists[(base * C + list) * K + i % K];
            f = (uint32_t)(k * A.V) + (0xFFFFFFFFu - (uint32_t)key);
            return total(k, key);
        }
        f = (uint32_t)(k * A.V) + (uint32_t)A.eos;
        return i % K == 0 ? ordered64((double)score[k]) : 0;
    };
    const auto write = [&](int i, uint64_t t, uint32_t f) {
        const int k = t ? (int)(f / (uint32_t)A.V) : i;
        const int64_t token = t ? (int64_t)(f % (uint32_t)A.V) : -1;
        A.scores_out[base + i] = t ? (float)total_of(t) : -INFINITY;
        A.parents[base + i] = k;
        A.tokens[base + i] = token;
        if (A.done_out != nullptr) A.done_out[base + i] = t == 0 || fin[k] || token == A.eos ? 1 : 0;
    };
    if constexpr (COUNT) {
        // calls found(cell, its place) for the candidates among the n cells: a cell's place is how many come before it, two
        // at a time (cells past the last are 0: no candidates, which come after all others), counted by `help` neighbouring
        // lanes; a head's tag is its cell
        const auto rank = [&](int n, bool tagged, auto found) {
            int help = 1;
            while (help < 16 && 2 * help * n <= THREADS) help <<= 1;
            const int cell = tid / help, part = tid & (help - 1);
            if (cell >= n) return;
            const uint64_t t = tot[cell];
            const uint32_t f = tagged ? tag[cell] : (uint32_t)cell;
            int r = 0;
            if (t != 0) {
#pragma unroll 8
                for (int j = 2 * part; j < n; j += 2 * help) {
                    const ulonglong2 a = *reinterpret_cast<const ulonglong2 *>(tot + j);
                    const uint2 g = tagged ? *reinterpret_cast<const uint2 *>(tag + j) : make_uint2(j, j + 1);
                    r += (int)(a.x > t) | ((int)(a.x == t) & (int)(g.x < f));
                    r += (int)(a.y > t) | ((int)(a.y == t) & (int)(g.y < f));
                }
            }
            for (int off = help / 2; off > 0; off >>= 1) r += __shfl_xor(r, off, kWave);
            if (t != 0 && part == 0) found(cell, r);
        };
        const uint64_t h = tid < K * C ? head_of(tid, head) : 0;
        if (tid < cells) tot[tid] = h;
        __syncthreads();
        rank(K * C, false, [&](int cell, int r) {
            if (r < K) pick[r] = cell;
        });
        __syncthreads();
        uint32_t f;
        const uint64_t t = entry_of(tid, f);
        if (tid < cells) {
            tot[tid] = t;
            tag[tid] = f;
        }
        const int some = __syncthreads_count(t != 0);
        rank(K * K, true, [&](int cell, int r) {
            if (r < K) write(r, tot[cell], tag[cell]);
        });
        if (tid < K && tid >= some) write(tid, 0, 0);
    } else {
        const auto before = [&](int i, int j) { return tot[i] > tot[j] || (tot[i] == tot[j] && tag[i] < tag[j]); };
        const auto swap = [&](int i, int j) {
            const uint64_t t = tot[i];
            tot[i] = tot[j];
            tot[j] = t;
            const uint32_t g = tag[i];
            tag[i] = tag[j];
            tag[j] = g;
        };
        int n = 1;
        while (n < K * C) n <<= 1;
        for (int i = tid; i < n; i += THREADS) {
            tot[i] = i < K * C ? head_of(i, A.lists[(base * C + i) * K]) : 0;
            tag[i] = (uint32_t)i;
        }
        __syncthreads();
        sort_shared<THREADS>(n, before, swap);
        if (tid < K && tot[tid] != 0) pick[tid] = (int)tag[tid];
        __syncthreads();
        n = 1;
        while (n < K * K) n <<= 1;
        for (int i = tid; i < n; i += THREADS) {
            uint32_t f;
            const uint64_t t = entry_of(i, f);
            tot[i] = t;
            tag[i] = f;
        }
        __syncthreads();
        sort_shared<THREADS>(n, before, swap);
        if (tid < K) write(tid, tot[tid], tag[tid]);
    }
}

// Chunks of 4096 logits, or of 8192 once those fill the GPU or the join has many heads to rank (4 beams over 32000 logits
// 10.4 us with 4096 and 11.4 with 8192, both launches; 8 beams over 151665 logits 19.2 and 14.3, 16 groups of them 34 and 28).
int64_t chunk_of(int64_t rows, int64_t K, int64_t V) {
    return K * ((V + 4095) / 4096) > 128 || rows * ((V + 8191) / 8192) >= 1024 ? 8192 : 4096;
}
int64_t chunks_of(int64_t rows, int64_t K, int64_t V) { return (V + chunk_of(rows, K, V) - 1) / chunk_of(rows, K, V); }

}  // namespace

extern "C" {

int64_t vgx_beam_select_workspace_bytes(int64_t groups, int64_t K, int64_t V) {
    if (groups < 0 || K <= 0 || V <= 0) return VGX_E_SIZE;
    if (K > kMaxK || V > kMaxV || groups * K > 65535) return VGX_E_LIMIT;
    const int64_t n = groups * K * chunks_of(groups * K, K, V);
    return n * (K * 8 + 8);
}

int vgx_beam_select(const float *logits, int64_t ld, int64_t groups, int64_t K, int64_t V, const float *scores,
                    const uint8_t *done, int64_t eos, float *scores_out, int32_t *parents, int64_t *tokens,
                    uint8_t *done_out, void *workspace, int64_t workspace_bytes, void *stream) {
    const int64_t need = vgx_beam_select_workspace_bytes(groups, K, V);
    if (need < 0) return (int)need;
    if (groups == 0) return VGX_OK;
    if (!logits || !scores || !scores_out || !parents || !tokens) return VGX_E_ARG;
    if (ld < V || eos >= V) return VGX_E_SIZE;
    if (done && eos < 0) return VGX_E_ARG;
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16) return VGX_E_ARENA;
    const int64_t rows = groups * K, C = chunks_of(rows, K, V);
    auto *lists = static_cast<uint64_t *>(workspace);
    auto *sums = reinterpret_cast<float2 *>(lists + rows * C * K);
    const dim3 grid((unsigned)C, (unsigned)rows);
    hipStream_t st = (hipStream_t)stream;
    if (chunk_of(rows, K, V) == 8192)
        hipLaunchKernelGGL((chunk_kernel<32>), grid, dim3(kThreads), 0, st, logits, ld, (int)V, (int)K, done, lists, sums);
    else
        hipLaunchKernelGGL((chunk_kernel<16>), grid, dim3(kThreads), 0, st, logits, ld, (int)V, (int)K, done, lists, sums);
    VGX_CHECK_LAUNCH();
    const JoinArgs A{lists, sums, scores, done, scores_out, parents, tokens, done_out, eos, (int)V, (int)K, (int)C};
    const int most = (int)(std::max(K * C, K * K) + 1) & ~1;
    const auto join = [&](auto kernel, int cells) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(kJoinThreads), (size_t)cells * 12, st, A, cells);
    };
    if (most <= kJoinThreads) {
        join(join_kernel<kJoinThreads, true>, most);
    } else {
        int cells = 1;
        while (cells < most) cells <<= 1;
        join(join_kernel<kJoinThreads, false>, cells);
    }
    VGX_CHECK_LAUNCH();
    return VGX_OK;
}

}  // extern "C"
