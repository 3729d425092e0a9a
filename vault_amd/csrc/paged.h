// The paged 8-bit K/V cache: formats, addresses and the split of a batch's rows over workgroups
// (include/vault_amd.h describes the layout).
#pragma once

#include "common.h"

#include <algorithm>
#include <type_traits>

namespace vgx {

constexpr int64_t kMaxGroups = (1 << 24) - 1;      // workgroups of 256 threads in a launch of less than 2^32 threads
constexpr float kQMaxI8 = 127.0f, kQMaxE4M3 = 448.0f;

// A layer's pages as kernels see them.
struct PagedLayer {
    uint8_t *k, *v;
    float *ks, *vs;
    int64_t head_bytes;         // page * D
    int n_pages, G, log_page;
};

// The value of a code byte, without its scale.
template <int FMT>
VGX_DEV float code_value(uint32_t u) {
    if constexpr (FMT == VGX_I8) return (float)((int)(u & 0xFFu) - 128);
    return __builtin_amdgcn_cvt_f32_fp8((int)u, 0);
}

// Four codes of a word to floats.
template <int FMT>
VGX_DEV void code_values4(uint32_t w, float (&o)[4]) {
    if constexpr (FMT == VGX_I8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = (float)((w >> (8 * i)) & 0xFFu) - 128.0f;
    } else {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        o[0] = lo[0];
        o[1] = lo[1];
        o[2] = hi[0];
        o[3] = hi[1];
    }
}

// Four quotients (finite) to codes, to nearest even, saturating.
template <int FMT>
VGX_DEV uint32_t to_codes4(const float (&x)[4]) {
    if constexpr (FMT == VGX_I8) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= (uint32_t)((int)fminf(fmaxf(rintf(x[i]), -127.0f), 127.0f) + 128) << (8 * i);
        return w;
    } else {
        const auto c = [](float v) { return fminf(fmaxf(v, -kQMaxE4M3), kQMaxE4M3); };
        const int w = __builtin_amdgcn_cvt_pk_fp8_f32(c(x[0]), c(x[1]), 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c(x[2]), c(x[3]), w, true);
    }
}

// Rows [lo, hi) of a batch's N rows belong to sequence b.
struct SeqRows {
    int lo, hi;
};
VGX_DEV SeqRows seq_rows(const int32_t *__restrict__ q_start, int b, int N) {
    if (q_start == nullptr) return {b, b + 1};
    const int lo = min(max(q_start[b], 0), N);
    return {lo, min(max(q_start[b + 1], lo), N)};
}

// Unit `x` of the units count(b) that every sequence has, in order of b: finds b and the unit's place in it (every lane of
// a wave with the same x takes part); b < 0 past the last.  A wave sums 64 sequences at a time.
template <class Count>
VGX_DEV int find_unit(int64_t x, int B, Count count, int64_t &place) {
    const int lane = threadIdx.x & 63;
    int64_t base = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int mine = b0 + lane < B ? count(b0 + lane) : 0;
        int sum = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int up = __shfl_up(sum, off, kWave);
            if (lane >= off) sum += up;
        }
        const int total = __shfl(sum, 63, kWave);
        if (x < base + total) {
            const uint64_t past = __ballot(base + sum > x);       // lanes whose units end after x
            const int l = __ffsll((unsigned long long)past) - 1;
            place = x - base - __shfl(sum - mine, l, kWave);
            return b0 + l;
        }
        base += total;
    }
    return -1;
}

inline int check_paged(const vgx_paged_kv *kv, int64_t layer) {
    if (!kv || !kv->k || !kv->v || !kv->k_scale || !kv->v_scale) return VGX_E_ARG;
    if (kv->fmt != VGX_I8 && kv->fmt != VGX_E4M3) return VGX_E_DTYPE;
    if (kv->D != 64 && kv->D != 128) return VGX_E_SHAPE;
    if (kv->page != 16 && kv->page != 32 && kv->page != 64 && kv->page != 128 && kv->page != 256) return VGX_E_SHAPE;
    if (kv->G <= 0 || kv->n_pages <= 0 || kv->n_layers <= 0 || layer < 0 || layer >= kv->n_layers) return VGX_E_SIZE;
    if (kv->G > 65535 || kv->n_pages > 0x7FFFFFFF || kv->n_layers > 65535) return VGX_E_LIMIT;
    if (kv->n_layers > 1 && (kv->layer_stride < kv->n_pages * kv->G * kv->page * kv->D ||
                             kv->scale_layer_stride < kv->n_pages * kv->G))
        return VGX_E_SIZE;
    if (((uintptr_t)kv->k | (uintptr_t)kv->v) % 16 || kv->layer_stride % 16) return VGX_E_ALIGN;
    if (((uintptr_t)kv->k_scale | (uintptr_t)kv->v_scale) % 4) return VGX_E_ALIGN;
    return VGX_OK;
}

inline PagedLayer paged_layer(const vgx_paged_kv *kv, int64_t layer) {
    PagedLayer p;
    p.k = kv->k + layer * kv->layer_stride;
    p.v = kv->v + layer * kv->layer_stride;
    p.ks = kv->k_scale + layer * kv->scale_layer_stride;
    p.vs = kv->v_scale + layer * kv->scale_layer_stride;
    p.head_bytes = kv->page * kv->D;
    p.n_pages = (int)kv->n_pages;
    p.G = (int)kv->G;
    p.log_page = __builtin_ctzll((unsigned long long)kv->page);
    return p;
}

// A device table of `cols` page ids per sequence.
inline int check_table(const int32_t *table, int64_t ldt, int64_t cols) {
    if (!table) return VGX_E_ARG;
    if (cols <= 0 || ldt < cols) return VGX_E_SIZE;
    if (cols > 0x7FFFFFFF) return VGX_E_LIMIT;
    return VGX_OK;
}

// f(format, D, whether bf16) with the three as compile-time constants.
template <class F>
inline int with_format(int fmt, int64_t D, bool bf16, F f) {
    const auto dims = [&](auto fm) {
        if (D == 128) return bf16 ? f(fm, std::integral_constant<int, 128>{}, std::true_type{})
                                  : f(fm, std::integral_constant<int, 128>{}, std::false_type{});
        return bf16 ? f(fm, std::integral_constant<int, 64>{}, std::true_type{})
                    : f(fm, std::integral_constant<int, 64>{}, std::false_type{});
    };
    return fmt == VGX_I8 ? dims(std::integral_constant<int, VGX_I8>{}) : dims(std::integral_constant<int, VGX_E4M3>{});
}

}  // namespace vgx
