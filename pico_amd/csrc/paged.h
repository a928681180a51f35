// pico_amd/csrc/paged.h -- what the kernels of the paged cache share: its sequences as the
// device reads them, and a page's power of two.
#pragma once

#include "pk_common.h"

namespace pk {

constexpr int kExpMin = -40, kExpMax = 40;

// one sequence of a call: rows [row, row + n) of the inputs, at positions past, past + 1,
// .. below end; whatever the arrays hold stays within the inputs and the table
struct Seq {
    int row, n, past, end;
};
__device__ __forceinline__ int held(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }
__device__ __forceinline__ Seq sequence(const PkKvCache& c, int N, int b) {
    const int cap = (int)(c.width * c.page);
    Seq s;
    s.row = held(c.offsets[b], 0, N);
    s.n = held(c.offsets[b + 1], s.row, N) - s.row;
    s.past = held(c.lens[b], 0, cap);
    s.end = s.n < cap - s.past ? s.past + s.n : cap;
    return s;
}

// the sequence in whose share of a sum over the sequences `at` falls, and where in it
// (-1: beyond all): 64 sequences at a time, one a lane
template <class I, class F>
__device__ __forceinline__ int find_sequence(int B, I& at, F share) {
    const int lane = threadIdx.x % kWave;
    for(int base = 0; base < B; base += kWave) {
        const I mine = base + lane < B ? share(base + lane) : 0;
        I upto = mine;
#pragma unroll
        for(int o = 1; o < kWave; o <<= 1) {
            const I other = __shfl_up(upto, o, kWave);
            if(lane >= o) upto += other;
        }
        const uint64_t above = __ballot(upto > at);
        if(above) {
            const int first = __builtin_ctzll(above);
            at -= __shfl(upto - mine, first, kWave);
            return base + first;
        }
        at -= __shfl(upto, kWave - 1, kWave);
    }
    return -1;
}

// the smallest e, from -40 to 40, with amax <= 448 2^e; 448 is 0.875 2^9
__device__ __forceinline__ int block_exponent(float amax) {
    if(!(amax > 0.0f)) return kExpMin;
    const int x = __builtin_amdgcn_frexp_expf(amax);
    return held(x - (__builtin_amdgcn_frexp_mantf(amax) <= 0.875f ? 9 : 8), kExpMin, kExpMax);
}

inline int head_size(int64_t hd) {
    return hd < 1 || hd > 256 ? 0 : hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 96 ? 96 : hd <= 128 ? 128 : 256;
}

// refuses a cache that the kernels' index arithmetic or its layout does not cover
inline int check_cache(const char* who, const PkKvCache* c, int64_t N) {
    if(!c) return fail("%s: NULL cache", who);
    if(!head_size(c->hd)) return fail("%s: head size %lld: 1 to 256", who, (long long)c->hd);
    if(c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128)
        return fail("%s: pages of %lld tokens: 16, 32, 64 or 128", who, (long long)c->page);
    if(c->kv_heads < 1 || c->kv_heads > 4096 || c->pages < 1 || c->pages >= (int64_t)1 << 31 ||
       c->B < 0 || c->B > (1 << 20) || c->width < 1 || c->width > (((int64_t)1 << 30) - 1) / c->page)
        return fail("%s: kv_heads %lld, pages %lld, B %lld, width %lld: 1 to 4096 heads, 1 to 2^31 - 1 "
                    "pages, up to 2^20 sequences of fewer than 2^30 positions",
                    who, (long long)c->kv_heads, (long long)c->pages, (long long)c->B,
                    (long long)c->width);
    if(N < 0 || N >= (int64_t)1 << 24)
        return fail("%s: N %lld: 0 to 2^24 - 1 rows", who, (long long)N);
    if(!c->k || !c->v || !c->k_exp || !c->v_exp || !c->table || !c->lens || !c->offsets)
        return fail("%s: NULL pointer in the cache", who);
    if(!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_exp) || !aligned16(c->v_exp))
        return fail("%s: k, v and their exponents must be 16-byte aligned", who);
    return PK_OK;
}

}  // namespace pk
