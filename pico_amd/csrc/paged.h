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

// n / d for 0 <= n < 2^31: with 2^(l-1) < d <= 2^l and m = floor(2^(31+l) / d) + 1, m d
// exceeds 2^(31+l) by d at most, which leaves n m / 2^(31+l) below the next whole number
struct Quotient {
    uint32_t m;
    int s, d;
    __device__ __forceinline__ int of(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n, m) >> s); }
};
inline Quotient quotient(int d) {
    int l = 0;
    while(((int64_t)1 << l) < d) ++l;
    return {d == 1 ? 0u : (uint32_t)(((uint64_t)1 << (31 + l)) / (uint64_t)d + 1), l - 1, d};
}

// sums over the lanes up to one's own
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // from 1, 2, 4 and 8 lanes
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);  // before in a row of 16
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // the last lane of row 0
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // and 2; of rows 0 and 1
    return v;
}
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// The sequences' shares stand in one line, whose length fits 31 bits; start(length) is a
// place in it.  Finds the sequence there, its number `b` and the place `at` within its
// share; false beyond the end, and where offsets that decrease make the sums wrap.  64
// sequences at a time, one a lane; up to 64 of them take one trip to memory, more of them two
// walks over all: a token in each of 256 sequences, 64 behind, 4 heads on 1 of 64, is appended in
// 6 us and attends in 7, of 1024 in 14 and 19, of 4096 in 86 and 138.
template <class F, class G>
__device__ __forceinline__ bool locate(const PkKvCache& c, int N, F share, G start, int& at, int& b,
                                       Seq& s) {
    const int lane = threadIdx.x % kWave, B = (int)c.B;
    int all = 0;
    if(B > kWave) {
        for(int i = lane; i < B; i += kWave) all += share(sequence(c, N, i));
        all = lane_of(wave_scan(all), kWave - 1);
        at = start(all);
        if(at >= all) return false;
    }
    for(int base = 0; base < B; base += kWave) {
        Seq mine = {};
        if(base + lane < B) mine = sequence(c, N, base + lane);
        const int len = base + lane < B ? share(mine) : 0, upto = wave_scan(len);
        if(B <= kWave) at = start(lane_of(upto, kWave - 1));
        const uint64_t above = __ballot(upto > at);
        if(above) {
            const int first = __builtin_ctzll(above);
            at -= lane_of(upto - len, first);
            b = base + first;
            s = {lane_of(mine.row, first), lane_of(mine.n, first), lane_of(mine.past, first),
                 lane_of(mine.end, first)};
            return at >= 0 && at < lane_of(len, first);
        }
        at -= lane_of(upto, kWave - 1);
    }
    return false;
}

// the smallest e, from -40 to 40, with amax <= 448 2^e; 448 is 0.875 2^9
__device__ __forceinline__ int block_exponent(float amax) {
    if(!(amax > 0.0f)) return kExpMin;
    const int x = __builtin_amdgcn_frexp_expf(amax);
    return held(x - (__builtin_amdgcn_frexp_mantf(amax) <= 0.875f ? 9 : 8), kExpMin, kExpMax);
}

// A page's byte, e + 127, or the nearest that there is where it is none.  (Two instructions
// with a constant each; one with both takes a register for the length of a loop, and tiles of
// 128 rows of heads of 64 a third wave.)
__device__ __forceinline__ int exponent_byte(int b) {
    int x = b > 127 + kExpMin ? b : 127 + kExpMin;
    asm("" : "+v"(x));
    return x < 127 + kExpMax ? x : 127 + kExpMax;
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
    if(c->kv_heads < 1 || c->kv_heads > 4096 || c->pages < 1 ||
       c->pages > (((int64_t)1 << 31) - 1) / c->kv_heads ||
       c->B < 0 || c->B > (1 << 20) || c->width < 1 || c->width > (((int64_t)1 << 30) - 1) / c->page)
        return fail("%s: kv_heads %lld, pages %lld, B %lld, width %lld: 1 to 4096 heads, fewer than "
                    "2^31 pages times heads, up to 2^20 sequences of fewer than 2^30 positions",
                    who, (long long)c->kv_heads, (long long)c->pages, (long long)c->B,
                    (long long)c->width);
    if(N < 0 || N >= (int64_t)1 << 24)
        return fail("%s: N %lld: 0 to 2^24 - 1 rows", who, (long long)N);
    if(!c->k || !c->v || !c->k_exp || !c->v_exp || (c->B > 0 && (!c->table || !c->lens || !c->offsets)))
        return fail("%s: NULL pointer in the cache", who);
    if(!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_exp) || !aligned16(c->v_exp))
        return fail("%s: k, v and their exponents must be 16-byte aligned", who);
    return PK_OK;
}

}  // namespace pk
