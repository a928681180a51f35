// pico_amd/csrc/rope.h -- rotary positions, as the kernel that turns activations and the
// one that fills a cache take them.
#pragma once

#include "pk_common.h"

namespace pk {

struct RopeArgs {
    const double* freqs;
    int half;  // pairs
    int interleaved;
    double magnitude;
};

// m cos a and m sin a of a = pos f.  In 64 bits up to the last rounding: a position of
// 2^20 leaves a product in 32 bits off by 2^-4 radians.  The angle is taken as turns, so
// that its whole part drops out exactly.
__device__ __forceinline__ void rope_angle(int pos, double f, double m, float& c, float& s) {
    const double turns = (double)pos * f * 0.15915494309189533577;
    double ds, dc;
    sincospi(2.0 * (turns - rint(turns)), &ds, &dc);
    c = (float)(dc * m);
    s = (float)(ds * m);
}

// (x1, x2) turned; each product rounded by itself, as the formula stands, so that a value
// does not depend on which kernel turned it
__device__ __forceinline__ void rope_turn(float& x1, float& x2, float c, float s) {
#pragma clang fp contract(off)
    const float y1 = x1 * c - x2 * s;
    x2 = x2 * c + x1 * s;
    x1 = y1;
}
template <class V>
__device__ __forceinline__ void turn(V& a, int i, V& b, int j, float c, float s) {
    float p = a[i], q = b[j];
    rope_turn(p, q, c, s);
    a[i] = p;
    b[j] = q;
}

// n / d for n d < 2^36 as a product with ceil(2^36 / d)
struct Div {
    uint64_t m;
    int d;
    __device__ int of(int n) const { return (int)(((uint64_t)n * m) >> 36); }
};
inline Div div_by(int64_t d) { return {(((uint64_t)1 << 36) + d - 1) / d, (int)d}; }

constexpr int kTurnTable = 512;  // angles a workgroup holds in LDS
constexpr int kTurnUnits = 4;    // units a thread has in flight
constexpr int kTurnHead = 1024;  // largest head, so that one token's fit there

// heads of `tokens` rows, t0 onwards, of x turned into y
struct TurnArgs {
    const float* x;
    float* y;
    int64_t ldx, ldy;
    int H, hd;
    Div per_head, per_token;  // units of a head, heads of a token that a workgroup takes
    int back, accum;
};

// One workgroup: the sines and cosines of the tokens' angles once, in LDS, for all heads;
// then units of 8 values (V = 4: two float4 of a head, neighbouring threads' side by side)
// or of a pair (V = 1), four in flight a thread, those of the first round loaded before the angles.  where(t, pos): the
// position of token t0 + t; false leaves the row.
template <int V, bool INTER, class P>
__device__ __forceinline__ void turn_rows(const TurnArgs& g, const RopeArgs& r, int64_t t0,
                                          int tokens, int heads, P where, float* tc, float* ts) {
    typedef float vec __attribute__((ext_vector_type(V)));
    const int half = r.half, rot = 2 * half, threads = blockDim.x;
    const int total = tokens * g.per_token.d * g.per_head.d;
    constexpr int U = kTurnUnits;
    for(int base = 0; base < total; base += threads * U) {
        vec a[U], b[U];
        int tok[U], at[U], da[U], db[U];  // where a and b are in their head; db < 0: no b
#pragma unroll
        for(int i = 0; i < U; ++i) {
            const int u = base + i * threads + (int)threadIdx.x;
            tok[i] = -1;
            int pos;
            if(u >= total) continue;
            const int hr = g.per_head.of(u), j = u - hr * g.per_head.d, t = g.per_token.of(hr);
            const int h = hr - t * g.per_token.d;
            if(h >= heads || !where(t, pos)) continue;
            tok[i] = t;
            at[i] = h * g.hd;
            if(V == 4) {
                if(INTER || 8 * j >= rot) {
                    const int from = INTER ? 0 : rot, k = INTER ? j : j - rot / 8;
                    da[i] = from + 4 * k;
                    db[i] = da[i] + (g.hd - from + 7) / 8 * 4;
                    if(db[i] >= g.hd) db[i] = -1;
                } else {
                    da[i] = 4 * j;
                    db[i] = 4 * j + half;
                }
            } else if(j < half) {
                da[i] = INTER ? 2 * j : j;
                db[i] = INTER ? 2 * j + 1 : j + half;
            } else {
                da[i] = j + half;
                db[i] = -1;
            }
            const float* p = g.x + (t0 + t) * g.ldx + at[i];
            a[i] = ld_stream((const vec*)(p + da[i]));
            if(db[i] >= 0) b[i] = ld_stream((const vec*)(p + db[i]));
        }
        if(base == 0) {
            for(int e = threadIdx.x; e < tokens * half; e += threads) {
                const int t = e / half;
                int pos;
                if(!where(t, pos)) continue;
                float c, s;
                rope_angle(pos, r.freqs[e - t * half], r.magnitude, c, s);
                tc[e] = c;
                ts[e] = g.back ? -s : s;
            }
            __syncthreads();
        }
#pragma unroll
        for(int i = 0; i < U; ++i) {
            if(tok[i] < 0) continue;
            const float *c = tc + tok[i] * half, *s = ts + tok[i] * half;
            if constexpr(V == 4) {
                if(INTER) {
                    if(da[i] < rot) {
                        const int e = da[i] / 2;
                        turn(a[i], 0, a[i], 1, c[e], s[e]);
                        turn(a[i], 2, a[i], 3, c[e + 1], s[e + 1]);
                    }
                    if(db[i] >= 0 && db[i] < rot) {
                        const int e = db[i] / 2;
                        turn(b[i], 0, b[i], 1, c[e], s[e]);
                        turn(b[i], 2, b[i], 3, c[e + 1], s[e + 1]);
                    }
                } else if(da[i] < half) {
                    const int e = da[i];
#pragma unroll
                    for(int q = 0; q < 4; ++q) turn(a[i], q, b[i], q, c[e + q], s[e + q]);
                }
            } else if(db[i] >= 0) {
                const int e = INTER ? da[i] / 2 : da[i];
                turn(a[i], 0, b[i], 0, c[e], s[e]);
            }
            float* p = g.y + (t0 + tok[i]) * g.ldy + at[i];
            if(g.accum) {
                a[i] += *(const vec*)(p + da[i]);
                if(db[i] >= 0) b[i] += *(const vec*)(p + db[i]);
            }
            st_stream((vec*)(p + da[i]), a[i]);
            if(db[i] >= 0) st_stream((vec*)(p + db[i]), b[i]);
        }
    }
}

inline bool rope_ok(const PkRope* r, int64_t hd) {
    return r->rot >= 0 && r->rot <= hd && r->rot % 2 == 0 && (r->rot == 0 || r->freqs);
}
inline RopeArgs rope_args(const PkRope* r) {
    if(!r) return {nullptr, 0, 0, 1.0};
    return {r->freqs, (int)(r->rot / 2), r->interleaved != 0, r->magnitude};
}
// whether a row is turned in float4, and the arguments for that
inline bool turn_args(TurnArgs& g, const RopeArgs& r, int64_t H, int64_t hd, const float* x,
                      int64_t ldx, float* y, int64_t ldy, int flags) {
    const int rot = 2 * r.half;
    const bool vec = hd % 4 == 0 && rot % (r.interleaved ? 4 : 8) == 0 && ldx % 4 == 0 &&
                     ldy % 4 == 0 && aligned16(x) && aligned16(y);
    g = {x, y, ldx, ldy, (int)H, (int)hd, div_by(vec ? (hd + 7) / 8 : hd - r.half), div_by(H),
         (flags & PK_ROPE_BACKWARD) != 0, (flags & PK_ACCUM) != 0};
    return vec;
}
// tokens a workgroup turns: as many as share a table, fewer where that leaves less than two
// workgroups to a CU, and one where the index arithmetic would pass 2^36
inline int turn_tokens(int64_t N, int64_t H, int half) {
    int T = half ? kTurnTable / 2 / half : 8;
    T = T < 1 || H > 4096 ? 1 : T > 8 ? 8 : T;
    while(T > 1 && (N + T - 1) / T < 512) T /= 2;
    return T;
}

}  // namespace pk
