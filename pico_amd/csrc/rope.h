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
__device__ __forceinline__ void rope_turns(int pos, double f, double& c, double& s) {
    const double turns = (double)pos * f * 0.15915494309189533577;
    sincospi(2.0 * (turns - rint(turns)), &s, &c);
}
__device__ __forceinline__ void rope_angle(int pos, double f, double m, float& c, float& s) {
    double ds, dc;
    rope_turns(pos, f, dc, ds);
    c = (float)(dc * m);
    s = (float)(ds * m);
}

// (x1, x2) turned; each product rounded by itself, as the formula stands, so that the same
// sine and cosine give the same value in every kernel
__device__ __forceinline__ void rope_turn(float& x1, float& x2, float c, float s) {
#pragma clang fp contract(off)
    const float y1 = x1 * c - x2 * s;
    x2 = x2 * c + x1 * s;
    x1 = y1;
}
__device__ __forceinline__ void turn(f32x4& a, int i, f32x4& b, int j, float c, float s) {
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

// (such pieces share lines, which stay in the caches for that: 8192 tokens of 32 heads of 126,
// 42 turned, 160 to 130 us both ways)
typedef float f32x4_anywhere __attribute__((ext_vector_type(4), aligned(4)));
// 4 values of a row of n from `at` on, or those that there are; any of the row in their
// place behind them
__device__ __forceinline__ f32x4 ld_in_row(const float* row, int at, int n) {
    return *(const f32x4_anywhere*)(row + (at < n - 4 ? at : n - 4));
}
__device__ __forceinline__ f32x4 from_window(f32x4 v, int at, int n) {
    const int behind = at - (n - 4);
    if(behind > 0) {
        if(behind & 1) v = f32x4{v[1], v[2], v[3], v[3]};
        if(behind & 2) v = f32x4{v[2], v[3], v[3], v[3]};
    }
    return v;
}
__device__ __forceinline__ void st_first(float* to, f32x4 v, int n) {
    if(n >= 4) {
        *(f32x4_anywhere*)to = v;
    } else {
#pragma unroll
        for(int k = 0; k < 3; ++k)
            if(k < n) to[k] = v[k];
    }
}

// One workgroup: the sines and cosines of the tokens' angles once, in LDS, for all heads;
// then units of 8 values, two times 4 in a row of a head, neighbouring threads' side by
// side: pairs of the first half with those of the second, or what is next to each other.
// Four units are in flight a thread, those of the first round loaded before the angles.
// EVEN: head, halves and strides are multiples of 4 and aligned.  Where they are not, a
// part's last 4 may be fewer; all are loaded as 4, and without a branch, so
// that none is waited for before the others are issued (8192 tokens of 12 heads of 80, 20
// turned: 30 us both ways, 40 from HBM, pair by pair 69; 25 at the rate of a copy).
// where(t, pos): the position of token t0 + t; false leaves the row.
template <bool EVEN, bool INTER, class P>
__device__ __forceinline__ void turn_rows(const TurnArgs& g, const RopeArgs& r, int64_t t0,
                                          int tokens, int heads, P where, float* tc, float* ts) {
    const int half = r.half, rot = 2 * half, threads = blockDim.x, turned = (half + 3) / 4;
    const int total = tokens * g.per_token.d * g.per_head.d, row = heads * g.hd;
    if(!EVEN && row < 4) {  // (too short to load 4)
        for(int t = threadIdx.x; t < tokens; t += threads) {
            int pos;
            if(!where(t, pos)) continue;
            const float* x = g.x + (t0 + t) * g.ldx;
            float* y = g.y + (t0 + t) * g.ldy;
            for(int i = 0; i < row; ++i) {
                // (the only pair of such a head is of its first two)
                const int d = i % g.hd;
                float a = x[i], b = 0.0f;
                if(d < rot) {
                    float c, s;
                    rope_angle(pos, r.freqs[0], r.magnitude, c, s);
                    b = x[++i];
                    rope_turn(a, b, c, g.back ? -s : s);
                    y[i] = g.accum ? y[i] + b : b;
                }
                float* to = y + (d < rot ? i - 1 : i);
                *to = g.accum ? *to + a : a;
            }
        }
        return;
    }
    constexpr int U = EVEN ? kTurnUnits : kTurnUnits / 2;  // (the windows' selections take registers)
    for(int base = 0; base < total; base += threads * U) {
        f32x4 a[U], b[U];
        // where a and b are in their head, and of how many values (b of none, where nb < 1)
        int tok[U], at[U], da[U], db[U], na[U], nb[U];
#pragma unroll
        for(int i = 0; i < U; ++i) {
            const int u = base + i * threads + (int)threadIdx.x;
            tok[i] = -1;
            int pos;
            if(EVEN && u >= total) continue;
            const int hr = g.per_head.of(u < total ? u : 0), j = u - hr * g.per_head.d;
            const int t = tokens == 1 ? 0 : g.per_token.of(hr), h = hr - t * g.per_token.d;
            const bool there = u < total && h < heads && where(t, pos);
            if(EVEN && !there) continue;
            if(there) tok[i] = t;
            at[i] = h * g.hd;
            const bool pairs = !INTER && j < turned;  // of the first half and the second
            const int from = INTER ? 0 : rot, k = INTER ? j : j - turned;
            da[i] = pairs ? 4 * j : from + 4 * k;
            db[i] = da[i] + (pairs ? half : (g.hd - from + 7) / 8 * 4);
            na[i] = (pairs ? half : g.hd) - da[i];
            nb[i] = (pairs ? rot : g.hd) - db[i];
            const float* p = g.x + (t0 + t) * g.ldx;
            if(EVEN) {
                a[i] = ld_stream((const f32x4*)(p + at[i] + da[i]));
                if(nb[i] > 0) b[i] = ld_stream((const f32x4*)(p + at[i] + db[i]));
            } else {
                a[i] = ld_in_row(p, there ? at[i] + da[i] : 0, row);
                b[i] = ld_in_row(p, there ? at[i] + db[i] : 0, row);
            }
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
            if(!EVEN) {
                a[i] = from_window(a[i], at[i] + da[i], row);
                b[i] = from_window(b[i], at[i] + db[i], row);
            }
            if(INTER) {
#pragma unroll
                for(int k = 0; k < 4; k += 2) {
                    const int e = (da[i] + k) / 2, f = (db[i] + k) / 2;
                    if(da[i] + k < rot) turn(a[i], k, a[i], k + 1, c[e], s[e]);
                    if(db[i] + k < rot) turn(b[i], k, b[i], k + 1, c[f], s[f]);
                }
            } else if(da[i] < half) {
                const int e = da[i];
#pragma unroll
                for(int k = 0; k < 4; ++k)
                    if(EVEN || k < na[i]) turn(a[i], k, b[i], k, c[e + k], s[e + k]);
            }
            float *pa = g.y + (t0 + tok[i]) * g.ldy + at[i] + da[i], *pb = pa + (db[i] - da[i]);
            if(EVEN) {
                if(g.accum) {
                    a[i] += *(const f32x4*)pa;
                    if(nb[i] > 0) b[i] += *(const f32x4*)pb;
                }
                st_stream((f32x4*)pa, a[i]);
                if(nb[i] > 0) st_stream((f32x4*)pb, b[i]);
            } else {
                if(g.accum) {
#pragma unroll
                    for(int k = 0; k < 4; ++k) {
                        if(k < na[i]) a[i][k] += pa[k];
                        if(k < nb[i]) b[i][k] += pb[k];
                    }
                }
                st_first(pa, a[i], na[i]);
                st_first(pb, b[i], nb[i]);
            }
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
// the arguments, and whether all is multiples of 4 and aligned
inline bool turn_args(TurnArgs& g, const RopeArgs& r, int64_t H, int64_t hd, const float* x,
                      int64_t ldx, float* y, int64_t ldy, int flags) {
    const int rot = 2 * r.half;
    g = {x, y, ldx, ldy, (int)H, (int)hd,
         div_by(r.interleaved ? (hd + 7) / 8 : (r.half + 3) / 4 + (hd - rot + 7) / 8), div_by(H),
         (flags & PK_ROPE_BACKWARD) != 0, (flags & PK_ACCUM) != 0};
    return hd % 4 == 0 && rot % (r.interleaved ? 4 : 8) == 0 && ldx % 4 == 0 && ldy % 4 == 0 &&
           aligned16(x) && aligned16(y);
}
// tokens a workgroup turns: as many as share a table, fewer where that leaves less than two
// workgroups to a CU, and one of many heads, whose
// index arithmetic would pass 2^36
inline int turn_tokens(int64_t N, int64_t H, int half) {
    int T = half ? kTurnTable / 2 / half : 8;
    T = T < 1 || H > 4096 ? 1 : T > 8 ? 8 : T;
    while(T > 1 && (N + T - 1) / T < 512) T /= 2;
    return T;
}

}  // namespace pk
