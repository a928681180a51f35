// pico_amd/csrc/scan.hip -- a gated linear recurrence along the tokens of each
// sequence, channel by channel, and its gradients.
//
//   s_t = sigmoid(f_t),  h_t = s_t h_{t-1} + (1 - s_t) x_t,  h_0 given or zero
// and backwards, with the gradient u that a token hands to the one before it,
//   G_t = dh_t + u_{t+1},  u_t = s_t G_t
//   dx_t = (1 - s_t) G_t,  df_t = G_t (h_{t-1} - x_t) s_t (1 - s_t),  dh_0 = u_1
//
// A gate that is shut or open in fp32 (s or 1 - s is 0) leaves the other side out, whatever
// that holds: with s = 0 no infinity or NaN passes from the tokens before to this one
// and those after it, nor back with the gradients; with 1 - s = 0 none from x_t.
//
// Both directions are chains of p -> A p + H (forward A = s, H = q x; backward A = s,
// H = s dh), and a run of steps is again one: (A2, H2) after (A1, H1) is
// (A1 A2, A2 H1 + H2).  A workgroup walks its steps in tiles: a thread has 4
// consecutive steps of 4 channels, composes them, the threads' results are scanned
// across the lanes and through LDS, and every thread goes over its steps again, in
// registers, from the value that reaches it.  The next tile's loads are in flight
// meanwhile, so memory is read once: 12 bytes an element forward, 24 backward.
// Sums are fp32, in an order that depends on the sizes alone.
#include <type_traits>

#include "pk_common.h"

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kThreads = 256, kWaves = kThreads / 64, LT = 4;  // LT steps a thread

// s = sigmoid(f) and q = 1 - s = sigmoid(-f): with t = exp(-|f|) they are 1 / (1 + t) and
// t / (1 + t), the smaller one not got by subtraction.  t is 2^(-|f| log2 e), log2 e in two
// parts as in Cody and Waite's reduction, with what the exponent's product rounds off put
// back to first order (|f| below 200, beyond which t is 0); the quotient is the
// hardware's reciprocal after one step of Newton's.  That is half the instructions of expf
// and a division, which bound the kernels (47 a value in all, 8192 x 768 forward and
// backward 19 + 35 us; now 28).  With u = 2^-24, exp2 and the reciprocal within an ulp (2 u):
// t is off by 2 u and a rounding, 1 + t by half of that at most and a rounding, so the
// larger one by 3.5 u, the smaller by 6 u (2.0 and 4.1 at most over 4 million f).  From |f| =
// 87.34 on, where t is below 2^-126, exp2 gives 0, and so is the smaller one.
__device__ __forceinline__ void gate(float f, float& s, float& q) {
    constexpr float kLog2e = 1.44269502162933349609375f, kLow = 1.925963033500011079e-8f;
    float a = fabsf(f);
    a = a > 200.0f ? 200.0f : a;  // (NaN stays NaN)
    const float hi = a * kLog2e, lo = fmaf(a, kLow, fmaf(a, kLog2e, -hi));
    float t = __builtin_amdgcn_exp2f(-hi);
    t = fmaf(t, -0.693147182464599609375f * lo, t);
    const float d = 1.0f + t, r0 = __builtin_amdgcn_rcpf(d);
    const float big = fmaf(r0, fmaf(-d, r0, 1.0f), r0), small = t * big;
    s = f >= 0.0f ? big : small;
    q = f >= 0.0f ? small : big;
}

// V channels from `at`.  A lane at the end of a row with fewer than 4 left reads the
// row's last 4 (rows of fewer than 4 channels have V = 1): `skip` of them belong
// to the lane before it and are not stored.
template <int V, bool NT = false>
__device__ __forceinline__ void load(const float* at, float (&v)[V]) {
    if constexpr(V == 4) {
        const f32x4u* const a = reinterpret_cast<const f32x4u*>(at);
        const f32x4 x = NT ? __builtin_nontemporal_load(a) : *a;
#pragma unroll
        for(int i = 0; i < 4; ++i) v[i] = x[i];
    } else {
        v[0] = *at;
    }
}
// (nontemporal: outputs that stay in the cache cost the inputs their place there; 32x2048x256
// backward 93 -> 68 us, 1x65536x512 forward 116 -> 104)
template <int V>
__device__ __forceinline__ void store(float* at, const float (&v)[V], int skip, bool accum) {
    if constexpr(V == 4) {
        if(skip == 0) {
            f32x4 x = {v[0], v[1], v[2], v[3]};
            f32x4u* o = reinterpret_cast<f32x4u*>(at);
            if(accum) x = *o + x;
            __builtin_nontemporal_store(x, o);
            return;
        }
    }
#pragma unroll
    for(int i = 0; i < V; ++i)
        if(i >= skip) at[i] = accum ? at[i] + v[i] : v[i];
}

struct ScanParams {
    int64_t B, T, C;
    const float *f, *x, *h0, *h, *dh;
    int64_t ldf, ldx, lddf, lddx;
    float *out, *df, *dx, *dh0;  // forward: out
    int flags;
    float* ws;      // [S][B][C] A, then the same of H
    int S;          // chunks along the tokens
    int64_t L;      // steps of a chunk
    int groups;     // channel groups of a sequence
};

// CL lanes along the channels, V channels each
template <int V, int CL>
struct Place {
    static constexpr int TL = kThreads / CL, TT = TL * LT;  // lanes along the steps, steps of a tile
    int64_t b, c, chunk;
    int tl, cl, skip;
    bool on;

    // a run of channel groups to each XCD: groups narrower than a cache line meet
    // in one L2
    __device__ __forceinline__ explicit Place(const ScanParams& p) {
        const int64_t n = p.B * p.groups, run = (n + 7) / 8;
        const int64_t id = (blockIdx.x & 7) * run + (blockIdx.x >> 3);
        on = (blockIdx.x >> 3) < run && id < n;
        b = id / p.groups;
        tl = threadIdx.x / CL;
        cl = threadIdx.x % CL;
        chunk = blockIdx.y;
        c = ((id % p.groups) * CL + cl) * V;
        skip = 0;
        if(c + V > p.C) {
            // (lanes wholly past the row repeat its last channels and store nothing)
            skip = (int)min(c + V - p.C, (int64_t)V);
            c = p.C - V;
        }
    }
};

// a b, and 0 where one of them is, whatever the other holds (the instruction has no
// builtin; equal to a multiplication bit for bit where neither is 0)
__device__ __forceinline__ float product(float a, float b) {
    float r;
    asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// The arithmetic of runs has two forms.  BAD is for values that may be infinite or NaN: a
// run with a shut gate has A = -0, which leaves p out, while the product of many gates
// that are not shut may come to +0, through which an infinity or NaN does go on.  The
// other form multiplies by 0 like by anything else, and in it no value of a chain is
// finite behind one that is not: the last one tells whether all has to be done again, in
// the other form, a step at a time, after the loops (in them it takes registers or time:
// selects throughout 8x1024x768 forward and backward 21.5 + 34.5 us, a tile at a time
// 18.2 + 30.6, so 18.0 + 29.1, and 55 + 79 with a NaN at the first token).
constexpr float kShut = -0.0f;
__device__ __forceinline__ bool shut(float A) { return __float_as_uint(A) == 0x80000000u; }

template <int V>
__device__ __forceinline__ bool any_bad(const float (&p)[V]) {
    float sum = 0.0f;
#pragma unroll
    for(int i = 0; i < V; ++i) sum = fmaf(p[i], 0.0f, sum);
    return __any(sum != 0.0f);
}

// p behind a run of steps, and (A, H) of a run behind (a, h) of the one before it
template <bool BAD>
__device__ __forceinline__ float behind(float A, float H, float p) {
    return BAD && shut(A) ? H : fmaf(A, p, H);
}
template <bool BAD>
__device__ __forceinline__ void compose(float& A, float& H, float a, float h) {
    H = behind<BAD>(A, H, h);
    if(!BAD || !shut(A)) A *= a;
}

// one step of the chain (forward v = q x, backward dh), and one at the end of a run
template <bool BWD, bool BAD>
__device__ __forceinline__ float step(float p, float s, float v) {
    if(BWD) return BAD && s == 0.0f ? 0.0f : s * (v + p);
    return BAD && s == 0.0f ? v : fmaf(s, p, v);
}
template <bool BWD, bool BAD>
__device__ __forceinline__ void extend_run(float s, float v, float& A, float& H) {
    A = BAD && s == 0.0f ? kShut : A * s;
    H = step<BWD, BAD>(H, s, v);
}

// dx and df of a token; returns the gradient it hands to the one before it.  (h and x may
// be bad where the chain of the gradients is not)
template <bool BAD>
__device__ __forceinline__ float gradients(float G, float h, float x, float s, float q, float& dx, float& df) {
    dx = BAD && q == 0.0f ? 0.0f : q * G;
    df = BAD ? (s == 0.0f || q == 0.0f ? 0.0f : G * (h - x) * (s * q)) : product(G * (h - x), s * q);
    return BAD && s == 0.0f ? 0.0f : s * G;
}

// (A, H) of the lanes' steps, in step order -> the value that reaches each lane
// from `carry`; carry becomes the one behind the last lane, the same in every wave.  One
// barrier; `turn` alternates between calls.
template <int V, int CL, bool BAD>
__device__ __forceinline__ void through(float (&A)[V], float (&H)[V], float (&carry)[V], float (&in)[V],
                                        float (*lds)[kWaves][2][V * CL], int turn) {
    const int lane = threadIdx.x % 64, w = threadIdx.x / 64, cl = threadIdx.x % CL;
#pragma unroll
    for(int o = CL; o < 64; o <<= 1) {
#pragma unroll
        for(int i = 0; i < V; ++i) {
            const float a = __shfl_up(A[i], o, 64), h = __shfl_up(H[i], o, 64);
            if(lane >= o) compose<BAD>(A[i], H[i], a, h);
        }
    }
    typedef float Lane __attribute__((ext_vector_type(V)));
    if(lane >= 64 - CL) {
        Lane a, h;
#pragma unroll
        for(int i = 0; i < V; ++i) {
            a[i] = A[i];
            h[i] = H[i];
        }
        *reinterpret_cast<Lane*>(&lds[turn][w][0][cl * V]) = a;
        *reinterpret_cast<Lane*>(&lds[turn][w][1][cl * V]) = h;
    }
    __syncthreads();
    Lane a[kWaves], h[kWaves];
#pragma unroll
    for(int q = 0; q < kWaves; ++q) {
        a[q] = *reinterpret_cast<const Lane*>(&lds[turn][q][0][cl * V]);
        h[q] = *reinterpret_cast<const Lane*>(&lds[turn][q][1][cl * V]);
    }
    float own[V];
#pragma unroll
    for(int i = 0; i < V; ++i) {
        own[i] = carry[i];
#pragma unroll
        for(int q = 0; q < kWaves; ++q) {
            if(q == w) own[i] = carry[i];
            carry[i] = behind<BAD>(a[q][i], h[q][i], carry[i]);
        }
        const float a = __shfl_up(A[i], CL, 64), h = __shfl_up(H[i], CL, 64);
        in[i] = lane >= CL ? behind<BAD>(a, h, own[i]) : own[i];
    }
}

// the composed (A, H) of every chunk but the last, tile by tile like scan_tiles (a
// thread with a run of the chunk of its own read 64 rows apart: 4.1 TB/s), the last tile
// first: what is read last is what scan_tiles starts with, out of the last-level cache
// (1x32768x256 forward 32.8 -> 27.5 us, 1x262144x256 274 -> 234, backward 436 -> 391)
template <int V, int CL, bool BWD>
__global__ __launch_bounds__(kThreads, 4) void scan_chunks(ScanParams p) {
    using Pl = Place<V, CL>;
    __shared__ alignas(16) float lds[2][kWaves][2][V * CL];
    const Pl at(p);
    if(!at.on) return;
    const int64_t g0 = at.chunk * p.L + p.L - Pl::TT + at.tl * LT, t0 = BWD ? p.T - 1 - g0 : g0;
    const int64_t ldv = BWD ? p.C : p.ldx, df = BWD ? -p.ldf : p.ldf, dv = BWD ? -ldv : ldv;
    const float* fp = p.f + (at.b * p.T + t0) * p.ldf + at.c;
    const float* vp = (BWD ? p.dh : p.x) + (at.b * p.T + t0) * ldv + at.c;
    float all[V], carry[V], in[V], fr[LT][V], vr[LT][V];
#pragma unroll
    for(int i = 0; i < V; ++i) {
        all[i] = 1.0f;
        carry[i] = 0.0f;
    }
    auto fetch = [&]() {
#pragma unroll
        for(int e = 0; e < LT; ++e) {
            load<V>(fp + e * df, fr[e]);
            load<V>(vp + e * dv, vr[e]);
        }
        fp -= Pl::TT * df;
        vp -= Pl::TT * dv;
    };
    fetch();
    // the least s of the thread's steps
    float least[V];
#pragma unroll
    for(int i = 0; i < V; ++i) least[i] = 1.0f;
    int turn = 0;
    float A[V], H[V];
    // (all, carry), of the tiles behind this one, with its own before them
    auto add = [&](auto bad) {
        constexpr bool BAD = decltype(bad)::value;
        float own[V];
#pragma unroll
        for(int i = 0; i < V; ++i) own[i] = 0.0f;
        through<V, CL, BAD>(A, H, own, in, lds, turn);
#pragma unroll
        for(int i = 0; i < V; ++i) {
            carry[i] = behind<BAD>(all[i], carry[i], own[i]);
#pragma unroll
            for(int q = kWaves - 1; q >= 0; --q)
                if(!BAD || !shut(all[i])) all[i] *= lds[turn][q][0][at.cl * V + i];
        }
        turn ^= 1;
    };
    auto walk = [&](auto last) {
        float s[LT][V];
#pragma unroll
        for(int e = 0; e < LT; ++e)
#pragma unroll
            for(int i = 0; i < V; ++i) {
                float q;
                gate(fr[e][i], s[e][i], q);
                if(!BWD) vr[e][i] = product(q, vr[e][i]);
            }
#pragma unroll
        for(int i = 0; i < V; ++i) {
            A[i] = s[0][i];
            H[i] = BWD ? s[0][i] * vr[0][i] : vr[0][i];
            least[i] = fminf(least[i], s[0][i]);
        }
#pragma unroll
        for(int e = 1; e < LT; ++e)
#pragma unroll
            for(int i = 0; i < V; ++i) {
                extend_run<BWD, false>(s[e][i], vr[e][i], A[i], H[i]);
                least[i] = fminf(least[i], s[e][i]);
            }
        if constexpr(!decltype(last)::value) fetch();
        add(std::false_type());
    };
    for(int64_t k = Pl::TT; k < p.L; k += Pl::TT) walk(std::false_type());
    walk(std::true_type());
    auto result = [&]() {
        if(at.tl != 0) return;
        float* const o = p.ws + (at.chunk * p.B + at.b) * p.C + at.c;
        store<V>(o, all, at.skip, false);
        store<V>(o + (int64_t)p.S * p.B * p.C, carry, at.skip, false);
    };
    if(any_bad(carry)) {  // (the same in every wave)
#pragma unroll
        for(int i = 0; i < V; ++i) {
            all[i] = 1.0f;
            carry[i] = 0.0f;
        }
        for(int64_t left = p.L; left > 0; left -= Pl::TT) {
#pragma unroll
            for(int i = 0; i < V; ++i) {
                A[i] = 1.0f;
                H[i] = 0.0f;
            }
#pragma unroll 1
            for(int e = 0; e < LT; ++e) {
                const int64_t g = at.chunk * p.L + left - Pl::TT + at.tl * LT + e, t = BWD ? p.T - 1 - g : g;
                float f[V], v[V];
                load<V>(p.f + (at.b * p.T + t) * p.ldf + at.c, f);
                load<V>((BWD ? p.dh : p.x) + (at.b * p.T + t) * ldv + at.c, v);
#pragma unroll
                for(int i = 0; i < V; ++i) {
                    float s, q;
                    gate(f[i], s, q);
                    extend_run<BWD, true>(s, BWD ? v[i] : product(q, v[i]), A[i], H[i]);
                }
            }
            add(std::true_type());
        }
        result();
        return;
    }
    // a shut gate leaves the product at 0
    bool zero = false;
#pragma unroll
    for(int i = 0; i < V; ++i) zero |= all[i] == 0.0f;
    if(__any(zero)) {  // (the same in every wave)
        __shared__ int shut_at[V * CL];
        if(threadIdx.x < V * CL) shut_at[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for(int i = 0; i < V; ++i)
            if(least[i] == 0.0f) shut_at[at.cl * V + i] = 1;
        __syncthreads();
#pragma unroll
        for(int i = 0; i < V; ++i)
            if(shut_at[at.cl * V + i]) all[i] = kShut;
    }
    result();
}

// token t of sequence b at V channels from c on, from `state` on: h and the new state, or
// the gradients and what is handed to the token before
template <int V, bool BWD>
__device__ __forceinline__ void token(const ScanParams& p, int64_t b, int64_t t, int64_t c, int skip,
                                      float (&state)[V]) {
    const int64_t row = b * p.T + t;
    float f[V], x[V];
    load<V>(p.f + row * p.ldf + c, f);
    load<V>(p.x + row * p.ldx + c, x);
    if constexpr(!BWD) {
#pragma unroll
        for(int i = 0; i < V; ++i) {
            float s, q;
            gate(f[i], s, q);
            state[i] = step<false, true>(state[i], s, product(q, x[i]));
        }
        store<V>(p.out + row * p.C + c, state, skip, false);
    } else {
        float dh[V], h[V], df[V], dx[V];
        load<V>(p.dh + row * p.C + c, dh);
#pragma unroll
        for(int i = 0; i < V; ++i) h[i] = 0.0f;
        if(t > 0) load<V>(p.h + (row - 1) * p.C + c, h);
        else if(p.h0) load<V>(p.h0 + b * p.C + c, h);
#pragma unroll
        for(int i = 0; i < V; ++i) {
            float s, q;
            gate(f[i], s, q);
            state[i] = gradients<true>(dh[i] + state[i], h[i], x[i], s, q, dx[i], df[i]);
        }
        if(p.df) store<V>(p.df + row * p.lddf + c, df, skip, p.flags & PK_ACCUM);
        if(p.dx) store<V>(p.dx + row * p.lddx + c, dx, skip, p.flags & PK_ACCUM2);
    }
}

// BIG: x and h, which only this pass of the backward reads, leave the caches to f and
// dh and to the next kernel (1x65536x512 backward 195 -> 167 us, 4x8192x1024 214 ->
// 200; now 164 and 194; tensors that fit the last-level cache are better read from there: 8x1024x768
// 30 against 37, 32x2048x256 68 against 75)
template <int V, int CL, bool BWD, bool BIG, bool ACC>
__global__ __launch_bounds__(kThreads) void scan_tiles(ScanParams p) {
    using Pl = Place<V, CL>;
    __shared__ alignas(16) float lds[2][kWaves][2][V * CL];
    const Pl at(p);
    if(!at.on) return;
    const int64_t g0 = at.chunk * p.L, g1 = min(p.T, g0 + p.L);
    const float* const f = p.f + at.b * p.T * p.ldf + at.c;
    const float* const x = p.x + at.b * p.T * p.ldx + at.c;
    const float* const h = BWD ? p.h + at.b * p.T * p.C + at.c : nullptr;
    const float* const dh = BWD ? p.dh + at.b * p.T * p.C + at.c : nullptr;
    const float* const h0 = p.h0 ? p.h0 + at.b * p.C + at.c : nullptr;
    float* const out = BWD ? nullptr : p.out + at.b * p.T * p.C + at.c;

    float carry[V], in[V];
#pragma unroll
    for(int i = 0; i < V; ++i) carry[i] = 0.0f;
    if(!BWD && h0) load<V>(h0, carry);
    int turn = 0;

    struct Regs {
        float f[LT][V], x[LT][V], h[BWD ? LT : 1][V], dh[BWD ? LT : 1][V];
    };
    Regs next;
    // a thread's steps from position `tile` on.  Where fewer than LT are left of the
    // sequence it has the last LT, the first `shift` of which are the threads'
    // before it and change nothing here: no load is out of range, and none is
    // conditional.
    auto start = [&](int64_t tile) { return min(tile + at.tl * LT, p.T - LT); };
    auto fetch = [&](int64_t tile) {
        const int64_t g = start(tile), t0 = BWD ? p.T - 1 - g : g;
        const float *fp = f + t0 * p.ldf, *xp = x + t0 * p.ldx, *dp = nullptr, *hp = nullptr;
        if constexpr(BWD) {
            dp = dh + t0 * p.C;
            hp = h + (t0 - 1) * p.C;
        }
#pragma unroll
        for(int e = 0; e < LT; ++e) {
            load<V>(fp, next.f[e]);
            load<V, BIG>(xp, next.x[e]);
            fp += BWD ? -p.ldf : p.ldf;
            xp += BWD ? -p.ldx : p.ldx;
            if constexpr(BWD) {
                // (before the first token: h0, or a zero put in later)
                if(e == LT - 1 && t0 == LT - 1) hp = h0 ? h0 : dp;
                load<V>(dp, next.dh[e]);
                load<V, BIG>(hp, next.h[e]);
                dp -= p.C;
                hp -= p.C;
            }
        }
    };
    fetch(g0);
    if(at.chunk > 0) {
        // the value behind the chunks before this one
        float A[V], H[V], given[V];
#pragma unroll
        for(int i = 0; i < V; ++i) given[i] = carry[i];
        auto gather = [&](auto bad) {
            constexpr bool BAD = decltype(bad)::value;
            const int64_t m = (at.chunk + Pl::TL - 1) / Pl::TL;
#pragma unroll
            for(int i = 0; i < V; ++i) {
                A[i] = 1.0f;
                H[i] = 0.0f;
                carry[i] = given[i];
            }
            for(int64_t k = at.tl * m; k < min(at.tl * m + m, at.chunk); ++k) {
                const float* o = p.ws + (k * p.B + at.b) * p.C + at.c;
                float a[V], e[V];
                load<V>(o, a);
                load<V>(o + (int64_t)p.S * p.B * p.C, e);
#pragma unroll
                for(int i = 0; i < V; ++i) {
                    compose<BAD>(a[i], e[i], A[i], H[i]);
                    A[i] = a[i];
                    H[i] = e[i];
                }
            }
            through<V, CL, BAD>(A, H, carry, in, lds, turn);
            turn ^= 1;
        };
        gather(std::false_type());
        if(any_bad(carry)) gather(std::true_type());  // (the same in every wave)
    }
    // where the bad form would start: at the first tile, or, where the stores add to what is
    // there and cannot be done twice, at the tile that has the first bad values
    int64_t from = g0;
    float reached[V];
#pragma unroll
    for(int i = 0; i < V; ++i) reached[i] = carry[i];
    // (the last tile apart: were its fetch a branch's, the waits for one tile's values
    // would be for the next one's as well)
    auto walk = [&](int64_t tile, auto last) {
        constexpr bool LAST = decltype(last)::value;
        Regs r = next;
        if constexpr(!LAST) {
            fetch(tile + Pl::TT);
            __builtin_amdgcn_sched_barrier(0);
        }
        const int64_t first = start(tile);
        const int shift = (int)min(tile + at.tl * LT - first, (int64_t)LT);
        const bool whole = !LAST || tile + Pl::TT <= g1;
        float s[LT][V], q[LT][V], A[V], H[V];
#pragma unroll
        for(int e = 0; e < LT; ++e)
#pragma unroll
            for(int i = 0; i < V; ++i) {
                gate(r.f[e][i], s[e][i], q[e][i]);
                if(!BWD) r.x[e][i] = product(q[e][i], r.x[e][i]);
            }
        if(!whole) {
#pragma unroll
            for(int e = 0; e < LT; ++e)
#pragma unroll
                for(int i = 0; i < V; ++i)
                    if(e < shift) {  // a step that changes nothing
                        s[e][i] = 1.0f;
                        if(BWD) r.dh[BWD ? e : 0][i] = 0.0f;
                        else r.x[e][i] = 0.0f;
                    }
        }
#pragma unroll
        for(int i = 0; i < V; ++i) {
            A[i] = s[0][i];
            H[i] = BWD ? s[0][i] * r.dh[0][i] : r.x[0][i];
        }
#pragma unroll
        for(int e = 1; e < LT; ++e)
#pragma unroll
            for(int i = 0; i < V; ++i)
                extend_run<BWD, false>(s[e][i], BWD ? r.dh[BWD ? e : 0][i] : r.x[e][i], A[i], H[i]);
        through<V, CL, false>(A, H, carry, in, lds, turn);
        turn ^= 1;
        if constexpr(ACC) {
            if(any_bad(carry)) return false;
            from = tile + Pl::TT;
#pragma unroll
            for(int i = 0; i < V; ++i) reached[i] = carry[i];
        }
#pragma unroll
        for(int e = 0; e < LT; ++e) {
            const int64_t g = first + e, t = BWD ? p.T - 1 - g : g;
            if(!whole && e < shift) continue;
            if constexpr(!BWD) {
#pragma unroll
                for(int i = 0; i < V; ++i) in[i] = step<false, false>(in[i], s[e][i], r.x[e][i]);
                store<V>(out + t * p.C, in, at.skip, false);
            } else {
                float df[V], dx[V];
#pragma unroll
                for(int i = 0; i < V; ++i) {
                    if(e == LT - 1 && t == 0 && !h0) r.h[e][i] = 0.0f;
                    in[i] = gradients<false>(r.dh[e][i] + in[i], r.h[e][i], r.x[e][i], s[e][i], q[e][i], dx[i],
                                             df[i]);
                }
                const int64_t row = at.b * p.T + t;
                if(p.df) store<V>(p.df + row * p.lddf + at.c, df, at.skip, ACC && (p.flags & PK_ACCUM));
                if(p.dx) store<V>(p.dx + row * p.lddx + at.c, dx, at.skip, ACC && (p.flags & PK_ACCUM2));
            }
        }
        return true;
    };
    int64_t tile = g0;
    while(tile + Pl::TT < g1 && walk(tile, std::false_type())) tile += Pl::TT;
    if(tile + Pl::TT >= g1) walk(tile, std::true_type());
    const bool again = any_bad(carry);  // (the same in every wave)
    if(again) {
#pragma unroll
        for(int i = 0; i < V; ++i) carry[i] = reached[i];
    }
    // (each step's values loaded anew: what the tiles have in flight fills the registers)
    for(tile = from; again && tile < g1; tile += Pl::TT) {
        const int64_t end = min(tile + (at.tl + 1) * LT, g1);
        float A[V], H[V];
#pragma unroll
        for(int i = 0; i < V; ++i) {
            A[i] = 1.0f;
            H[i] = 0.0f;
        }
#pragma unroll 1
        for(int64_t g = tile + at.tl * LT; g < end; ++g) {
            const int64_t t = BWD ? p.T - 1 - g : g;
            float fe[V], ve[V];
            load<V>(f + t * p.ldf, fe);
            load<V>(BWD ? dh + t * p.C : x + t * p.ldx, ve);
#pragma unroll
            for(int i = 0; i < V; ++i) {
                float s, q;
                gate(fe[i], s, q);
                extend_run<BWD, true>(s, BWD ? ve[i] : product(q, ve[i]), A[i], H[i]);
            }
        }
        through<V, CL, true>(A, H, carry, in, lds, turn);
        turn ^= 1;
#pragma unroll 1
        for(int64_t g = tile + at.tl * LT; g < end; ++g)
            token<V, BWD>(p, at.b, BWD ? p.T - 1 - g : g, at.c, at.skip, in);
    }
    if(BWD && p.dh0 && at.tl == 0 && g1 == p.T)
        store<V>(p.dh0 + at.b * p.C + at.c, carry, at.skip, p.flags & PK_ACCUM3);
}

// a few tokens of many sequences: a thread to V channels, token after token
template <int V, bool BWD>
__global__ __launch_bounds__(kThreads) void scan_serial(ScanParams p) {
    const int64_t per = (p.C + V - 1) / V, id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if(id >= p.B * per) return;
    const int64_t b = id / per;
    int64_t c = (id % per) * V;
    int skip = 0;
    if(c + V > p.C) {
        skip = (int)(c + V - p.C);
        c = p.C - V;
    }
    float state[V];
#pragma unroll
    for(int i = 0; i < V; ++i) state[i] = 0.0f;
    if(!BWD && p.h0) load<V>(p.h0 + b * p.C + c, state);
    for(int64_t g = 0; g < p.T; ++g) token<V, BWD>(p, b, BWD ? p.T - 1 - g : g, c, skip, state);
    if(BWD && p.dh0) store<V>(p.dh0 + b * p.C + c, state, skip, p.flags & PK_ACCUM3);
}

// How a shape is split: token after token (lanes 0), or groups of `lanes` lanes along
// the channels (4 channels each, 1 below 4) and S chunks of L steps.  Times are
// forward + backward, us, from graphs of 20 calls.
struct Plan {
    int lanes, S;
    int64_t L;
};

Plan plan_of(int64_t B, int64_t T, int64_t C) {
    const int V = C < 4 ? 1 : 4;
    auto groups = [&](int lanes) { return B * ((C + V * lanes - 1) / (V * lanes)); };
    auto steps = [](int lanes) { return (int64_t)(kThreads / lanes * LT); };  // of a tile
    // Token after token where there are few, and up to some tens of them where the
    // sequences are so many that tiles mostly empty fill the chip more than once:
    // 64x8x768 11.6, tiles 14.7; 128x9x768 12.9, 23.4; 128x16x768 22.7, 23.6; 512x32x768
    // 72.8, 90.7 (but 32x12x768 15.2, tiles 11.1; 128x24x768 34.6, 27.7; 512x64x768 176, 157)
    if(T <= 8 || (T <= 16 && groups(16) >= 1024) || (T <= 40 && groups(16) >= 4096)) return {0, 1, T};
    // One chunk, which reads everything once, where it fills most of the chip, with
    // the widest rows that do: 8x1024x768 8 lanes 46.6, 4 lanes 52.8, 2 chunks 59.1;
    // 4x2000x768 4 lanes 53.5, 16 chunks 62.0; 16x512x512 8 lanes 29.9, 2 chunks 37.7
    for(const int lanes : {16, 8, 4})
        if(groups(lanes) >= 192) return {lanes, 1, T};
    // ... and where it is a tile or two long: 8x64x768 9.9 (8 lanes 10.1), 1x300x2048
    // 4 lanes 14.4, 3 chunks 19.1
    for(const int lanes : {16, 8})
        if(T <= steps(lanes)) return {lanes, 1, T};
    if(T <= 2 * steps(4)) return {4, 1, T};
    // Chunks.  Few tiles in all: one to a chunk, narrow ones, so that the chunks to
    // gather the state from are few (3x1001x333 4 lanes 24.3, 16 lanes 23.5, one chunk
    // 28.2; 1x9000x20 23.4, 8 lanes 27.8).  Else 512 workgroups: rows of 128 bytes (1x32768x256 8
    // lanes 73.5, 16 lanes 101, 4 lanes 82.5; 1x4096x768 34.5, 41.9, 36.1), of 64 where
    // few channels would leave chunks many (1x20000x64 40.5, 8 lanes 42.9), of 256
    // beyond what the last-level cache holds (1x65536x512 260, 8 lanes 288; both in turn
    // 286, with half as many workgroups 297)
    const int64_t tiles = groups(8) * ((T + steps(8) - 1) / steps(8));
    const int lanes = tiles <= 384 || groups(8) < 4 ? 4 : tiles >= 8192 && groups(16) >= 8 ? 16 : 8;
    const int64_t want = tiles <= 384 ? T : (512 + groups(lanes) - 1) / groups(lanes);
    const int64_t per = ((T + want - 1) / want + steps(lanes) - 1) / steps(lanes);
    const int64_t L = per * steps(lanes);
    return {lanes, (int)((T + L - 1) / L), L};
}

template <int V, int CL, bool BWD>
void launch(ScanParams& p, const Plan& plan, hipStream_t st) {
    p.groups = (int)((p.C + V * CL - 1) / (V * CL));
    const unsigned grid = (unsigned)((p.B * p.groups + 7) / 8 * 8);
    if(plan.S > 1) scan_chunks<V, CL, BWD><<<dim3(grid, plan.S - 1), kThreads, 0, st>>>(p);
    auto tiles = [&](auto big, auto acc) {
        scan_tiles<V, CL, BWD, decltype(big)::value, decltype(acc)::value>
            <<<dim3(grid, plan.S), kThreads, 0, st>>>(p);
    };
    auto with = [&](auto big) {
        if constexpr(BWD)
            if(p.flags & (PK_ACCUM | PK_ACCUM2)) return tiles(big, std::true_type());
        tiles(big, std::false_type());
    };
    // (values of a tensor: between 17 and 33 million)
    if constexpr(BWD)
        if(p.B * p.T * p.C >= (int64_t)24 << 20) return with(std::true_type());
    with(std::false_type());
}

template <bool BWD>
int run(const char* who, ScanParams& p, void* workspace, size_t workspace_bytes, pk_stream_t stream) {
    const Plan plan = plan_of(p.B, p.T, p.C);
    const size_t need = pk_gated_scan_workspace(p.B, p.T, p.C);
    if(need && (!workspace || workspace_bytes < need)) return pk::fail("%s: workspace needs %zu bytes", who, need);
    hipStream_t st = pk::as_stream(stream);
    p.ws = static_cast<float*>(workspace);
    p.S = plan.S;
    p.L = plan.L;
    if(plan.lanes == 0) {
        const int64_t V = p.C < 4 ? 1 : 4;
        const unsigned grid = (unsigned)((p.B * ((p.C + V - 1) / V) + kThreads - 1) / kThreads);
        if(V == 1) scan_serial<1, BWD><<<grid, kThreads, 0, st>>>(p);
        else scan_serial<4, BWD><<<grid, kThreads, 0, st>>>(p);
    } else {
        auto with = [&](auto v) {
            constexpr int V = decltype(v)::value;
            if(plan.lanes == 16) launch<V, 16, BWD>(p, plan, st);
            else if(plan.lanes == 8) launch<V, 8, BWD>(p, plan, st);
            else launch<V, 4, BWD>(p, plan, st);
        };
        if(p.C < 4) with(std::integral_constant<int, 1>());
        else with(std::integral_constant<int, 4>());
    }
    return pk::launch_status(who);
}

int check(const char* who, int64_t B, int64_t T, int64_t C, const float* f, int64_t ldf,
          const float* x, int64_t ldx) {
    if(B < 0 || T < 0 || C < 0) return pk::fail("%s: negative size", who);
    if(B > INT32_MAX || T > INT32_MAX || C > INT32_MAX || B * T > INT32_MAX)
        return pk::fail("%s: B*T rows too many for one call", who);
    if(B == 0 || T == 0 || C == 0) return PK_OK;
    // (4 channels to a thread, and 256 threads to a workgroup of at least a sequence)
    const Plan plan = plan_of(B, T, C);
    const int64_t V = C < 4 ? 1 : 4, lanes = plan.lanes ? plan.lanes : 1,
                  groups = (C + V * lanes - 1) / (V * lanes);
    if(groups > (((int64_t)1 << 32) / (plan.lanes ? kThreads : 1) - 2 * kThreads) / B)
        return pk::fail("%s: B*C channels too many for one launch", who);
    if(!f || !x) return pk::fail("%s: NULL f or x", who);
    if(ldf < C || ldx < C) return pk::fail("%s: row stride < C", who);
    return PK_OK;
}

}  // namespace

extern "C" size_t pk_gated_scan_workspace(int64_t B, int64_t T, int64_t C) {
    if(B <= 0 || T <= 0 || C <= 0) return 0;
    const Plan plan = plan_of(B, T, C);
    return plan.S > 1 ? (size_t)plan.S * (size_t)B * (size_t)C * 2 * sizeof(float) : 0;
}

extern "C" int pk_gated_scan_fwd_f32(int64_t B, int64_t T, int64_t C, const float* f, int64_t ldf,
                                     const float* x, int64_t ldx, const float* h0, float* h,
                                     void* workspace, size_t workspace_bytes, pk_stream_t stream) {
    if(int st = check("pk_gated_scan_fwd_f32", B, T, C, f, ldf, x, ldx)) return st;
    if(B == 0 || T == 0 || C == 0) return PK_OK;
    if(!h) return pk::fail("pk_gated_scan_fwd_f32: NULL h");
    ScanParams p = {};
    p.B = B;
    p.T = T;
    p.C = C;
    p.f = f;
    p.ldf = ldf;
    p.x = x;
    p.ldx = ldx;
    p.h0 = h0;
    p.out = h;
    return run<false>("pk_gated_scan_fwd_f32", p, workspace, workspace_bytes, stream);
}

extern "C" int pk_gated_scan_bwd_f32(int64_t B, int64_t T, int64_t C, const float* f, int64_t ldf,
                                     const float* x, int64_t ldx, const float* h0, const float* h,
                                     const float* dh, float* df, int64_t lddf, float* dx,
                                     int64_t lddx, float* dh0, int flags, void* workspace,
                                     size_t workspace_bytes, pk_stream_t stream) {
    if(int st = check("pk_gated_scan_bwd_f32", B, T, C, f, ldf, x, ldx)) return st;
    if(B == 0 || C == 0) return PK_OK;
    if(T == 0)
        return dh0 && !(flags & PK_ACCUM3) ? pk_fill_f32(B * C, 0.0f, dh0, stream) : PK_OK;
    if(!h || !dh) return pk::fail("pk_gated_scan_bwd_f32: NULL h or dh");
    if((df && lddf < C) || (dx && lddx < C))
        return pk::fail("pk_gated_scan_bwd_f32: row stride of a gradient < C");
    ScanParams p = {};
    p.B = B;
    p.T = T;
    p.C = C;
    p.f = f;
    p.ldf = ldf;
    p.x = x;
    p.ldx = ldx;
    p.h0 = h0;
    p.h = h;
    p.dh = dh;
    p.df = df;
    p.lddf = lddf;
    p.dx = dx;
    p.lddx = lddx;
    p.dh0 = dh0;
    p.flags = flags;
    return run<true>("pk_gated_scan_bwd_f32", p, workspace, workspace_bytes, stream);
}
