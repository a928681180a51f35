// pico_amd/csrc/kv_cache.hip -- new tokens into a paged cache of keys and values: the keys
// turned by their positions, both rounded to e4m3 with a power of two for each page and
// head, and the queries turned along in the same launch.
#include "paged.h"
#include "rope.h"

namespace {

using namespace pk;

__device__ __forceinline__ float held448(float x) {
    return x != x ? x : fminf(fmaxf(x, -448.0f), 448.0f);
}
__device__ __forceinline__ uint32_t codes(float a, float b, float c, float d) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(held448(a), held448(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(held448(c), held448(d), lo, true);
}
__device__ __forceinline__ uint8_t code_again(uint8_t c, float shift) {
    return (uint8_t)codes(__builtin_amdgcn_cvt_f32_fp8(c, 0) * shift, 0.0f, 0.0f, 0.0f);
}

constexpr int kThreads = 256;

struct AppendArgs {
    PkKvCache c;
    int N, hp;
    unsigned halves;  // workgroups for k, and as many for v: pages that may be written to, times heads
    const float *k, *v;
    int64_t ldk, ldv;
    RopeArgs rope;
    TurnArgs q;
    int q_tokens, q_vec;
};

// one page's new tokens of one head's keys or values.  A page's head is written to by one
// workgroup, which turns the new values on their way to LDS, finds the largest of them, and
// writes their codes from there, in words of 4: k's rows are the tokens', v's the columns.
template <bool IS_V>
__device__ __forceinline__ void append_page(const AppendArgs& a, unsigned task, int h, float* tile,
                                            float* red) {
    const PkKvCache& c = a.c;
    const int page = (int)c.page, hd = (int)c.hd, hp = a.hp;
    int nth, b;
    Seq s;
    if(!locate(
           c, a.N, [&](const Seq& t) { return t.end > t.past ? (t.end - 1) / page - t.past / page + 1 : 0; },
           [&](int) { return (int)task; }, nth, b, s))
        return;
    const int index = s.past / page + nth;
    const int pid = c.table[(int64_t)b * c.width + index];
    if(pid < 0 || pid >= c.pages) return;
    // the page's new tokens: slots [s0, s1), the first of them in row `row`
    const int p0 = s.past > index * page ? s.past : index * page;
    const int s0 = p0 - index * page;
    const int s1 = s.end - index * page < page ? s.end - index * page : page;
    const int n = s1 - s0;
    const int64_t ld = IS_V ? a.ldv : a.ldk;
    const float* src = (IS_V ? a.v : a.k) + (int64_t)(s.row + p0 - s.past) * ld + (int64_t)h * hd;
    const int64_t at = (int64_t)pid * c.kv_heads + h;
    uint8_t* exps = (IS_V ? c.v_exp : c.k_exp) + at;
    uint8_t* out = (IS_V ? c.v : c.k) + at * (int64_t)(hp * page);
    const int old = s0 ? held((int)*exps - 127, kExpMin, kExpMax) : kExpMin;

    const int half = IS_V ? 0 : a.rope.half, pairs = hp / 2, apart = pairs - half;
    const int stride = IS_V ? page + 1 : hp;
    float amax = 0.0f;
    for(int e = threadIdx.x; e < n * pairs; e += kThreads) {
        const int t = e / pairs, p = e - t * pairs;
        const bool turned = p < half;
        const int d1 = turned ? (a.rope.interleaved ? 2 * p : p) : half + p;
        const int d2 = turned ? (a.rope.interleaved ? d1 + 1 : p + half) : half + p + apart;
        const float* r = src + t * ld;
        float x1 = d1 < hd ? r[d1] : 0.0f, x2 = d2 < hd ? r[d2] : 0.0f;
        if(turned) {
            float co, si;
            rope_angle(p0 + t, a.rope.freqs[p], a.rope.magnitude, co, si);
            rope_turn(x1, x2, co, si);
        }
        const float m1 = fabsf(x1), m2 = fabsf(x2);
        if(m1 <= 3.402823466e38f) amax = fmaxf(amax, m1);  // (not infinities or NaN)
        if(m2 <= 3.402823466e38f) amax = fmaxf(amax, m2);
        // (v's columns are at their slots, so that words of 4 tokens line up)
        tile[IS_V ? d1 * stride + s0 + t : t * stride + d1] = x1;
        tile[IS_V ? d2 * stride + s0 + t : t * stride + d2] = x2;
    }
    amax = block_max<kThreads / kWave>(amax, red);
    const int fresh = block_exponent(amax), e = fresh > old ? fresh : old;
    const float scale = ldexpf(1.0f, -e);
    if(!IS_V) {
        for(int i = 4 * (int)threadIdx.x; i < n * hp; i += 4 * kThreads) {
            const f32x4 x = *(const f32x4*)(tile + i) * scale;
            *(uint32_t*)(out + s0 * hp + i) = codes(x[0], x[1], x[2], x[3]);
        }
    } else {
        // words of tokens that are all new, single bytes at the ends
        const int w0 = s0 / 4, words = (s1 + 3) / 4 - w0;
        for(int i = threadIdx.x; i < hd * words; i += kThreads) {
            const int d = i / words, t = 4 * (w0 + i - d * words);
            const float* x = tile + d * stride + t;
            float y[4];
#pragma unroll
            for(int q = 0; q < 4; ++q) y[q] = t + q >= s0 && t + q < s1 ? x[q] * scale : 0.0f;
            const uint32_t w = codes(y[0], y[1], y[2], y[3]);
            uint8_t* to = out + d * page + t;
            if(t >= s0 && t + 4 <= s1) {
                *(uint32_t*)to = w;
            } else {
#pragma unroll
                for(int q = 0; q < 4; ++q)
                    if(t + q >= s0 && t + q < s1) to[q] = (uint8_t)(w >> (8 * q));
            }
        }
    }
    if(e > old && s0) {  // what the page held, at its new scale
        const float shift = ldexpf(1.0f, old - e);
        for(int i = threadIdx.x; i < s0 * hd; i += kThreads) {
            const int j = IS_V ? i / s0 * page + i % s0 : i / hd * hp + i % hd;
            out[j] = code_again(out[j], shift);
        }
    }
    // (every thread has read the old one: block_max waited for all)
    if(threadIdx.x == 0) *exps = (uint8_t)(e + 127);
}

__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
    extern __shared__ __align__(16) float tile[];
    __shared__ float red[kThreads / kWave];
    const unsigned block = blockIdx.x, heads = (unsigned)a.c.kv_heads;
    if(block < a.halves) return append_page<false>(a, block / heads, (int)(block % heads), tile, red);
    if(block < 2 * a.halves) {
        const unsigned i = block - a.halves;
        return append_page<true>(a, i / heads, (int)(i % heads), tile, red);
    }
    // queries: rows [t0, t0 + tokens), each at the position of its token
    const int t0 = (int)(block - 2 * a.halves) * a.q_tokens;
    const int tokens = a.N - t0 < a.q_tokens ? a.N - t0 : a.q_tokens;
    __shared__ int place[8];
    __shared__ __align__(16) float tc[kTurnTable], ts[kTurnTable];
    const int lane = threadIdx.x % kWave, B = (int)a.c.B;
    for(int t = threadIdx.x / kWave; t < tokens; t += kThreads / kWave) {
        // the last sequence that begins at this row or before, and whether the row is in it
        int before = 0;
        for(int base = 0; base < B; base += kWave) {
            const int b = base + lane;
            before += __popcll(__ballot(b < B && a.c.offsets[b] <= t0 + t));
        }
        if(lane == 0) {
            int pos = -1;
            if(before > 0) {
                const Seq s = sequence(a.c, a.N, before - 1);
                if(t0 + t >= s.row && t0 + t < s.row + s.n) pos = s.past + t0 + t - s.row;
            }
            place[t] = pos;
        }
    }
    __syncthreads();
    auto where = [&](int t, int& pos) {
        pos = place[t];
        return pos >= 0;
    };
    if(a.rope.interleaved)
        a.q_vec ? turn_rows<4, true>(a.q, a.rope, t0, tokens, where, tc, ts)
                : turn_rows<1, true>(a.q, a.rope, t0, tokens, where, tc, ts);
    else
        a.q_vec ? turn_rows<4, false>(a.q, a.rope, t0, tokens, where, tc, ts)
                : turn_rows<1, false>(a.q, a.rope, t0, tokens, where, tc, ts);
}

}  // namespace

extern "C" int64_t pk_kv_head_size(int64_t hd) { return head_size(hd); }

extern "C" int pk_kv_append_f32(const PkKvCache* cache, int64_t N, const float* k, int64_t ldk,
                                const float* v, int64_t ldv, const PkRope* rope, int64_t H,
                                const float* q, int64_t ldq, float* q_out, int64_t ldqo,
                                pk_stream_t stream) {
    if(int st = check_cache("pk_kv_append_f32", cache, N)) return st;
    const int64_t hd = cache->hd, width = cache->kv_heads * hd;
    if(rope && !rope_ok(rope, hd))
        return fail("pk_kv_append_f32: rope must have an even rot of 0 to hd, and its frequencies");
    if(N == 0 || cache->B == 0) return PK_OK;
    if(!k || !v) return fail("pk_kv_append_f32: NULL keys or values");
    if(ldk < width || ldv < width)
        return fail("pk_kv_append_f32: row strides must be at least kv_heads*hd = %lld", (long long)width);
    if(q && (!q_out || H < 1 || H > (1 << 20) / hd || ldq < H * hd || ldqo < H * hd))
        return fail("pk_kv_append_f32: q needs q_out, 1 <= H, H*hd <= 2^20 and row strides of H*hd");
    AppendArgs a = {};
    a.c = *cache;
    a.N = (int)N;
    a.hp = head_size(hd);
    a.k = k;
    a.v = v;
    a.ldk = ldk;
    a.ldv = ldv;
    a.rope = rope_args(rope);
    const int64_t page = cache->page, kvh = cache->kv_heads;
    // a sequence with n > 0 new tokens writes to at most n pages, and n / page + 2
    const int64_t tasks = N < N / page + 2 * cache->B ? N : N / page + 2 * cache->B;
    int64_t blocks = 2 * tasks * kvh;
    if(!grid_fits(blocks + N, kThreads))
        return fail("pk_kv_append_f32: too many pages and heads for one launch");
    a.halves = (unsigned)(tasks * kvh);
    if(q) {
        a.q_vec = turn_args(a.q, a.rope, H, hd, q, ldq, q_out, ldqo, 0);
        a.q_tokens = turn_tokens(N, H, a.rope.half);
        blocks += (N + a.q_tokens - 1) / a.q_tokens;
    }
    append_kernel<<<(unsigned)blocks, kThreads, sizeof(float) * a.hp * (page + 1), as_stream(stream)>>>(a);
    return launch_status("pk_kv_append_f32");
}
