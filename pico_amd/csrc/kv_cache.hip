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

struct AppendArgs {
    PkKvCache c;
    int N, hp;
    int cap;          // tokens of a page that the LDS tile holds
    unsigned halves;  // workgroups for k, and as many for v: pages that may be written to, times heads
    const float *k, *v;
    int64_t ldk, ldv;
    RopeArgs rope;
    TurnArgs q;  // of the heads that a workgroup turns
    int q_tokens, q_parts, q_heads, q_even;
    unsigned q_blocks;
};

// One page's new tokens of one head's keys or values.  A page's head is written to by one
// workgroup, which turns the new values on their way to LDS, finds the largest of them, and
// writes their codes from there, in words of 4: k's rows are the tokens', v's the columns.
// Where the tile holds fewer tokens than are new, the values are read twice.
// Prompts are bound by HBM: 12288 tokens of 8 heads of 128, with 32 heads of queries, 108 us
// (4.9 TB/s).  Single tokens are bound by the way to the page, lengths, its number, its
// power: 64 tokens 6 us, where no page's power grows.  Where one does, what the page held is
// rounded again a byte at a time: with 32 tokens of 128 values held, 16 us more for one page's
// head, 21 for all.
template <bool IS_V, int THREADS, int U>
__device__ __forceinline__ void append_page(const AppendArgs& a, unsigned task, int h, float* tile,
                                            float* red) {
    const PkKvCache& c = a.c;
    const int page = (int)c.page, hd = (int)c.hd, hp = a.hp, shift = __builtin_ctz(page);
    int nth, b;
    Seq s;
    if(!locate(
           c, a.N,
           [&](const Seq& t) { return t.end > t.past ? ((t.end - 1) >> shift) - (t.past >> shift) + 1 : 0; },
           [&](int) { return (int)task; }, nth, b, s))
        return;
    const int index = (s.past >> shift) + nth;
    const int name = c.table[(int64_t)b * c.width + index];
    // the page's new tokens: slots [s0, s1), the first of them at position p0
    const int p0 = s.past > index * page ? s.past : index * page;
    const int s0 = p0 - index * page;
    const int s1 = s.end - index * page < page ? s.end - index * page : page;
    const int64_t ld = IS_V ? a.ldv : a.ldk;
    const float* src = (IS_V ? a.v : a.k) + (int64_t)(s.row + p0 - s.past) * ld + (int64_t)h * hd;

    const int half = IS_V ? 0 : a.rope.half, pairs = hp / 2, apart = pairs - half;
    const int stride = IS_V ? a.cap + 5 : hp;
    // a thread has one pair of a head (one of each 64, where heads have more and threads are
    // few), of every `abreast`th token, U of them in flight
    const int across = pairs < THREADS ? pairs : THREADS, abreast = THREADS / across;
    const int my_t = (int)threadIdx.x / across, my_p = (int)threadIdx.x - my_t * across;
    struct Pair {
        int d1, d2;
    };
    auto pair_of = [&](int p) {
        const bool turned = p < half;
        const int d1 = turned ? (a.rope.interleaved ? 2 * p : p) : half + p;
        return Pair{d1, turned ? (a.rope.interleaved ? d1 + 1 : p + half) : half + p + apart};
    };
    float x1[U], x2[U], amax = 0.0f;
    auto load = [&](const Pair& q, int t, int end) {
#pragma unroll
        for(int k = 0; k < U; ++k) {
            const float* r = src + (int64_t)(t + k * abreast) * ld;
            const bool there = t + k * abreast < end;
            x1[k] = there && q.d1 < hd ? r[q.d1] : 0.0f;
            x2[k] = there && q.d2 < hd ? r[q.d2] : 0.0f;
        }
    };
    const int n = s1 - s0, parts = (n + a.cap - 1) / a.cap;
    if(my_t < abreast) load(pair_of(my_p), my_t, n < a.cap ? n : a.cap);  // (beside the page's number)
    if(name < 0 || name >= c.pages) return;
    const int64_t at = (int64_t)name * c.kv_heads + h;
    uint8_t* exps = (IS_V ? c.v_exp : c.k_exp) + at;
    uint8_t* out = (IS_V ? c.v : c.k) + at * (int64_t)(hp * page);
    const int old = s0 ? exponent_byte(*exps) - 127 : kExpMin;

    int e = 0;
    float scale = 1.0f;
    for(int i = 0; i < (parts == 1 ? 1 : 2 * parts); ++i) {
        const int t0 = (i < parts ? i : i - parts) * a.cap, tokens = n - t0 < a.cap ? n - t0 : a.cap;
        const int c0 = s0 + t0, c1 = c0 + tokens;  // slots
        if(i) __syncthreads();
        for(int p = my_t < abreast ? my_p : pairs; p < pairs; p += across) {
            const Pair q = pair_of(p);
            // the angle of the next token `abreast` on by the angles' sum, in 64 bits too: 64 of
            // these are off by 2^-46, and their rounding to 32 bits hardly ever by its last one
            double c = 0.0, s = 0.0, cs = 0.0, ss = 0.0;
            if(p < half) {
                rope_turns(p0 + t0 + my_t, a.rope.freqs[p], c, s);
                if(my_t + abreast < tokens) rope_turns(abreast, a.rope.freqs[p], cs, ss);
            }
            for(int t = my_t; t < tokens; t += U * abreast) {
                if(i || t > my_t || p > my_p) load(q, t0 + t, t0 + tokens);
#pragma unroll
                for(int k = 0; k < U; ++k) {
                    const int now = t + k * abreast;
                    if(now >= tokens) break;
                    if(p < half) {
                        rope_turn(x1[k], x2[k], (float)(c * a.rope.magnitude), (float)(s * a.rope.magnitude));
                        const double next = c * cs - s * ss;
                        s = s * cs + c * ss;
                        c = next;
                    }
                    const float m1 = fabsf(x1[k]), m2 = fabsf(x2[k]);
                    if(m1 <= 3.402823466e38f) amax = fmaxf(amax, m1);  // (not infinities or NaN)
                    if(m2 <= 3.402823466e38f) amax = fmaxf(amax, m2);
                    // (v's columns are at their slots from a multiple of 4 on, so that words line up)
                    tile[IS_V ? q.d1 * stride + c0 % 4 + now : now * stride + q.d1] = x1[k];
                    tile[IS_V ? q.d2 * stride + c0 % 4 + now : now * stride + q.d2] = x2[k];
                }
            }
        }
        if(i == parts - 1) {
            amax = block_max<THREADS / kWave>(amax, red);
            const int fresh = block_exponent(amax);
            e = fresh > old ? fresh : old;
            scale = ldexpf(1.0f, -e);
        }
        if(parts > 1 && i < parts) continue;  // (the page's largest is not known yet)
        __syncthreads();
        if(!IS_V) {
            for(int j = 4 * (int)threadIdx.x; j < tokens * hp; j += 4 * THREADS) {
                const f32x4 x = *(const f32x4*)(tile + j) * scale;
                *(uint32_t*)(out + c0 * hp + j) = codes(x[0], x[1], x[2], x[3]);
            }
            continue;
        }
        // words of tokens that are all new, single bytes at the ends
        const int w0 = c0 / 4, words = (c1 + 3) / 4 - w0;
        for(int j = threadIdx.x; j < hd * words; j += THREADS) {
            const int d = j / words, w = j - d * words, t = 4 * (w0 + w);
            const float* x = tile + d * stride + 4 * w;
            float y[4];
#pragma unroll
            for(int q = 0; q < 4; ++q) y[q] = t + q >= c0 && t + q < c1 ? x[q] * scale : 0.0f;
            const uint32_t word = codes(y[0], y[1], y[2], y[3]);
            uint8_t* to = out + d * page + t;
            if(t >= c0 && t + 4 <= c1) {
                *(uint32_t*)to = word;
            } else {
#pragma unroll
                for(int q = 0; q < 4; ++q)
                    if(t + q >= c0 && t + q < c1) to[q] = (uint8_t)(word >> (8 * q));
            }
        }
    }
    if(e > old && s0) {  // what the page held, at its new scale
        const float to = ldexpf(1.0f, old - e);
        for(int i = threadIdx.x; i < s0 * hd; i += THREADS) {
            const int j = IS_V ? i / s0 * page + i % s0 : i / hd * hp + i % hd;
            out[j] = code_again(out[j], to);
        }
    }
    // (every thread has read the old one: the exchange of amax waited for all)
    if(threadIdx.x == 0) *exps = (uint8_t)(e + 127);
}

// the queries of some tokens and heads, each at the position of its token
template <int THREADS>
__device__ __forceinline__ void turn_queries(const AppendArgs& a, unsigned block) {
    __shared__ int place[8];
    __shared__ __align__(16) float tc[kTurnTable], ts[kTurnTable];
    const int t0 = (int)(block / a.q_parts) * a.q_tokens, h0 = (int)(block % a.q_parts) * a.q_heads;
    const int tokens = a.N - t0 < a.q_tokens ? a.N - t0 : a.q_tokens;
    const int lane = threadIdx.x % kWave, B = (int)a.c.B;
    for(int t = threadIdx.x / kWave; t < tokens; t += THREADS / kWave) {
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
    TurnArgs q = a.q;  // (the last part may have fewer heads)
    q.x += h0 * q.hd;
    q.y += h0 * q.hd;
    const int heads = q.H - h0 < a.q_heads ? q.H - h0 : a.q_heads;
    if(a.rope.interleaved)
        a.q_even ? turn_rows<true, true>(q, a.rope, t0, tokens, heads, where, tc, ts)
                : turn_rows<false, true>(q, a.rope, t0, tokens, heads, where, tc, ts);
    else
        a.q_even ? turn_rows<true, false>(q, a.rope, t0, tokens, heads, where, tc, ts)
                : turn_rows<false, false>(q, a.rope, t0, tokens, heads, where, tc, ts);
}

template <int THREADS, int U>
__global__ __launch_bounds__(THREADS, 4) void append_kernel(AppendArgs a) {
    extern __shared__ __align__(16) float tile[];
    __shared__ float red[THREADS / kWave];
    // (queries first where a few tokens' workgroups all start at once, last where they are
    // waited for in turn)
    const unsigned heads = (unsigned)a.c.kv_heads, pages = 2 * a.halves;
    const unsigned block = U == 1 ? (blockIdx.x + pages) % (pages + a.q_blocks) : blockIdx.x;
    if(block >= pages) return turn_queries<THREADS>(a, block - pages);
    if(block < a.halves)
        return append_page<false, THREADS, U>(a, block / heads, (int)(block % heads), tile, red);
    append_page<true, THREADS, U>(a, (block - a.halves) / heads, (int)((block - a.halves) % heads), tile, red);
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
    // Up to 2 tokens a sequence, as tokens are generated: a wave to a page's head, and a tile
    // of 4 tokens, so that all of a step's workgroups have room at once.  (On average over all
    // of the table's sequences, those that wait too: a prompt of 512, 8 + 32 heads of 128, takes
    // 11 us alone, 12 among 64 sequences and 60 among 256.)  Of prompts, whose
    // workgroups take turns: a wave too for pages of 16, most of whose time is the way to the
    // page (8192 tokens, 8 and 16 heads of 64: 45 to 32 us; of 128: 59 to 54; 640 tokens: 7 and
    // 8 to 10); and pages of 128 with heads of 256, which would be alone on a CU, in quarters,
    // read twice (152 to 106 us; few of them in halves).
    const bool few = N <= 2 * cache->B, turns = 2 * tasks * kvh > 1024;
    const bool wave = few || (turns && page == 16 && a.hp <= 128);
    const int threads = wave ? 64 : 256;
    a.cap = few ? 4 : page * a.hp <= 16384 ? (int)page : (turns ? 8192 : 16384) / a.hp;
    a.halves = (unsigned)(tasks * kvh);
    int64_t q_blocks = 0;
    if(q) {
        a.q_even = turn_args(a.q, a.rope, H, hd, q, ldq, q_out, ldqo, 0);
        a.q_tokens = few ? 1 : turn_tokens(N, H, a.rope.half);
        // of a single token, as many heads as a wave turns with its loads in flight at once
        a.q_heads = few ? (int)(threads * kTurnUnits / a.q.per_head.d) : (int)H;
        a.q_heads = a.q_heads < 1 ? 1 : a.q_heads > H ? (int)H : a.q_heads;
        a.q_parts = (int)((H + a.q_heads - 1) / a.q_heads);
        a.q.per_token = div_by(a.q_heads);
        q_blocks = (N + a.q_tokens - 1) / a.q_tokens * a.q_parts;
    }
    if(!grid_fits(2 * tasks * kvh + q_blocks, threads))
        return fail("pk_kv_append_f32: too many pages and heads for one launch");
    a.q_blocks = (unsigned)q_blocks;
    const unsigned blocks = a.q_blocks + 2 * a.halves;
    const size_t lds = sizeof(float) * a.hp * (a.cap + 5);
    if(few)
        append_kernel<64, 1><<<blocks, 64, lds, as_stream(stream)>>>(a);
    else if(wave)
        append_kernel<64, 4><<<blocks, 64, lds, as_stream(stream)>>>(a);
    else
        append_kernel<256, 4><<<blocks, 256, lds, as_stream(stream)>>>(a);
    return launch_status("pk_kv_append_f32");
}
