// pico_amd/csrc/paged_attention.hip -- attention of new tokens over a paged cache of e4m3
// keys and values.
//
// A power of two times e4m3 (4 significant bits) is exact in f16, so a product with a key
// or a value needs no more than the other operand in f16 parts: x = hi + lo, each the
// nearest f16, keeps 22 bits, which leaves sums of a head's length as near as fp32's own
// rounding does.  Queries are first brought to [2^14, 2^15) by a power of two a row;
// probabilities are taken relative to 2^7 below their running maximum: the largest stay in
// f16's range, one of 2^-10 of it keeps the 22 bits, and smaller ones are off by 2^-32 of it.
//
// The scores are computed transposed, S^T = K.Q^T: a column of the result, a query, is in
// one lane's registers and the three lanes 16 apart, and the tokens that a lane holds are
// those that it needs as the operand of O^T = V^T.P^T, for which v is stored with its
// tokens innermost.  So the probabilities stay where they are computed, and keys and values
// go from memory to the matrix cores without LDS.
//
// The value scale 2^ev of a token's page goes into its probability's exponent, and comes
// out of the sum of probabilities again: p = 2^(s + ev - m), l += p 2^-ev, where m is the
// maximum of s + ev.
#include "paged.h"

namespace {

using namespace pk;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kUnit = 64;          // tokens a wave takes at a time
constexpr int kFew = 16;           // query rows a tile, where a sequence has few
constexpr int kMinShare = 4;       // units a workgroup takes at least, where they share a tile
constexpr float kTop = 7.0f;       // probabilities are relative to 2^7 below the maximum m
constexpr float kRaise = 8.0f;     // m is raised when a score passes it by 2^8: p <= 2^15
constexpr float kNone = -INFINITY;  // the maximum of no scores
constexpr float kLeast = -3.402823466e38f;  // and what those of parts are relative to, where all have none

struct AttnArgs {
    PkKvCache c;
    int N, H, group;  // query heads, those of one head of the cache
    float scale;      // times log2(e)
    const float* q;
    int64_t ldq;
    float* o;
    int64_t ldo;
    float* ws;
    int W;    // workgroups that share the units of all tiles
    int splits;  // workgroups to a tile of many rows
    int vec;  // q can be read in float4, and o written
    Quotient by_group;
};

__device__ __forceinline__ f16x8 widen(uint32_t lo, uint32_t hi) {
    union {
        f16x8 v;
        f16x2 p[4];
    } u;
    u.p[0] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
    u.p[1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
    u.p[2] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
    u.p[3] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
    return u.v;
}

// 8 values as their nearest f16 and the nearest f16 to what is left
__device__ __forceinline__ void two_parts(const float* x, f16x8& hi, f16x8& lo) {
#pragma unroll
    for(int i = 0; i < 8; i += 2) {
        const f16x2 h = __builtin_convertvector((f32x2{x[i], x[i + 1]}), f16x2);
        float l0, l1;  // x - h, for which the compiler takes two instructions each
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(l0) : "v"(h), "v"(x[i]));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
            : "=v"(l1)
            : "v"(h), "v"(x[i + 1]));
        const f16x2 l = __builtin_convertvector((f32x2{l0, l1}), f16x2);
        hi[i] = h[0];
        hi[i + 1] = h[1];
        lo[i] = l[0];
        lo[i + 1] = l[1];
    }
}

// a page's power of two from its byte
__device__ __forceinline__ float power(uint8_t e) { return __uint_as_float((uint32_t)e << 23); }

// 0x80 in every byte that is a NaN
__device__ __forceinline__ u32x4 nan_bytes(u32x4 w) {
    return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// a bit for every byte of 16 that is one
__device__ __forceinline__ uint32_t nan_bits(u32x4 w) {
    const u32x4 b = ((nan_bytes(w) >> 7) * 0x01020408u) >> 24 & 0xfu;
    return b[0] | b[1] << 4 | b[2] << 8 | b[3] << 12;
}

// the first n of 16 bytes
__device__ __forceinline__ u32x4 first_bytes(int n) {
    u32x4 keep;
#pragma unroll
    for(int i = 0; i < 4; ++i) {
        const int k = held(n - 4 * i, 0, 4);
        keep[i] = k == 0 ? 0u : 0xffffffffu >> (32 - 8 * k);
    }
    return keep;
}

// What the reference m of a row's probabilities rises by, where their largest exponent is
// mx: to 2^7 below mx where that is above `limit`, 2^15.  The first time, which limit =
// kNone stands for, down too; not where there is no score yet.
__device__ __forceinline__ float raise(float mx, float& limit) {
    if(!(mx > kNone)) return 0.0f;
    const float up = limit == kNone ? mx - kTop : fmaxf(mx - kTop, 0.0f);
    limit = kTop + kRaise;
    return up;
}

// row (token, head of the group) of a sequence -> token
__device__ __forceinline__ int group_of(const AttnArgs& a, int row) { return a.by_group.of(row); }

// the first n of 4 values
__device__ __forceinline__ void store4(float* to, f32x4 v, int n, int vec) {
    if(vec) {
        if(n > 0) *(f32x4*)to = v;
    } else {
#pragma unroll
        for(int k = 0; k < 4; ++k)
            if(k < n) to[k] = v[k];
    }
}

// Loads before it in the source are issued before those after it: results come in the order
// of the loads, so one that is waited for first must not be behind others.
__device__ __forceinline__ void in_order() { asm volatile("" ::: "memory"); }

// A lane's values of a query: step st's are 8 from at(st) on.  Those behind the head's end
// are its first, which the zeros there in the cache leave out (were the first infinite or
// NaN, the row's scores would not be numbers anyway).  All loads are issued before the
// first is used.
template <int STEPS, class F>
__device__ __forceinline__ void load_query(const float* head, int hd, int vec, F at, float (&x)[STEPS][8]) {
    if(vec) {
#pragma unroll
        for(int st = 0; st < STEPS; ++st)
#pragma unroll
            for(int i = 0; i < 8; i += 4) {
                const int d = at(st) + i;
                const f32x4 v = *(const f32x4*)(head + (d < hd ? d : 0));
#pragma unroll
                for(int k = 0; k < 4; ++k) x[st][i + k] = v[k];
            }
    } else {
#pragma unroll
        for(int st = 0; st < STEPS; ++st)
#pragma unroll
            for(int i = 0; i < 8; ++i) x[st][i] = head[at(st) + i < hd ? at(st) + i : 0];
    }
}

// A query, held by lanes W apart, brought to [2^14, 2^15) by 2^-e and cut in two parts;
// returns e.  (Below 2^-86 a query's scores are nothing beside each other: e ends there,
// so that 2^-e is a float.)
template <int W, int STEPS>
__device__ __forceinline__ int bring_up(float (&x)[STEPS][8], f16x8 (&hi)[STEPS], f16x8 (&lo)[STEPS]) {
    float amax = 0.0f;
#pragma unroll
    for(int st = 0; st < STEPS; ++st)
#pragma unroll
        for(int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[st][i]));
#pragma unroll
    for(int o = W; o < kWave; o *= 2) amax = fmaxf(amax, __shfl_xor(amax, o, kWave));
    const int e = amax > 0x1p-86f && amax <= 0x1.fffffep127f ? __builtin_amdgcn_frexp_expf(amax) - 15 : -100;
    const float by = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for(int st = 0; st < STEPS; ++st) {
#pragma unroll
        for(int i = 0; i < 8; ++i) x[st][i] *= by;
        two_parts(x[st], hi[st], lo[st]);
    }
    return e;
}

// Marks, in LDS, of the results that a NaN reaches: a bit for each row of a wave's tile and
// value of the head.  mark: from the NaN (a bit each) among 16 tokens' values d of the head,
// the rows that see them.
__device__ __forceinline__ void clear_marks(uint32_t* marks, int words) {
    for(int i = threadIdx.x % kWave; i < words; i += kWave) marks[i] = 0;
}
template <int HP>
__device__ __forceinline__ void mark(uint32_t nan, int token0, int d, int rows, int first, int group, int past,
                                     uint32_t* marks) {
    for(; nan; nan &= nan - 1) {
        const int t = token0 + __builtin_ctz(nan);
        for(int r = 0; r < rows; ++r)
            if(t <= past + (first + r) / group) atomicOr(&marks[r * (HP / 32) + d / 32], 1u << d % 32);
    }
}
template <int HP>
__device__ __forceinline__ bool marked(const uint32_t* marks, int r, int d) {
    return marks[r * (HP / 32) + d / 32] >> d % 32 & 1;
}

// how a sequence's work is cut: groups of R query rows (token, head of the group) for each
// head of the cache, each over units of the sequence's tokens
template <int R>
__device__ __forceinline__ int tiles_of(const AttnArgs& a, const Seq& s) {
    return (s.n * a.group + R - 1) / R;
}
__device__ __forceinline__ int units_of(const Seq& s) { return (s.end + kUnit - 1) / kUnit; }
// of a line of `all` units, those of one workgroup
__device__ __forceinline__ int share_of(int all, int W) {
    const int s = (all + W - 1) / W;
    return s < kMinShare ? kMinShare : s;
}

// a part's maximum and sum of each row, then its weighted values
template <int HP>
constexpr int kPart = kFew * (HP + 2);

// ------------------------------------------------- few query rows a sequence
// A workgroup's waves take a tile's units in turn and join in LDS.  WHOLE: a workgroup to
// a tile.  Otherwise the units of all sequences, heads and tiles stand in one line, which
// the workgroups share out evenly, whatever the lengths: one takes the end of a tile's
// units, whole tiles, and the beginning of another's.  Tiles that one workgroup covered
// are finished here, the others' parts are left for join_kernel: the one at the beginning
// of a workgroup's share in its place 0, the one at the end in place 1.
// Loads are issued in the order in which they are waited for, each a step before: the pages
// of the unit after the next, the next one's keys, and its values.
// Bound by the cache's bytes where it is long: 64 sequences of 8192 tokens, 32 heads on 8 of
// 128, 138 us (5.6 TB/s; a large copy reaches 5.1); 131072 tokens 50 (5.4), and 5 each for the
// parts to be joined.  8 sequences of 1024 tokens, 12 heads of 64: 7 us, a launch and one
// unit's way from length to page to key to sum.
// Eight waves, as many units at once, where the tiles are fewer than the CUs and the heads
// leave registers for two waves a SIMD (13 sequences of 1500 tokens, 4 heads of 96: 10.5 us,
// with four 10.9; 4 of 1900, 8 heads of 128: 16.1 and 15.4).
template <int HP, bool WHOLE, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, HP < 128 ? 2 : 1) void few_rows_kernel(AttnArgs a) {
    constexpr int C = HP / 64;  // chunks of 64 values of a key; then one of 32
    constexpr bool TAIL = HP % 64 != 0;
    constexpr int STEPS = HP / 32, DT = HP / 16;
    __shared__ __align__(16) float part[WAVES][kFew][HP + 4];
    __shared__ float part_m[WAVES][kFew], part_l[WAVES][kFew];
    __shared__ uint32_t poisoned[WAVES][kFew * HP / 32];
    const PkKvCache& c = a.c;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane % 16, quad = lane / 16;
    const int page = (int)c.page, kvh = (int)c.kv_heads, hd = (int)c.hd, width = (int)c.width;
    const int shift = __builtin_ctz(page);

    int begin = 0, end = 1, at, b;
    Seq s;
    if(!locate(
           c, a.N, [&](const Seq& t) { return tiles_of<kFew>(a, t) * kvh * (WHOLE ? 1 : units_of(t)); },
           [&](int all) {
               if(WHOLE) return (int)blockIdx.x;
               const int share = share_of(all, a.W);
               begin = (int)blockIdx.x * share;  // (at most all + share: fits)
               end = all - begin < share ? all : begin + share;
               return begin;
           },
           at, b, s))
        return;
    int tiles = tiles_of<kFew>(a, s), units = units_of(s);
    int item = WHOLE ? at : at / units, u0 = WHOLE ? 0 : at - item * units;

    for(int now = begin; now < end;) {
        if(!WHOLE) {
            while(item == tiles * kvh) {  // on to the next sequence that has any
                if(++b >= c.B) return;    // (there is one, unless offsets decrease)
                s = sequence(c, a.N, b);
                tiles = tiles_of<kFew>(a, s);
                units = units_of(s);
                item = 0;
            }
        }
        const int u1 = WHOLE || end - now >= units - u0 ? units : u0 + (end - now);

        // 16 tokens lie on one page, whose number and powers a lane of the wave holds for each
        // of the wave's next units: `per` to a unit.  A lane's keys (tokens 16 (col / 4) +
        // 4 t + col % 4) and its values and scores (16 quad ..) may be on two.
        const int32_t* names = c.table + (int64_t)b * width;
        const int per = page < kUnit ? kUnit / page : 1;
        const int x_key = 16 * (col / 4) >> shift, x_value = 16 * quad >> shift;
        const int h = tiles == 1 ? item : item / tiles, first = (item - h * tiles) * kFew;
        int pid, ek, ev, k = 0;
        auto name_units = [&](int u) {
            const int i = ((u + WAVES * (lane / per)) * kUnit + lane % per * page) >> shift;
            pid = names[i < width ? i : 0];
            if(i >= width || pid < 0 || pid >= c.pages) pid = -1;
            const uint32_t at = (uint32_t)(pid < 0 ? 0 : pid) * kvh + h;
            ek = c.k_exp[at];
            ev = c.v_exp[at];
            k = 0;
        };
        auto of_unit = [&](int v, int x) { return __builtin_amdgcn_ds_bpermute(4 * (k * per + x), v); };
        int u = u0 + wave;
        name_units(u);

        // the lane's query: a row of the tile, as operand of 32 values a step, the values in
        // the order that the lane's keys come in
        const int rows = s.n * a.group - first < kFew ? s.n * a.group - first : kFew;
        const int mine = first + (col < rows ? col : 0);
        const int token = group_of(a, mine);
        const int reach = s.past + token;                    // the last key that it sees
        const int clear = s.past + group_of(a, first) + 1;   // tokens that every row sees
        const float* qr = a.q + (int64_t)(s.row + token) * a.ldq +
                          (int64_t)(h * a.group + mine - token * a.group) * hd;
        float x[STEPS][8];
        auto of_step = [&](int st) {
            return TAIL && st == STEPS - 1 ? 64 * C + 8 * quad : 64 * (st / 2) + 16 * quad + 8 * (st % 2);
        };
        load_query(qr, hd, a.vec, of_step, x);
        in_order();
        __builtin_amdgcn_sched_barrier(0);

        u32x4 kr[4][C > 0 ? C : 1], vr[DT];
        u32x2 kt[4];
        // (always the same number of loads, so that the compiler knows how many are younger
        // than those that it waits for: where there is no unit, of one line)
        auto load_keys = [&](int u, int pid) {
            const int slot = ((u * kUnit + 16 * (col / 4)) & (page - 1)) + col % 4;
            const uint8_t* p = c.k + (uint64_t)((uint32_t)(pid < 0 ? 0 : pid) * kvh + h) * (uint32_t)(HP * page) +
                               (slot * HP + 16 * quad);
            if(u >= u1) p = c.k;
#pragma unroll
            for(int t = 0; t < 4; ++t) {
#pragma unroll
                for(int i = 0; i < C; ++i)
                    kr[t][i] = *(const u32x4*)(p + 4 * t * HP + 64 * i);
                if(TAIL) kt[t] = *(const u32x2*)(p + 4 * t * HP + 64 * C - (u >= u1 ? 0 : 8 * quad));
                in_order();
            }
        };
        auto load_values = [&](int u, int pid) {
            const int slot = (u * kUnit + 16 * quad) & (page - 1);
            const uint8_t* p = c.v + (uint64_t)((uint32_t)(pid < 0 ? 0 : pid) * kvh + h) * (uint32_t)(HP * page) +
                               (col * page + slot);
            if(u >= u1) p = c.v;
#pragma unroll
            for(int i = 0; i < DT; ++i) vr[i] = *(const u32x4*)(p + (uint32_t)(16 * i * page));
            in_order();
        };
        int pv = of_unit(pid, x_value);
        load_keys(u, of_unit(pid, x_key));
        load_values(u, pv);
        __builtin_amdgcn_sched_barrier(0);  // (nor is the query waited for before)

        f16x8 qh[STEPS], ql[STEPS];
        const int eq = bring_up<16>(x, qh, ql);
        const float coef = ldexpf(a.scale, eq);

        f32x4 acc[DT];
#pragma unroll
        for(int i = 0; i < DT; ++i) acc[i] = f32x4{};
        float m = 0.0f, l = 0.0f, limit = kNone;  // (of no score yet)
        bool poison = false;
        for(; u < u1; u += WAVES) {
            const int next = u + WAVES;
            f32x4 sc[4];
#pragma unroll
            for(int t = 0; t < 4; ++t) {
                sc[t] = f32x4{};
#pragma unroll
                for(int st = 0; st < STEPS; ++st) {
                    f16x8 kf;
                    if(TAIL && st == STEPS - 1)
                        kf = widen(kt[t][0], kt[t][1]);
                    else if(st % 2 == 0)
                        kf = widen(kr[t][st / 2][0], kr[t][st / 2][1]);
                    else
                        kf = widen(kr[t][st / 2][2], kr[t][st / 2][3]);
                    sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[st], sc[t], 0, 0, 0);
                    sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[st], sc[t], 0, 0, 0);
                }
            }
            // (of pages that hold no key these may be any byte, and 0 times 2^-ev has to be 0; here, not
            // where they are loaded, which would wait for them)
            const int ek_now = exponent_byte(of_unit(ek, x_value)), ev_now = exponent_byte(of_unit(ev, x_value));
            const float kc = coef * power(ek_now), vexp = (float)(ev_now - 127), vinv = power(254 - ev_now);
            const bool absent = pv < 0;
            if(++k * per == kWave) name_units(next);
            pv = of_unit(pid, x_value);
            load_keys(next, of_unit(pid, x_key));
            float p[16], mx = kNone;
            const float low = vexp - (m - kTop);
#pragma unroll
            for(int t = 0; t < 4; ++t)
#pragma unroll
                for(int r = 0; r < 4; ++r) p[4 * t + r] = fmaf(sc[t][r], kc, low);
            const int token0 = u * kUnit + 16 * quad;
            const bool edge = u * kUnit + kUnit > clear || __ballot(absent) != 0;
            if(edge) {
#pragma unroll
                for(int i = 0; i < 16; ++i)
                    if(absent || token0 + i > reach) p[i] = -INFINITY;
            }
#pragma unroll
            for(int i = 0; i < 16; ++i) mx = fmaxf(mx, p[i]);
            if(__ballot(mx > limit)) {
                mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
                mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
                const bool some = __ballot(limit != kNone) != 0;  // (else there is nothing to scale)
                const float up = raise(mx, limit);
                m += up;
                if(some) {
                    const float down = __builtin_amdgcn_exp2f(fminf(-up, 0.0f));
                    l *= down;
#pragma unroll
                    for(int i = 0; i < DT; ++i) acc[i] *= down;
                }
#pragma unroll
                for(int i = 0; i < 16; ++i) p[i] -= up;
            }
            f32x4 sums = {};
#pragma unroll
            for(int i = 0; i < 16; ++i) {
                p[i] = __builtin_amdgcn_exp2f(p[i]);
                sums[i % 4] += p[i];
            }
            const float sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
            l = fmaf(sum, vinv, l);
            f16x8 ph[2], pl[2];
            two_parts(p, ph[0], pl[0]);
            two_parts(p + 8, ph[1], pl[1]);
            if(edge) {
                // tokens behind the sequence's last, or on no page, may hold anything
                const u32x4 keep = first_bytes(absent ? 0 : held(s.end - token0, 0, 16));
#pragma unroll
                for(int i = 0; i < DT; ++i) vr[i] &= keep;
                u32x4 nan = {};
                if(s.n > 1) {  // (of a single token, all rows see all that are left)
#pragma unroll
                    for(int i = 0; i < DT; ++i) nan |= nan_bytes(vr[i]);
                }
                if(__builtin_expect(__ballot((nan[0] | nan[1] | nan[2] | nan[3]) != 0) != 0, 0)) {
                    // a NaN among the values of tokens that some rows do not see must not
                    // reach them by 0 times it: zeros in its place, and the rows that do
                    // see it are noted
                    if(!poison) clear_marks(poisoned[wave], kFew * HP / 32);
                    poison = true;
                    auto* found = (volatile uint16_t*)&part[wave][0][0];
#pragma unroll
                    for(int i = 0; i < DT; ++i) {
                        found[kWave * i + lane] = nan_bits(vr[i]);
                        vr[i] &= ~((nan_bytes(vr[i]) >> 7) * 0xff);
                    }
#pragma unroll 1
                    for(int i = 0; i < DT; ++i)
                        mark<HP>(found[kWave * i + lane], token0, 16 * i + col, rows, first, a.group, s.past,
                                 poisoned[wave]);
                }
            }
#pragma unroll
            for(int i = 0; i < DT; ++i) {
                const f16x8 v0 = widen(vr[i][0], vr[i][1]), v1 = widen(vr[i][2], vr[i][3]);
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[0], acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[1], acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[0], acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[1], acc[i], 0, 0, 0);
            }
            load_values(next, pv);
        }

        // the waves' parts together
        l += __shfl_xor(l, 16, kWave);
        l += __shfl_xor(l, 32, kWave);
        if(poison) {
#pragma unroll
            for(int i = 0; i < DT; ++i)
#pragma unroll
                for(int r = 0; r < 4; ++r)
                    if(marked<HP>(poisoned[wave], col, 16 * i + 4 * quad + r)) acc[i][r] = NAN;
        }
#pragma unroll
        for(int i = 0; i < DT; ++i) *(f32x4*)&part[wave][col][16 * i + 4 * quad] = acc[i];
        if(lane < 16) {
            part_m[wave][lane] = limit == kNone ? kNone : m;
            part_l[wave][lane] = l;
        }
        __syncthreads();
        const bool whole = WHOLE || (u0 == 0 && u1 == units);
        float* out = a.ws + ((int64_t)blockIdx.x * 2 + (now == begin ? 0 : 1)) * kPart<HP>;
        for(int i = threadIdx.x; i < rows * (HP / 4); i += WAVES * kWave) {
            const int r = i / (HP / 4), d = 4 * (i % (HP / 4));
            float top = kLeast, total = 0.0f;
#pragma unroll
            for(int k = 0; k < WAVES; ++k) top = fmaxf(top, part_m[k][r]);
            f32x4 v = {};
#pragma unroll
            for(int k = 0; k < WAVES; ++k) {
                const float f = __builtin_amdgcn_exp2f(part_m[k][r] - top);
                total = fmaf(f, part_l[k][r], total);
                v += f * *(const f32x4*)&part[k][r][d];
            }
            if(!whole) {
                if(d == 0) {
                    out[r] = top;
                    out[kFew + r] = total;
                }
                *(f32x4*)(out + 2 * kFew + r * HP + d) = v;
                continue;
            }
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;  // (0: no key at all)
            const int t = group_of(a, first + r);
            float* to = a.o + (int64_t)(s.row + t) * a.ldo + (int64_t)(h * a.group + first + r - t * a.group) * hd + d;
            store4(to, v * inv, hd - d, a.vec);
        }
        if(WHOLE) return;
        __syncthreads();
        now += u1 - u0;
        u0 = 0;
        ++item;
    }
}

// The tiles that several workgroups have parts of: a workgroup here stands for the one
// there that has a tile's last part, and a wave for one of the tile's rows, its lanes on 4
// values each of as many parts at once as there are lanes for.
template <int HP>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a) {
    constexpr int D4 = HP / 4, PARTS = kWave / D4;
    const PkKvCache& c = a.c;
    const int lane = threadIdx.x % kWave, r = blockIdx.y * 4 + threadIdx.x / kWave;
    int share = 1, at, b;
    Seq s;
    if(!locate(
           c, a.N, [&](const Seq& t) { return tiles_of<kFew>(a, t) * (int)c.kv_heads * units_of(t); },
           [&](int all) {
               share = share_of(all, a.W);
               return (int)blockIdx.x * share;
           },
           at, b, s))
        return;
    const int tiles = tiles_of<kFew>(a, s), units = units_of(s), item = at / units, u0 = at - item * units;
    if(u0 == 0 || units - u0 > share) return;  // it begins here, or has parts behind
    const int h = item / tiles, row = (item - h * tiles) * kFew + r;
    if(row >= s.n * a.group) return;
    // the first part's workgroup, where it is in that one's place 0 if it begins its share
    const int before = (u0 + share - 1) / share, w1 = blockIdx.x, w0 = w1 - before;
    if(w0 < 0) return;  // (offsets that decrease)
    const int first_place = before * share == u0 ? 0 : 1;
    auto part = [&](int w) { return a.ws + ((int64_t)w * 2 + (w == w0 ? first_place : 0)) * kPart<HP>; };
    float top = kLeast;
    for(int w = w0 + lane; w <= w1; w += kWave) top = fmaxf(top, part(w)[r]);
    top = wave_max(top);
    const int d = 4 * (lane % D4), mine = lane / D4;
    f32x4 v = {};
    float total = 0.0f;
    if(mine < PARTS) {
#pragma unroll 4
        for(int w = w0 + mine; w <= w1; w += PARTS) {
            const float* p = part(w);
            const float f = __builtin_amdgcn_exp2f(p[r] - top);
            total = fmaf(f, p[kFew + r], total);
            v += f * *(const f32x4*)(p + 2 * kFew + r * HP + d);
        }
    }
    f32x4 sum = v;
    float all = total;
#pragma unroll
    for(int k = 1; k < PARTS; ++k) {
        all += __shfl(total, lane + k * D4, kWave);
#pragma unroll
        for(int i = 0; i < 4; ++i) sum[i] += __shfl(v[i], lane + k * D4, kWave);
    }
    if(mine) return;
    const float inv = all == 0.0f ? 0.0f : 1.0f / all;
    const int t = group_of(a, row);
    float* to = a.o + (int64_t)(s.row + t) * a.ldo + (int64_t)(h * a.group + row - t * a.group) * c.hd + d;
    store4(to, sum * inv, (int)c.hd - d, a.vec);
}

// ------------------------------------------------ many query rows a sequence
// A workgroup takes 128 query rows of one head of the cache, a wave 32 of them as the
// columns of 32x32 products, whose results' rows are in a lane and the one 32 further.
// Units of 64 tokens go through LDS, still in 8 bits, two at a time: one is read while the
// next is on its way through registers.  Keys stand in LDS in the order of the product's
// rows, so that a lane's 16 scores are of 16 tokens in a row, on one page; rows of both are
// 16 bytes apart from a power of two, which spreads 8 lanes' 16 bytes over all banks.
// `splits` workgroups share a tile's units where the tiles are too few for the chip, and
// leave their parts for finish_kernel.
// Heads of 128: 2 chunks of 2048 tokens behind 6144, 32 heads on 8, 720 us, 1.07 PFLOP/s of
// f16 products, where a large library product reaches 1.18 and the matrix cores fed from
// registers 2.1: two waves a SIMD, all that there are registers for, overlap the one's products
// with the other's exponentials 1.6 times.  Heads of 64 and less are held by the exponentials
// and roundings of each score (8 chunks of 256 behind 16000, 32 heads of 64: 410 us, 298 by the
// products at the library's rate).
constexpr int kRows = 128;

template <int HP>
constexpr int64_t kManyPart = (int64_t)kRows * (HP + 2);

template <int HP>
__global__ __launch_bounds__(256, HP == 256 ? 1 : 2) void many_rows_kernel(AttnArgs a) {
    constexpr int STEPS = HP / 16, DT = HP / 32;
    constexpr int KS = HP + 16, VS = kUnit + 16;       // bytes between rows in LDS
    constexpr int CHUNKS = kUnit * HP / 16, LOADS = (CHUNKS + 255) / 256;  // of 16 bytes; a thread's
    __shared__ __align__(16) uint8_t keys[2][kUnit * KS], values[2][HP * VS];
    __shared__ __align__(16) float4 pages[2][kUnit / 16];  // 2^ek, ev, 2^-ev, whether there
    __shared__ uint32_t poisoned[4][HP];
    const PkKvCache& c = a.c;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane % 32, half = lane / 32;
    const int page = (int)c.page, kvh = (int)c.kv_heads, hd = (int)c.hd, shift = __builtin_ctz(page);

    // heads of the cache in turn, so that one stays with an XCD; then parts, then tiles
    const int h = (int)(blockIdx.x % (unsigned)kvh);
    const int rest = (int)(blockIdx.x / (unsigned)kvh), split = rest % a.splits;
    int at, b;
    Seq s;
    if(!locate(
           c, a.N, [&](const Seq& t) { return tiles_of<kRows>(a, t); }, [&](int) { return rest / a.splits; },
           at, b, s))
        return;
    const int tile = tiles_of<kRows>(a, s) - 1 - at;  // those that see the most first
    const int first = tile * kRows + wave * 32, total = s.n * a.group;
    const int last = (tile + 1) * kRows < total ? (tile + 1) * kRows - 1 : total - 1;
    int units = s.past + last / a.group + 1;
    units = ((units < s.end ? units : s.end) + kUnit - 1) / kUnit;
    const int each = (units + a.splits - 1) / a.splits;
    const int u0 = split * each, u1 = u0 + each < units ? u0 + each : units;

    // the lane's query
    const int row = first + col, rows = total - first < 32 ? total - first : 32;
    const int real_row = col < rows ? row : tile * kRows;
    const int token = group_of(a, real_row);
    const float* qr = a.q + (int64_t)(s.row + token) * a.ldq +
                      (int64_t)(h * a.group + real_row - token * a.group) * hd;
    const int reach = s.past + token;
    f16x8 qh[STEPS], ql[STEPS];
    float coef;
    {
        float x[STEPS][8];
        auto of_step = [&](int st) { return 32 * (st / 2) + 16 * half + 8 * (st % 2); };
        load_query(qr, hd, a.vec, of_step, x);
        coef = ldexpf(a.scale, bring_up<32>(x, qh, ql));
    }

    auto page_of = [&](int u, int g16) {
        const int i = (u * kUnit + 16 * g16) >> shift;
        const int pid = u < u1 && i < c.width ? c.table[(int64_t)b * c.width + i] : -1;
        return pid < 0 || pid >= c.pages ? -1 : pid;
    };
    // a thread's chunks: of keys, 16 values of token e / (HP / 16); of values, 16 tokens of
    // row e / 4, of which `real` are the sequence's
    int pk[LOADS], pv, real = 0;
    u32x4 kr[LOADS], vr[LOADS];
    float4 pr;
    const int g16 = threadIdx.x % 4;
    auto find_pages = [&](int u) {
#pragma unroll
        for(int i = 0; i < LOADS; ++i) pk[i] = page_of(u, (threadIdx.x + 256 * i) / (HP / 16) % kUnit / 16);
        pv = page_of(u, g16);
    };
    auto load = [&](int u) {
        const int64_t v_head = (int64_t)(pv < 0 ? 0 : pv) * kvh + h;
#pragma unroll
        for(int i = 0; i < LOADS; ++i) {
            const int e = threadIdx.x + 256 * i, t = e / (HP / 16), d16 = e % (HP / 16);
            if(e < CHUNKS) {
                const int64_t k_head = (int64_t)(pk[i] < 0 ? 0 : pk[i]) * kvh + h;
                kr[i] = *(const u32x4*)(c.k + (k_head * page + ((u * kUnit + t) & (page - 1))) * HP + 16 * d16);
                vr[i] = *(const u32x4*)(c.v + (v_head * HP + e / 4) * page +
                                        ((u * kUnit + 16 * g16) & (page - 1)));
            }
        }
        if(threadIdx.x < 4) {
            const int ek = exponent_byte(c.k_exp[v_head]), ev = exponent_byte(c.v_exp[v_head]);
            pr = {power(ek), (float)(ev - 127), power(254 - ev), pv < 0 ? 0.0f : 1.0f};
        }
        real = pv < 0 ? 0 : held(s.end - u * kUnit - 16 * g16, 0, 16);
    };
    auto store = [&](int buf) {
#pragma unroll
        for(int i = 0; i < LOADS; ++i) {
            const int e = threadIdx.x + 256 * i, t = e / (HP / 16), d16 = e % (HP / 16);
            if(e < CHUNKS) {
                // the row of the product that a token is: bits 4 3 2 1 0 become 3 2 4 1 0
                const int row = (t & 32) + ((t & 12) << 1) + ((t & 16) >> 2) + (t & 3);
                *(u32x4*)&keys[buf][row * KS + 16 * d16] = kr[i];
                // (values behind the sequence's end, or on no page, may be anything)
                if(real < 16) vr[i] &= first_bytes(real);
                *(u32x4*)&values[buf][e / 4 * VS + 16 * g16] = vr[i];
            }
        }
        if(threadIdx.x < 4) pages[buf][threadIdx.x] = pr;
    };

    f32x16 acc[DT];
#pragma unroll
    for(int i = 0; i < DT; ++i) acc[i] = f32x16{};
    float m = 0.0f, l = 0.0f, limit = kNone;
    bool poison = false;
    const int clear = s.past + (first < total ? group_of(a, first) : 0) + 1;  // tokens that all rows see
    const int reach_all = s.past + (first + rows - 1) / a.group;           // and that any does
    find_pages(u0);
    if(u0 < u1) {
        load(u0);
        store(0);
    }
    find_pages(u0 + 1);
    __syncthreads();
    for(int u = u0; u < u1; ++u) {
        const int buf = (u - u0) & 1;
        if(u + 1 < u1) {
            load(u + 1);
            find_pages(u + 2);
        }
#pragma unroll
        for(int j = 0; j < 2; ++j) {
            const int token0 = u * kUnit + 32 * j;
            if(rows <= 0 || token0 > reach_all) continue;
            // (of a SIMD's waves those that have products to give the matrix cores before those
            // that do not; heads of 256 leave room for one)
            if(HP < 256) __builtin_amdgcn_s_setprio(1);
            f32x16 sc = {};
#pragma unroll
            for(int st = 0; st < STEPS; st += 2) {
                const u32x4 w = *(const u32x4*)&keys[buf][(32 * j + col) * KS + 16 * st + 16 * half];
                const f16x8 k0 = widen(w[0], w[1]), k1 = widen(w[2], w[3]);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, qh[st], sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, qh[st + 1], sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, ql[st], sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, ql[st + 1], sc, 0, 0, 0);
            }
            if(HP < 256) __builtin_amdgcn_s_setprio(0);
            const float4 g = pages[buf][2 * j + half];
            const float kc = coef * g.x;
            const bool absent = g.w == 0.0f;
            const int mine0 = token0 + 16 * half;
            float p[16], mx = kNone;
            const float low = g.y - (m - kTop);
#pragma unroll
            for(int i = 0; i < 16; ++i) p[i] = fmaf(sc[i], kc, low);
            const bool edge = token0 + 32 > clear || __ballot(absent) != 0;
            if(edge) {
#pragma unroll
                for(int i = 0; i < 16; ++i)
                    if(absent || mine0 + i > reach) p[i] = -INFINITY;
            }
#pragma unroll
            for(int i = 0; i < 16; ++i) mx = fmaxf(mx, p[i]);
            if(__ballot(mx > limit)) {
                mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
                const bool some = __ballot(limit != kNone) != 0;  // (else there is nothing to scale)
                const float up = raise(mx, limit);
                m += up;
                if(some) {
                    const float down = __builtin_amdgcn_exp2f(fminf(-up, 0.0f));
                    l *= down;
#pragma unroll
                    for(int i = 0; i < DT; ++i) acc[i] *= down;
                }
#pragma unroll
                for(int i = 0; i < 16; ++i) p[i] -= up;
            }
            f32x4 sums = {};
#pragma unroll
            for(int i = 0; i < 16; ++i) {
                p[i] = __builtin_amdgcn_exp2f(p[i]);
                sums[i % 4] += p[i];
            }
            const float sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
            l = fmaf(sum, g.z, l);
            f16x8 ph[2], pl[2];
            two_parts(p, ph[0], pl[0]);
            two_parts(p + 8, ph[1], pl[1]);
            bool clean = false;  // NaN become zeros
            auto value = [&](int i) {
                return *(const u32x4*)&values[buf][(32 * i + col) * VS + 32 * j + 16 * half];
            };
            if(edge) {
                u32x4 nan = {};
#pragma unroll
                for(int i = 0; i < DT; ++i) nan |= nan_bytes(value(i));
                if(__builtin_expect(__ballot((nan[0] | nan[1] | nan[2] | nan[3]) != 0) != 0, 0)) {
                    if(!poison) clear_marks(poisoned[wave], HP);  // (as in few_rows_kernel)
                    poison = clean = true;
#pragma unroll 1
                    for(int i = 0; i < DT; ++i)
                        mark<HP>(nan_bits(value(i)), mine0, 32 * i + col, rows, first, a.group, s.past,
                                 poisoned[wave]);
                }
            }
#pragma unroll
            for(int i = 0; i < DT; ++i) {
                u32x4 w = value(i);
                if(__builtin_expect(clean, 0)) w &= ~((nan_bytes(w) >> 7) * 0xff);
                const f16x8 v0 = widen(w[0], w[1]), v1 = widen(w[2], w[3]);
                acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0, ph[0], acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1, ph[1], acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0, pl[0], acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1, pl[1], acc[i], 0, 0, 0);
            }
        }
        if(u + 1 < u1) store(buf ^ 1);
        __syncthreads();
    }

    l += __shfl_xor(l, 32, kWave);
    if(col >= rows) return;
    if(poison) {
#pragma unroll
        for(int i = 0; i < DT; ++i)
#pragma unroll
            for(int r = 0; r < 16; ++r)
                if(marked<HP>(poisoned[wave], col, 32 * i + 8 * (r / 4) + 4 * half + r % 4)) acc[i][r] = NAN;
    }
    if(a.splits > 1) {  // (a part without units has the maximum of no scores, and zeros)
        float* out = a.ws + (int64_t)blockIdx.x * kManyPart<HP>;
        const int r = wave * 32 + col;
        if(half == 0) {
            out[r] = limit == kNone ? kNone : m;
            out[kRows + r] = l;
        }
#pragma unroll
        for(int i = 0; i < DT; ++i)
#pragma unroll
            for(int q = 0; q < 4; ++q)
                *(f32x4*)(out + 2 * kRows + r * HP + 32 * i + 8 * q + 4 * half) =
                    f32x4{acc[i][4 * q], acc[i][4 * q + 1], acc[i][4 * q + 2], acc[i][4 * q + 3]};
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float* to = a.o + (int64_t)(s.row + token) * a.ldo + (int64_t)(h * a.group + row - token * a.group) * hd;
#pragma unroll
    for(int i = 0; i < DT; ++i)
#pragma unroll
        for(int q = 0; q < 4; ++q) {
            const int d = 32 * i + 8 * q + 4 * half;
            const f32x4 v = {acc[i][4 * q], acc[i][4 * q + 1], acc[i][4 * q + 2], acc[i][4 * q + 3]};
            store4(to + d, v * inv, hd - d, a.vec);
        }
}

// the parts of many_rows_kernel's tiles together: a wave to a row
template <int HP>
__global__ __launch_bounds__(256) void finish_kernel(AttnArgs a) {
    constexpr int D4 = HP / 4;
    const PkKvCache& c = a.c;
    const int lane = threadIdx.x % kWave, kvh = (int)c.kv_heads;
    const int h = (int)(blockIdx.x % (unsigned)kvh);
    const int rest = (int)(blockIdx.x / (unsigned)kvh);
    int at, b;
    Seq s;
    if(!locate(
           c, a.N, [&](const Seq& t) { return tiles_of<kRows>(a, t); }, [&](int) { return rest; }, at, b, s))
        return;
    const int r = blockIdx.y * 4 + threadIdx.x / kWave;
    const int row = (tiles_of<kRows>(a, s) - 1 - at) * kRows + r;
    if(row >= s.n * a.group) return;
    const float* base = a.ws + ((int64_t)rest * a.splits * kvh + h) * kManyPart<HP>;
    const int64_t apart = (int64_t)kvh * kManyPart<HP>;
    float top = kLeast, total = 0.0f;
    if(lane < a.splits) top = base[lane * apart + r];  // (at most a lane each)
    top = wave_max(top);
    const int d = 4 * lane;
    f32x4 v = {};
#pragma unroll 8
    for(int i = 0; i < a.splits; ++i) {
        const float* p = base + i * apart;
        const float f = __builtin_amdgcn_exp2f(p[r] - top);
        total = fmaf(f, p[kRows + r], total);
        if(lane < D4) v += f * *(const f32x4*)(p + 2 * kRows + r * HP + d);
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const int t = group_of(a, row);
    float* to = a.o + (int64_t)(s.row + t) * a.ldo + (int64_t)(h * a.group + row - t * a.group) * c.hd + d;
    if(lane < D4) store4(to, v * inv, (int)c.hd - d, a.vec);
}

// ------------------------------------------------------------------- launches
struct Plan {
    int rows;       // 16 or 128 query rows a tile
    int W;          // of few rows: workgroups that share the units of all tiles; 0: one to a tile
    int splits;     // of many: workgroups to a tile
    int64_t tiles;  // for each head of the cache, that there may be
};
Plan plan(const PkKvCache* c, int64_t N, int64_t H) {
    Plan p = {};
    const int64_t group = H / c->kv_heads, units = (c->width * c->page + kUnit - 1) / kUnit;
    const int64_t some = c->B < N ? c->B : N;
    // Tiles of 16 rows up to 96 rows a sequence on average, or 4096 of all heads together;
    // over up to 2048 tokens up to 24576 of heads of up to 64 values, 12288 of 128, 8192 of more.
    // Tiles of 128 read the cache less often but are left partly empty, and are less finely
    // shared out.  32 heads on 8 of 128: 16 sequences of 4000 tokens with up to 40 new ones 82
    // against 92 us, with up to 60 119 against 116; one of 4000 with 256 61 against 59; 4 of 1900
    // with 100 35 against 45; one with 700 40 against 36.  16 heads on 2 of 64: 16 of 1000 with 100
    // 25 against 44, 4 of 500 with 300 17 against 28; 32 on 8: 8 of 100 with 200 26 against 19.
    // The average is over all of the table's sequences, those that wait too: 1500 tokens behind
    // 4000, 32 heads on 8 of 128, take 254 us alone and 489 among 64 sequences.
    const int64_t most = units > 32 ? 4096 : c->hd <= 64 ? 24576 : c->hd <= 128 ? 12288 : 8192;
    p.rows = N * group <= 96 * c->B || N * H <= most ? kFew : kRows;
    p.tiles = N * group / p.rows + some;
    if(p.rows < kRows) {
        // A workgroup to a tile up to 2048 tokens, 1024 of heads of more than 128: 8 sequences of
        // 1024, 12 heads of 64, 7.6 us, shared out and joined 12.3; 4 of 3900, 8 heads of 128, 25
        // against 17; 4 of 1900, 8 heads of 256, 28 against 22.  256 workgroups share them, one
        // to a CU, which the loads of four waves suffice for: 131072 tokens 49 us, 512 of them 57.
        p.W = units <= (c->hd <= 128 ? 32 : 16) || p.tiles * c->kv_heads * units >= (int64_t)1 << 31 ? 0 : 256;
    } else {
        // The workgroups that there are for sure: one to a CU where they get 4 units each, as
        // many as a CU holds where they get 8.  One sequence of 32000 tokens with 64 new ones, 3
        // heads of 168: 63 parts a tile 65 us, 16 168; of 2000 tokens with 256, 8 parts 36, 4 57;
        // 2 of 4000 with 1024, 12 heads of 64: 4 parts 75, 2 96.  Long sequences of different
        // lengths in parts of 40 units, 3 at least, where there are more than run at once, which
        // levels them out: 8 up to 16000 with 256, 32 heads of 64: 4 parts 413, whole tiles 520.
        // The parts are of what the table has room for, the lengths are not known here: 2 prompts
        // of 256 tokens, 32 heads on 8 of 128, take 26 us with tables of 512 tokens, 74 of 131072.
        const int64_t sure = (N * group + kRows - 1) / kRows * c->kv_heads;
        auto parts = [&](int64_t blocks, int64_t each) {
            return blocks / sure < units / each ? blocks / sure : units / each;
        };
        const int64_t one = parts(256, 4), full = parts(c->hd <= 64 ? 768 : 512, 8), level = parts(2048, 40);
        int64_t n = one > full ? one : full;
        if(c->B > 1 && level >= 3 && level > n && level * sure >= 1024) n = level;
        p.splits = (int)(n < 1 ? 1 : n > kWave ? kWave : n);
    }
    return p;
}
size_t plan_bytes(const Plan& p, const PkKvCache* c) {
    const size_t hp = head_size(c->hd);
    if(p.W) return sizeof(float) * 2 * p.W * kFew * (hp + 2);
    if(p.splits > 1) return sizeof(float) * p.tiles * c->kv_heads * p.splits * kRows * (hp + 2);
    return 0;
}

int check_attn(const char* who, const PkKvCache* c, int64_t N, int64_t H) {
    if(int st = check_cache(who, c, N)) return st;
    if(H < 1 || H % c->kv_heads || H > (1 << 20) / c->hd)
        return fail("%s: %lld query heads on %lld of the cache: a multiple, with H*hd up to 2^20", who,
                    (long long)H, (long long)c->kv_heads);
    if(N * H >= (int64_t)1 << 31)
        return fail("%s: too many query rows, N*H up to 2^31 - 1", who);
    return PK_OK;
}

template <int HP>
void launch(const AttnArgs& a, const Plan& p, hipStream_t st) {
    const int64_t tiles = p.tiles * a.c.kv_heads;
    constexpr int MANY = HP < 128 ? 8 : 4;  // waves of few tiles
    if(p.rows == kRows) {
        many_rows_kernel<HP><<<(unsigned)(tiles * p.splits), 256, 0, st>>>(a);
        if(p.splits > 1) finish_kernel<HP><<<dim3((unsigned)tiles, kRows / 4), 256, 0, st>>>(a);
    } else if(p.W) {
        few_rows_kernel<HP, false, 4><<<(unsigned)p.W, 256, 0, st>>>(a);
        join_kernel<HP><<<dim3((unsigned)p.W, kFew / 4), 256, 0, st>>>(a);
    } else if(tiles < 256) {
        few_rows_kernel<HP, true, MANY><<<(unsigned)tiles, MANY * kWave, 0, st>>>(a);
    } else {
        few_rows_kernel<HP, true, 4><<<(unsigned)tiles, 256, 0, st>>>(a);
    }
}

}  // namespace

extern "C" size_t pk_attn_paged_workspace(const PkKvCache* cache, int64_t N, int64_t H) {
    if(check_attn("pk_attn_paged_workspace", cache, N, H) || N == 0 || cache->B == 0) return 0;
    return plan_bytes(plan(cache, N, H), cache);
}

extern "C" int pk_attn_paged_f32(const PkKvCache* cache, int64_t N, int64_t H, float scale,
                                 const float* q, int64_t ldq, float* o, int64_t ldo, void* workspace,
                                 size_t workspace_bytes, pk_stream_t stream) {
    if(int st = check_attn("pk_attn_paged_f32", cache, N, H)) return st;
    if(N == 0 || cache->B == 0) return PK_OK;
    const int64_t width = H * cache->hd;
    if(!q || !o) return fail("pk_attn_paged_f32: NULL pointer");
    if(ldq < width || ldo < width)
        return fail("pk_attn_paged_f32: row strides must be at least H*hd = %lld", (long long)width);
    const Plan p = plan(cache, N, H);
    const size_t need = plan_bytes(p, cache);
    if(need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail("pk_attn_paged_f32: workspace of %zu bytes, %zu needed, 16-byte aligned",
                    workspace ? workspace_bytes : 0, need);
    if(!p.W && !grid_fits(p.tiles * cache->kv_heads * (p.splits > 1 ? p.splits : 1), 256))
        return fail("pk_attn_paged_f32: too many rows for one launch");
    AttnArgs a = {};
    a.c = *cache;
    a.N = (int)N;
    a.H = (int)H;
    a.group = (int)(H / cache->kv_heads);
    a.scale = scale * 1.4426950408889634f;
    a.q = q;
    a.ldq = ldq;
    a.o = o;
    a.ldo = ldo;
    a.ws = (float*)workspace;
    a.W = p.W;
    a.splits = p.splits;
    a.vec = cache->hd % 4 == 0 && ldq % 4 == 0 && ldo % 4 == 0 && aligned16(q) && aligned16(o);
    a.by_group = quotient(a.group);
    const hipStream_t st = as_stream(stream);
    switch(head_size(cache->hd)) {
        case 32: launch<32>(a, p, st); break;
        case 64: launch<64>(a, p, st); break;
        case 96: launch<96>(a, p, st); break;
        case 128: launch<128>(a, p, st); break;
        default: launch<256>(a, p, st); break;
    }
    return launch_status("pk_attn_paged_f32");
}
