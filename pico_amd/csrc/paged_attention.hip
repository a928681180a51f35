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

constexpr int kUnit = 64;          // tokens a wave takes at a time
constexpr int kMinShare = 4;       // units a workgroup takes at least, where they share a tile
constexpr float kTop = 7.0f;       // probabilities are relative to 2^7 below the maximum m
constexpr float kRaise = 8.0f;     // m is raised when a score passes it by 2^8: p <= 2^15
constexpr float kNone = -1e30f;    // the maximum of no scores

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
    int vec;  // q can be read in float4
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

// the value of the lane 8 further in the row of 16
__device__ __forceinline__ float across8(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, false));
}

// a page's power of two from its byte
__device__ __forceinline__ float power(uint8_t e) { return __uint_as_float((uint32_t)e << 23); }

// 0x80 in every byte that is a NaN
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
    return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
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
constexpr int kPart = 32 + 16 * HP;

// ------------------------------------------------- few query rows a sequence
// (heads of 256 take the registers that two waves of smaller ones share)
constexpr int waves_of(int hp, bool whole) { return whole && hp < 256 ? 8 : 4; }

// A workgroup's waves take a tile's units in turn and join in LDS.  WHOLE: a workgroup to
// a tile.  Otherwise the units of all sequences, heads and tiles stand in one line, which
// the workgroups share out evenly, whatever the lengths: one takes the end of a tile's
// units, whole tiles, and the beginning of another's.  Tiles that one workgroup covered
// are finished here, the others' parts are left for join_kernel: the one at the beginning
// of a workgroup's share in its place 0, the one at the end in place 1.
// SPLIT: the 16 columns are 8 rows' high parts and their low parts; else 16 rows, for two
// products.
template <int HP, bool SPLIT, bool WHOLE>
__global__ __launch_bounds__(waves_of(HP, WHOLE) * kWave, HP == 256 ? 1 : 2)
void few_rows_kernel(AttnArgs a) {
    constexpr int kWaves = waves_of(HP, WHOLE);
    constexpr int R = SPLIT ? 8 : 16;  // query rows
    constexpr int C = HP / 64;         // chunks of 64 values of a key; then one of 32
    constexpr bool TAIL = HP % 64 != 0;
    constexpr int STEPS = HP / 32, DT = HP / 16;
    __shared__ __align__(16) float part[kWaves][R][HP + 4];
    __shared__ float part_m[kWaves][16], part_l[kWaves][16];
    const PkKvCache& c = a.c;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane % 16, quad = lane / 16;
    const int page = (int)c.page, kvh = (int)c.kv_heads, hd = (int)c.hd;
    const int shift = __builtin_ctz(page);

    int begin = 0, end = 1, at, b;
    Seq s;
    if(!locate(
           c, a.N, [&](const Seq& t) { return tiles_of<R>(a, t) * kvh * (WHOLE ? 1 : units_of(t)); },
           [&](int all) {
               if(WHOLE) return (int)blockIdx.x;
               const int share = share_of(all, a.W);
               begin = (int)blockIdx.x * share;  // (at most all + share: fits)
               end = all - begin < share ? all : begin + share;
               return begin;
           },
           at, b, s))
        return;
    int tiles = tiles_of<R>(a, s), units = units_of(s);
    int item = WHOLE ? at : at / units, u0 = WHOLE ? 0 : at - item * units;

    for(int now = begin; now < end;) {
        while(item == tiles * kvh) {  // on to the next sequence that has any
            if(++b >= c.B) return;    // (there is one, unless offsets decrease)
            s = sequence(c, a.N, b);
            tiles = tiles_of<R>(a, s);
            units = units_of(s);
            item = 0;
        }
        const int u1 = WHOLE || end - now >= units - u0 ? units : u0 + (end - now);
        const int h = item / tiles, first = (item - h * tiles) * R;
        const int rows = s.n * a.group - first < R ? s.n * a.group - first : R;

        // the lane's query: row `mine` of the tile, as operand of 32 values a step, the
        // values in the order that the lane's keys come in
        const int mine = SPLIT ? col % 8 : col;
        const int token = (first + (mine < rows ? mine : 0)) / a.group;
        const float* qr = a.q + (int64_t)(s.row + token) * a.ldq +
                          (int64_t)(h * a.group + (first + (mine < rows ? mine : 0)) % a.group) * hd;
        const int reach = s.past + token;  // the last key that it sees
        // the pages of a unit's tokens: 16 tokens lie on one page.  A lane's keys (tokens
        // 16 (col / 4) + 4 t + col % 4) and its values and scores (16 quad ..) are on two.
        auto page_of = [&](int u, int g16) {
            const int i = (u * kUnit + 16 * g16) >> shift;
            const int pid = i < c.width ? c.table[(int64_t)b * c.width + i] : -1;
            return pid < 0 || pid >= c.pages ? -1 : pid;
        };
        uint4 kr[4][C > 0 ? C : 1], vr[DT];
        uint2 kt[4];
        auto load_keys = [&](int u, int pid) {
            const int slot = ((u * kUnit + 16 * (col / 4)) & (page - 1)) + col % 4;
            const uint8_t* p = c.k + (((int64_t)(pid < 0 ? 0 : pid) * kvh + h) * page + slot) * HP;
#pragma unroll
            for(int t = 0; t < 4; ++t) {
#pragma unroll
                for(int i = 0; i < C; ++i)
                    kr[t][i] = *(const uint4*)(p + 4 * t * HP + 64 * i + 16 * quad);
                if(TAIL) kt[t] = *(const uint2*)(p + 4 * t * HP + 64 * C + 8 * quad);
            }
        };
        auto load_values = [&](int u, int pid) {
            const int slot = (u * kUnit + 16 * quad) & (page - 1);
            const uint8_t* p = c.v + (((int64_t)(pid < 0 ? 0 : pid) * kvh + h) * HP + col) * page + slot;
#pragma unroll
            for(int i = 0; i < DT; ++i) vr[i] = *(const uint4*)(p + (int64_t)16 * i * page);
        };

        // (the loads that others wait for first: pages, query, then keys and values)
        int u = u0 + wave;
        int pk = -1, pv = -1;
        if(u < u1) {
            pk = page_of(u, col / 4);
            pv = page_of(u, quad);
        }
        float x[STEPS][8];
#pragma unroll
        for(int st = 0; st < STEPS; ++st) {
            const int d = TAIL && st == STEPS - 1 ? 64 * C + 8 * quad
                                                  : 64 * (st / 2) + 16 * quad + 8 * (st % 2);
            if(a.vec) {
#pragma unroll
                for(int i = 0; i < 8; i += 4) {
                    const f32x4 v = d + i < hd ? *(const f32x4*)(qr + d + i) : f32x4{};
#pragma unroll
                    for(int k = 0; k < 4; ++k) x[st][i + k] = v[k];
                }
            } else {
#pragma unroll
                for(int i = 0; i < 8; ++i) x[st][i] = d + i < hd ? qr[d + i] : 0.0f;
            }
        }
        uint8_t ek = 127, ev = 127;
        if(u < u1) {
            load_keys(u, pk);
            load_values(u, pv);
            ek = c.k_exp[(int64_t)(pv < 0 ? 0 : pv) * kvh + h];
            ev = c.v_exp[(int64_t)(pv < 0 ? 0 : pv) * kvh + h];
        }
        float amax = 0.0f;
#pragma unroll
        for(int st = 0; st < STEPS; ++st)
#pragma unroll
            for(int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[st][i]));
        amax = fmaxf(amax, __shfl_xor(amax, 16, kWave));
        amax = fmaxf(amax, __shfl_xor(amax, 32, kWave));
        const int eq = amax > 0.0f && amax <= 3.402823466e38f ? __builtin_amdgcn_frexp_expf(amax) - 15 : 0;
        const float coef = ldexpf(a.scale, eq);
        f16x8 qf[SPLIT ? 1 : 2][STEPS];
#pragma unroll
        for(int st = 0; st < STEPS; ++st)
#pragma unroll
            for(int i = 0; i < 8; ++i) {
                const float y = mine < rows ? ldexpf(x[st][i], -eq) : 0.0f;
                const _Float16 hi = (_Float16)y, lo = (_Float16)(y - (float)hi);
                if(SPLIT) {
                    qf[0][st][i] = col < 8 ? hi : lo;
                } else {
                    qf[0][st][i] = hi;
                    qf[SPLIT ? 0 : 1][st][i] = lo;
                }
            }

        f32x4 acc[DT];
#pragma unroll
        for(int i = 0; i < DT; ++i) acc[i] = f32x4{};
        float m = kNone, l = 0.0f;
        const int clear = s.past + first / a.group + 1;  // tokens that every row sees
        for(; u < u1; u += kWaves) {
            const int next = u + kWaves;
            int pk_next = -1, pv_next = -1;
            if(next < u1) {
                pk_next = page_of(next, col / 4);
                pv_next = page_of(next, quad);
            }
            f32x4 sc[4];
#pragma unroll
            for(int t = 0; t < 4; ++t) {
                sc[t] = f32x4{};
#pragma unroll
                for(int st = 0; st < STEPS; ++st) {
                    f16x8 kf;
                    if(TAIL && st == STEPS - 1)
                        kf = widen(kt[t].x, kt[t].y);
                    else if(st % 2 == 0)
                        kf = widen(kr[t][st / 2].x, kr[t][st / 2].y);
                    else
                        kf = widen(kr[t][st / 2].z, kr[t][st / 2].w);
                    sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[0][st], sc[t], 0, 0, 0);
                    if(!SPLIT)
                        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[SPLIT ? 0 : 1][st], sc[t],
                                                                       0, 0, 0);
                }
            }
            const float kc = coef * power(ek), vexp = (float)((int)ev - 127), vinv = power(254 - ev);
            const bool absent = pv < 0;
            if(next < u1) {
                load_keys(next, pk_next);
                ek = c.k_exp[(int64_t)(pv_next < 0 ? 0 : pv_next) * kvh + h];
                ev = c.v_exp[(int64_t)(pv_next < 0 ? 0 : pv_next) * kvh + h];
            }
            float p[16], mx = kNone;
#pragma unroll
            for(int t = 0; t < 4; ++t)
#pragma unroll
                for(int r = 0; r < 4; ++r) {
                    float v = sc[t][r];
                    if(SPLIT) v += across8(v);
                    p[4 * t + r] = fmaf(v, kc, vexp);
                }
            const int token0 = u * kUnit + 16 * quad;
            const bool edge = u * kUnit + kUnit > clear || __ballot(absent) != 0;
            if(edge) {
#pragma unroll
                for(int i = 0; i < 16; ++i)
                    if(absent || token0 + i > reach) p[i] = -INFINITY;
            }
#pragma unroll
            for(int i = 0; i < 16; ++i) mx = fmaxf(mx, p[i]);
            if(__ballot(mx > m + kRaise)) {
                mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
                mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
                mx = fmaxf(mx, m);
                const float down = __builtin_amdgcn_exp2f(m - mx);
                l *= down;
#pragma unroll
                for(int i = 0; i < DT; ++i) acc[i] *= down;
                m = mx;
            }
            float sum = 0.0f;
            const float low = m - kTop;
#pragma unroll
            for(int i = 0; i < 16; ++i) {
                p[i] = __builtin_amdgcn_exp2f(p[i] - low);
                sum += p[i];
            }
            l = fmaf(sum, vinv, l);
            f16x8 pf[2][2];
#pragma unroll
            for(int i = 0; i < 16; ++i) {
                const _Float16 hi = (_Float16)p[i], lo = (_Float16)(p[i] - (float)hi);
                if(SPLIT) {
                    pf[0][i / 8][i % 8] = col < 8 ? hi : lo;
                } else {
                    pf[0][i / 8][i % 8] = hi;
                    pf[1][i / 8][i % 8] = lo;
                }
            }
            if(edge) {
                // tokens behind the sequence's last, or on no page, may hold anything
                const int real = absent ? 0 : held(s.end - token0, 0, 16);
                uint32_t keep[4], nan = 0;
#pragma unroll
                for(int i = 0; i < 4; ++i) {
                    const int k = held(real - 4 * i, 0, 4);
                    keep[i] = k == 4 ? 0xffffffffu : (1u << (8 * k)) - 1u;
                }
#pragma unroll
                for(int i = 0; i < DT; ++i) {
                    vr[i].x &= keep[0];
                    vr[i].y &= keep[1];
                    vr[i].z &= keep[2];
                    vr[i].w &= keep[3];
                    nan |= nan_bytes(vr[i].x) | nan_bytes(vr[i].y) | nan_bytes(vr[i].z) | nan_bytes(vr[i].w);
                }
                if(__builtin_expect(__ballot(nan != 0) != 0, 0)) {
                    // a NaN among the values of tokens that some rows do not see, where
                    // 0 times it must not reach them: how many of a column's NaN each row
                    // sees, as a product of ones, and zeros in their place
                    f16x8 seen[2];
#pragma unroll
                    for(int i = 0; i < 16; ++i)
                        seen[i / 8][i % 8] = absent || token0 + i > reach ? (_Float16)0.0f : (_Float16)1.0f;
#pragma unroll
                    for(int i = 0; i < DT; ++i) {
                        uint32_t word[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w}, one[4];
#pragma unroll
                        for(int k = 0; k < 4; ++k) {
                            const uint32_t bits = nan_bytes(word[k]) >> 7;
                            one[k] = bits * 0x38;  // e4m3's 1
                            word[k] &= ~(bits * 0xff);
                        }
                        f32x4 count = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen(one[0], one[1]), seen[0],
                                                                             f32x4{}, 0, 0, 0);
                        count = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen(one[2], one[3]), seen[1], count,
                                                                       0, 0, 0);
#pragma unroll
                        for(int r = 0; r < 4; ++r)
                            if(count[r] > 0.0f) acc[i][r] = NAN;
                        vr[i] = {word[0], word[1], word[2], word[3]};
                    }
                }
            }
#pragma unroll
            for(int i = 0; i < DT; ++i) {
                const f16x8 v0 = widen(vr[i].x, vr[i].y), v1 = widen(vr[i].z, vr[i].w);
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[0][0], acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[0][1], acc[i], 0, 0, 0);
                if(!SPLIT) {
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[1][0], acc[i], 0, 0, 0);
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[1][1], acc[i], 0, 0, 0);
                }
            }
            if(next < u1) load_values(next, pv_next);
            pv = pv_next;
        }

        // the waves' parts together
        l += __shfl_xor(l, 16, kWave);
        l += __shfl_xor(l, 32, kWave);
#pragma unroll
        for(int i = 0; i < DT; ++i) {
            if(SPLIT) {
#pragma unroll
                for(int r = 0; r < 4; ++r) acc[i][r] += across8(acc[i][r]);
            }
            if(col < R) *(f32x4*)&part[wave][col][16 * i + 4 * quad] = acc[i];
        }
        if(lane < 16) {
            part_m[wave][lane] = m;
            part_l[wave][lane] = l;
        }
        __syncthreads();
        const bool whole = WHOLE || (u0 == 0 && u1 == units);
        float* out = a.ws + ((int64_t)blockIdx.x * 2 + (now == begin ? 0 : 1)) * kPart<HP>;
        for(int i = threadIdx.x; i < rows * (HP / 4); i += kWaves * kWave) {
            const int r = i / (HP / 4), d = 4 * (i % (HP / 4));
            float top = part_m[0][r], total = 0.0f;
#pragma unroll
            for(int k = 1; k < kWaves; ++k) top = fmaxf(top, part_m[k][r]);
            f32x4 v = {};
#pragma unroll
            for(int k = 0; k < kWaves; ++k) {
                const float f = __builtin_amdgcn_exp2f(part_m[k][r] - top);
                total = fmaf(f, part_l[k][r], total);
                v += f * *(const f32x4*)&part[k][r][d];
            }
            if(!whole) {
                if(d == 0) {
                    out[r] = top;
                    out[16 + r] = total;
                }
                *(f32x4*)(out + 32 + r * HP + d) = v;
                continue;
            }
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;  // (0: no key at all)
            float* to = a.o + (int64_t)(s.row + (first + r) / a.group) * a.ldo +
                        (int64_t)(h * a.group + (first + r) % a.group) * hd + d;
#pragma unroll
            for(int k = 0; k < 4; ++k)
                if(d + k < hd) to[k] = v[k] * inv;
        }
        __syncthreads();
        now += u1 - u0;
        u0 = 0;
        ++item;
    }
}

// The tiles that several workgroups have parts of: a workgroup here stands for the one
// there that has a tile's last part, and a wave for one of the tile's rows, its lanes on 4
// values each of as many parts at once as there are lanes for.
template <int HP, int R>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a) {
    constexpr int D4 = HP / 4, PARTS = kWave / D4;
    const PkKvCache& c = a.c;
    const int lane = threadIdx.x % kWave, r = blockIdx.y * 4 + threadIdx.x / kWave;
    int share = 1, at, b;
    Seq s;
    if(!locate(
           c, a.N, [&](const Seq& t) { return tiles_of<R>(a, t) * (int)c.kv_heads * units_of(t); },
           [&](int all) {
               share = share_of(all, a.W);
               return (int)blockIdx.x * share;
           },
           at, b, s))
        return;
    const int tiles = tiles_of<R>(a, s), units = units_of(s), item = at / units, u0 = at - item * units;
    if(u0 == 0 || units - u0 > share) return;  // it begins here, or has parts behind
    const int h = item / tiles, row = (item - h * tiles) * R + r;
    if(row >= s.n * a.group) return;
    // the first part's workgroup, where it is in that one's place 0 if it begins its share
    const int before = (u0 + share - 1) / share, w1 = blockIdx.x, w0 = w1 - before;
    if(w0 < 0) return;  // (offsets that decrease)
    const int first_place = before * share == u0 ? 0 : 1;
    auto part = [&](int w) { return a.ws + ((int64_t)w * 2 + (w == w0 ? first_place : 0)) * kPart<HP>; };
    float top = kNone;
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
            total = fmaf(f, p[16 + r], total);
            v += f * *(const f32x4*)(p + 32 + r * HP + d);
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
    float* to = a.o + (int64_t)(s.row + row / a.group) * a.ldo + (int64_t)(h * a.group + row % a.group) * c.hd + d;
#pragma unroll
    for(int k = 0; k < 4; ++k)
        if(d + k < c.hd) to[k] = sum[k] * inv;
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
    const int token = real_row / a.group;
    const float* qr = a.q + (int64_t)(s.row + token) * a.ldq + (int64_t)(h * a.group + real_row % a.group) * hd;
    const int reach = s.past + token;
    f16x8 qh[STEPS], ql[STEPS];
    float coef;
    {
        float x[STEPS][8], amax = 0.0f;
#pragma unroll
        for(int st = 0; st < STEPS; ++st) {
            const int d = 32 * (st / 2) + 16 * half + 8 * (st % 2);
            if(a.vec) {
#pragma unroll
                for(int i = 0; i < 8; i += 4) {
                    const f32x4 v = d + i < hd ? *(const f32x4*)(qr + d + i) : f32x4{};
#pragma unroll
                    for(int k = 0; k < 4; ++k) x[st][i + k] = v[k];
                }
            } else {
#pragma unroll
                for(int i = 0; i < 8; ++i) x[st][i] = d + i < hd ? qr[d + i] : 0.0f;
            }
#pragma unroll
            for(int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[st][i]));
        }
        amax = fmaxf(amax, __shfl_xor(amax, 32, kWave));
        const int eq = amax > 0.0f && amax <= 3.402823466e38f ? __builtin_amdgcn_frexp_expf(amax) - 15 : 0;
        coef = ldexpf(a.scale, eq);
#pragma unroll
        for(int st = 0; st < STEPS; ++st)
#pragma unroll
            for(int i = 0; i < 8; ++i) {
                const float y = col < rows ? ldexpf(x[st][i], -eq) : 0.0f;
                qh[st][i] = (_Float16)y;
                ql[st][i] = (_Float16)(y - (float)qh[st][i]);
            }
    }

    auto page_of = [&](int u, int g16) {
        const int i = (u * kUnit + 16 * g16) >> shift;
        const int pid = u < u1 && i < c.width ? c.table[(int64_t)b * c.width + i] : -1;
        return pid < 0 || pid >= c.pages ? -1 : pid;
    };
    // a thread's chunks: of keys, 16 values of token e / (HP / 16); of values, 16 tokens of
    // row e / 4, of which `real` are the sequence's
    int pk[LOADS], pv, real = 0;
    uint4 kr[LOADS], vr[LOADS];
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
                kr[i] = *(const uint4*)(c.k + (k_head * page + ((u * kUnit + t) & (page - 1))) * HP + 16 * d16);
                vr[i] = *(const uint4*)(c.v + (v_head * HP + e / 4) * page +
                                        ((u * kUnit + 16 * g16) & (page - 1)));
            }
        }
        if(threadIdx.x < 4) {
            const uint8_t ek = c.k_exp[v_head], ev = c.v_exp[v_head];
            pr = {power(ek), (float)((int)ev - 127), power(254 - ev), pv < 0 ? 0.0f : 1.0f};
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
                *(uint4*)&keys[buf][row * KS + 16 * d16] = kr[i];
                if(real < 16) {  // values behind the sequence's end, or on no page, may be anything
                    uint32_t w[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
#pragma unroll
                    for(int k = 0; k < 4; ++k) {
                        const int n = held(real - 4 * k, 0, 4);
                        w[k] &= n == 4 ? 0xffffffffu : (1u << (8 * n)) - 1u;
                    }
                    vr[i] = {w[0], w[1], w[2], w[3]};
                }
                *(uint4*)&values[buf][e / 4 * VS + 16 * g16] = vr[i];
            }
        }
        if(threadIdx.x < 4) pages[buf][threadIdx.x] = pr;
    };

    f32x16 acc[DT];
#pragma unroll
    for(int i = 0; i < DT; ++i) acc[i] = f32x16{};
    float m = kNone, l = 0.0f;
    const int clear = s.past + (first < total ? first / a.group : 0) + 1;  // tokens that all rows see
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
            f32x16 sc = {};
#pragma unroll
            for(int st = 0; st < STEPS; st += 2) {
                const uint4 w = *(const uint4*)&keys[buf][(32 * j + col) * KS + 16 * st + 16 * half];
                const f16x8 k0 = widen(w.x, w.y), k1 = widen(w.z, w.w);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, qh[st], sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, qh[st + 1], sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, ql[st], sc, 0, 0, 0);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, ql[st + 1], sc, 0, 0, 0);
            }
            const float4 g = pages[buf][2 * j + half];
            const float kc = coef * g.x;
            const bool absent = g.w == 0.0f;
            const int mine0 = token0 + 16 * half;
            float p[16], mx = kNone;
#pragma unroll
            for(int i = 0; i < 16; ++i) p[i] = fmaf(sc[i], kc, g.y);
            const bool edge = token0 + 32 > clear || __ballot(absent) != 0;
            if(edge) {
#pragma unroll
                for(int i = 0; i < 16; ++i)
                    if(absent || mine0 + i > reach) p[i] = -INFINITY;
            }
#pragma unroll
            for(int i = 0; i < 16; ++i) mx = fmaxf(mx, p[i]);
            if(__ballot(mx > m + kRaise)) {
                mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
                mx = fmaxf(mx, m);
                const float down = __builtin_amdgcn_exp2f(m - mx);
                l *= down;
#pragma unroll
                for(int i = 0; i < DT; ++i) acc[i] *= down;
                m = mx;
            }
            const float low = m - kTop;
            float sum = 0.0f;
            f16x8 ph[2], pl[2];
#pragma unroll
            for(int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(p[i] - low);
                sum += e;
                ph[i / 8][i % 8] = (_Float16)e;
                pl[i / 8][i % 8] = (_Float16)(e - (float)ph[i / 8][i % 8]);
            }
            l = fmaf(sum, g.z, l);
#pragma unroll
            for(int i = 0; i < DT; ++i) {
                uint4 w = *(const uint4*)&values[buf][(32 * i + col) * VS + 32 * j + 16 * half];
                if(edge) {
                    const uint32_t nan = nan_bytes(w.x) | nan_bytes(w.y) | nan_bytes(w.z) | nan_bytes(w.w);
                    if(__builtin_expect(__ballot(nan != 0) != 0, 0)) {
                        // (as in few_rows_kernel: the NaN that a row sees, counted)
                        uint32_t word[4] = {w.x, w.y, w.z, w.w}, one[4];
                        f16x8 seen[2];
#pragma unroll
                        for(int k = 0; k < 16; ++k)
                            seen[k / 8][k % 8] = absent || mine0 + k > reach ? (_Float16)0.0f : (_Float16)1.0f;
#pragma unroll
                        for(int k = 0; k < 4; ++k) {
                            const uint32_t bits = nan_bytes(word[k]) >> 7;
                            one[k] = bits * 0x38;
                            word[k] &= ~(bits * 0xff);
                        }
                        f32x16 count = __builtin_amdgcn_mfma_f32_32x32x16_f16(widen(one[0], one[1]), seen[0],
                                                                              f32x16{}, 0, 0, 0);
                        count = __builtin_amdgcn_mfma_f32_32x32x16_f16(widen(one[2], one[3]), seen[1], count,
                                                                       0, 0, 0);
#pragma unroll
                        for(int r = 0; r < 16; ++r)
                            if(count[r] > 0.0f) acc[i][r] = NAN;
                        w = {word[0], word[1], word[2], word[3]};
                    }
                }
                const f16x8 v0 = widen(w.x, w.y), v1 = widen(w.z, w.w);
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
    if(a.splits > 1) {  // (a part without units has the maximum of no scores, and zeros)
        float* out = a.ws + (int64_t)blockIdx.x * kManyPart<HP>;
        const int r = wave * 32 + col;
        if(half == 0) {
            out[r] = m;
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
    float* to = a.o + (int64_t)(s.row + token) * a.ldo + (int64_t)(h * a.group + row % a.group) * hd;
#pragma unroll
    for(int i = 0; i < DT; ++i)
#pragma unroll
        for(int q = 0; q < 4; ++q)
#pragma unroll
            for(int k = 0; k < 4; ++k) {
                const int d = 32 * i + 8 * q + 4 * half + k;
                if(d < hd) to[d] = acc[i][4 * q + k] * inv;
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
    float top = kNone, total = 0.0f;
    for(int i = 0; i < a.splits; ++i) top = fmaxf(top, base[i * apart + r]);
    const int d = 4 * lane;
    f32x4 v = {};
    for(int i = 0; i < a.splits; ++i) {
        const float* p = base + i * apart;
        const float f = __builtin_amdgcn_exp2f(p[r] - top);
        total = fmaf(f, p[kRows + r], total);
        if(lane < D4) v += f * *(const f32x4*)(p + 2 * kRows + r * HP + d);
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    float* to = a.o + (int64_t)(s.row + row / a.group) * a.ldo + (int64_t)(h * a.group + row % a.group) * c.hd + d;
#pragma unroll
    for(int k = 0; k < 4; ++k)
        if(lane < D4 && d + k < c.hd) to[k] = v[k] * inv;
}

// ------------------------------------------------------------------- launches
struct Plan {
    int rows;       // 8, 16 or 128 query rows a tile
    int W;          // of few rows: workgroups that share the units of all tiles; 0: one to a tile
    int splits;     // of many: workgroups to a tile
    int64_t tiles;  // for each head of the cache, that there may be
};
Plan plan(const PkKvCache* c, int64_t N, int64_t H) {
    Plan p = {};
    const int64_t group = H / c->kv_heads, units = (c->width * c->page + kUnit - 1) / kUnit;
    const int64_t some = c->B < N ? c->B : N;
    p.rows = N * group <= 8 * c->B ? 8 : N * group <= 32 * c->B ? 16 : kRows;
    p.tiles = N * group / p.rows + some;
    if(p.rows < kRows) {
        p.W = units <= 32 || p.tiles * c->kv_heads * units >= (int64_t)1 << 31 ? 0 : 512;
    } else {
        // workgroups that there are for sure, two to a CU, of 8 units at least
        const int64_t sure = (N * group + kRows - 1) / kRows * c->kv_heads;
        int64_t n = 512 / sure;
        if(n > units / 8) n = units / 8;
        p.splits = (int)(n < 1 ? 1 : n > 16 ? 16 : n);
    }
    return p;
}
size_t plan_bytes(const Plan& p, const PkKvCache* c) {
    const size_t hp = head_size(c->hd);
    if(p.W) return sizeof(float) * 2 * p.W * (32 + 16 * hp);
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

template <int HP, bool SPLIT>
void launch_rows(const AttnArgs& a, const Plan& p, hipStream_t st) {
    if(!p.W) {
        few_rows_kernel<HP, SPLIT, true>
            <<<(unsigned)(p.tiles * a.c.kv_heads), waves_of(HP, true) * kWave, 0, st>>>(a);
        return;
    }
    few_rows_kernel<HP, SPLIT, false><<<(unsigned)p.W, 256, 0, st>>>(a);
    join_kernel<HP, SPLIT ? 8 : 16><<<dim3((unsigned)p.W, SPLIT ? 2 : 4), 256, 0, st>>>(a);
}
template <int HP>
void launch(const AttnArgs& a, const Plan& p, hipStream_t st) {
    if(p.rows == 8) return launch_rows<HP, true>(a, p, st);
    if(p.rows == 16) return launch_rows<HP, false>(a, p, st);
    const int64_t tiles = p.tiles * a.c.kv_heads;
    many_rows_kernel<HP><<<(unsigned)(tiles * p.splits), 256, 0, st>>>(a);
    if(p.splits > 1) finish_kernel<HP><<<dim3((unsigned)tiles, kRows / 4), 256, 0, st>>>(a);
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
    if(!grid_fits(p.tiles * cache->kv_heads * (p.splits > 1 ? p.splits : 1), 512))
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
    a.vec = cache->hd % 4 == 0 && ldq % 4 == 0 && aligned16(q);
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
