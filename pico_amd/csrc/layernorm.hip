// pico_amd/csrc/layernorm.hip -- layer norm over rows of [R, C] and its gradients.
//
//   y = (x - m) r g + b,  m = mean(x),  r = (mean((x - m)^2) + eps)^-1/2
//   xh = (x - m) r
//   dx = r (g dy - mean(g dy) - xh mean(g dy xh))
//   dg = sum over rows of dy xh,  db = sum over rows of dy
//
// Bound by memory: 8 bytes a value forward, 12 backward, each row read once and
// kept in registers between the sums and the result.  W waves share a row, NV 4-value
// vectors a lane; the mean and the squares around it are each wave's own, put
// together as
//   M2 = sum of M2_w + n_w (m_w - m)^2
// so that a row takes one exchange through LDS and no difference of squares.  128-bit
// accesses at any 4-byte alignment; of a row whose length is no multiple of 4 the
// last lane reads the last 4 values and leaves those before its own out.
#include <type_traits>

#include "pk_common.h"

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// (plain loads and nontemporal stores: with nontemporal loads 8192x4096 took 48 + 78 us
// forward and backward, with these 41 + 73, now 41 + 66)
__device__ __forceinline__ f32x4 load4(const float* p) { return *reinterpret_cast<const f32x4u*>(p); }

// A lane's share of a row: vector v starts at column `at[v]` and holds `skip[v]` values
// (0 to 3) of the lane before it, or lies past the row (4).  EXACT: every vector
// is whole.
template <int NV, int W, bool EXACT>
struct Share {
    int at[NV], skip[NV];
    float count;  // the wave's values

    __device__ __forceinline__ explicit Share(int C) {
        const int t = threadIdx.x % (64 * W);
        int mine = 0;
#pragma unroll
        for(int v = 0; v < NV; ++v) {
            const int c = 4 * (v * 64 * W + t);
            at[v] = EXACT ? c : min(c, C - 4);
            skip[v] = EXACT ? 0 : min(c - at[v], 4);
            mine += 4 - skip[v];
        }
        count = EXACT ? 256.0f * NV : pk::wave_sum((float)mine);
    }
    __device__ __forceinline__ void load(const float* row, f32x4 (&x)[NV]) const {
#pragma unroll
        for(int v = 0; v < NV; ++v) x[v] = load4(row + at[v]);
    }
    // whether value i of vector v is the lane's own
    __device__ __forceinline__ bool own(int v, int i) const { return EXACT || i >= skip[v]; }
    __device__ __forceinline__ void store(float* row, int v, f32x4 y) const {
        if(EXACT || skip[v] == 0) {
            __builtin_nontemporal_store(y, reinterpret_cast<f32x4u*>(row + at[v]));
        } else {
#pragma unroll
            for(int i = 1; i < 4; ++i)
                if(i >= skip[v]) row[at[v] + i] = y[i];
        }
    }
};

// rows of W waves each, 4 / W of them in a workgroup of 4 waves, the next one's
// values in flight
template <int NV, int W, bool EXACT>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256) void layernorm_fwd(int R, int C, float eps,
                                                                      const float* __restrict__ x,
                                                                      const float* __restrict__ g,
                                                                      const float* __restrict__ b,
                                                                      float* __restrict__ y,
                                                                      float* __restrict__ mean,
                                                                      float* __restrict__ rstd) {
    constexpr int ROWS = W > 4 ? 1 : 4 / W;
    __shared__ float part[2][ROWS][W][3];
    const Share<NV, W, EXACT> me(C);
    const int group = threadIdx.x / (64 * W), w = threadIdx.x / 64 % W;
    const int64_t step = (int64_t)gridDim.x * ROWS;
    int64_t row = (int64_t)blockIdx.x * ROWS + group;
    f32x4 cur[NV], next[NV];
    if(W > 1 || row < R) me.load(x + min(row, (int64_t)R - 1) * C, cur);
    // (the waves of a workgroup meet in every turn, so all take the same ones)
    for(int turn = 0; row - group < R; row += step, turn ^= 1) {
        if(W == 1 && row >= R) return;
        // (of one wave's rows the last is read twice: with a load that a branch may leave
        // out, the waits for this row's values wait for the next one's.  65536x512 us 39.5
        // against 41; of several waves, which wait for each other, 8192x4096 43.3 against
        // 41.0)
        const int64_t after = min(row + step, (int64_t)R - 1);
        if(W == 1 || row - group + step < R) me.load(x + after * C, next);
        float s = 0.0f;
#pragma unroll
        for(int v = 0; v < NV; ++v)
#pragma unroll
            for(int i = 0; i < 4; ++i) s += me.own(v, i) ? cur[v][i] : 0.0f;
        float m = pk::wave_sum(s) / me.count, q = 0.0f;
        if(!EXACT && me.count == 0.0f) m = 0.0f;
#pragma unroll
        for(int v = 0; v < NV; ++v)
#pragma unroll
            for(int i = 0; i < 4; ++i) {
                const float d = me.own(v, i) ? cur[v][i] - m : 0.0f;
                q = fmaf(d, d, q);
            }
        q = pk::wave_sum(q);
        if constexpr(W > 1) {
            if(threadIdx.x % 64 == 0) {
                part[turn][group][w][0] = me.count;
                part[turn][group][w][1] = m;
                part[turn][group][w][2] = q;
            }
            __syncthreads();
            s = 0.0f;
#pragma unroll
            for(int i = 0; i < W; ++i) s = fmaf(part[turn][group][i][0], part[turn][group][i][1], s);
            m = s / (float)C;
            q = 0.0f;
#pragma unroll
            for(int i = 0; i < W; ++i) {
                const float d = part[turn][group][i][1] - m;
                q += fmaf(part[turn][group][i][0] * d, d, part[turn][group][i][2]);
            }
        }
        const float r = 1.0f / sqrtf(q / (float)C + eps);
        if(row < R) {
            if(threadIdx.x % (64 * W) == 0) {
                if(mean) mean[row] = m;
                if(rstd) rstd[row] = r;
            }
            float* const yr = y + row * C;
#pragma unroll
            for(int v = 0; v < NV; ++v) {
                if(!EXACT && me.skip[v] == 4) continue;
                f32x4 o = (cur[v] - m) * r * load4(g + me.at[v]);
                if(b) o = o + load4(b + me.at[v]);
                me.store(yr, v, o);
            }
        }
#pragma unroll
        for(int v = 0; v < NV; ++v) cur[v] = next[v];
    }
}

// dx of every row, and the workgroup's part of dg and db in ws [P][2][C]: a workgroup of 8 waves walks rows 8 / W at a time, its
// lanes keeping the sums of their own columns; at the end the row groups' sums meet
// in LDS, in a fixed order.
constexpr int kBwdWaves = 8;
enum { kDx = 1, kSums = 2 };

template <int NV, int W, bool EXACT, bool IN>
__global__ __launch_bounds__(64 * kBwdWaves) void layernorm_bwd(
    int R, int C, const float* __restrict__ x, const float* __restrict__ g,
    const float* __restrict__ mean, const float* __restrict__ rstd, const float* __restrict__ dy,
    const float* dxin, float* dx, float* __restrict__ ws, int what) {
    constexpr int ROWS = kBwdWaves / W;
    __shared__ float part[2][ROWS][W][2];
    extern __shared__ float sums[];  // [ROWS / 2][2][C]
    const Share<NV, W, EXACT> me(C);
    const int group = threadIdx.x / (64 * W), w = threadIdx.x / 64 % W;
    const int64_t step = (int64_t)gridDim.x * ROWS;
    f32x4 gv[NV], sg[NV], sb[NV], xc[NV], dc[NV], xn[NV], dn[NV];
#pragma unroll
    for(int v = 0; v < NV; ++v) {
        gv[v] = load4(g + me.at[v]);
#pragma unroll
        for(int i = 0; i < 4; ++i) gv[v][i] = me.own(v, i) ? gv[v][i] : 0.0f;
        sg[v] = sb[v] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int64_t row = (int64_t)blockIdx.x * ROWS + group;
    float m, r, mn, rn;
    auto fetch = [&](int64_t r, f32x4 (&a)[NV], f32x4 (&d)[NV]) {
        r = min(r, (int64_t)R - 1);
        me.load(x + r * C, a);
        me.load(dy + r * C, d);
        mn = mean[r];
        rn = rstd[r];
    };
    // (8 vectors of every array leave no registers for the next row's)
    constexpr bool AHEAD = NV <= 4;
    if(AHEAD) {
        fetch(row, xc, dc);
        m = mn;
        r = rn;
    }
    for(int turn = 0; row - group < R; row += step, turn ^= 1) {
        // (before the next row's loads: those behind would be waited for with it.  In place,
        // 8192x4096 104 us, with the loads at their use 108; 2000x16384 109 and 122)
        f32x4 in[NV];
        if constexpr(IN) me.load(dxin + min(row, (int64_t)R - 1) * C, in);
        if(AHEAD) {
            // (a last row is read twice: with a load that a branch may leave out, the
            // waits for this row's values wait for the next one's; 8192x4096 66 us, so
            // 73, but 100x4096 10.3 and so 9.7)
            fetch(row - group + step < R ? row + step : row, xn, dn);
        } else {
            fetch(row, xc, dc);
            m = mn;
            r = rn;
        }
        const bool on = row < R;
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for(int v = 0; v < NV; ++v) {
            xc[v] = (xc[v] - m) * r;
#pragma unroll
            for(int i = 0; i < 4; ++i) {
                // (g is 0 where the value is not the lane's, which an infinity or NaN
                // there would not respect)
                const float t = me.own(v, i) ? gv[v][i] * dc[v][i] : 0.0f;
                s1 += t;
                s2 = fmaf(t, me.own(v, i) ? xc[v][i] : 0.0f, s2);
            }
        }
        if(what & kDx) {
            s1 = pk::wave_sum(s1);
            s2 = pk::wave_sum(s2);
            if constexpr(W > 1) {
                if(threadIdx.x % 64 == 0) {
                    part[turn][group][w][0] = s1;
                    part[turn][group][w][1] = s2;
                }
                __syncthreads();
                s1 = s2 = 0.0f;
#pragma unroll
                for(int i = 0; i < W; ++i) {
                    s1 += part[turn][group][i][0];
                    s2 += part[turn][group][i][1];
                }
            }
            s1 /= (float)C;
            s2 /= (float)C;
        }
#pragma unroll
        for(int v = 0; v < NV; ++v) {
            if(!on || (!EXACT && me.skip[v] == 4)) continue;
            sg[v] = sg[v] + dc[v] * xc[v];
            sb[v] = sb[v] + dc[v];
            if(what & kDx) {
                f32x4 o = r * (gv[v] * dc[v] - s1 - xc[v] * s2);
                if constexpr(IN) o = o + in[v];
                me.store(dx + row * C, v, o);
            }
        }
        if(AHEAD) {
#pragma unroll
            for(int v = 0; v < NV; ++v) {
                xc[v] = xn[v];
                dc[v] = dn[v];
            }
            m = mn;
            r = rn;
        }
    }
    if(!(what & kSums)) return;
    // the row groups' sums, by halves: the upper half puts its own down, the lower
    // adds them (a column belongs to one lane of every group)
#pragma unroll
    for(int half = ROWS / 2; half > 0; half /= 2) {
        float* const slot = sums + (int64_t)(group % half) * 2 * C;
        if(half < ROWS / 2) __syncthreads();
        if(group >= half && group < 2 * half) {
#pragma unroll
            for(int v = 0; v < NV; ++v)
#pragma unroll
                for(int i = 0; i < 4; ++i) {
                    if(!me.own(v, i)) continue;
                    slot[me.at[v] + i] = sg[v][i];
                    slot[C + me.at[v] + i] = sb[v][i];
                }
        }
        __syncthreads();
        if(group < half) {
#pragma unroll
            for(int v = 0; v < NV; ++v)
#pragma unroll
                for(int i = 0; i < 4; ++i) {
                    if(!me.own(v, i)) continue;
                    sg[v][i] += slot[me.at[v] + i];
                    sb[v][i] += slot[C + me.at[v] + i];
                }
        }
    }
    if(group != 0) return;
#pragma unroll
    for(int v = 0; v < NV; ++v)
#pragma unroll
        for(int i = 0; i < 4; ++i) {
            if(!me.own(v, i)) continue;
            float* const out = ws + (int64_t)blockIdx.x * 2 * C + me.at[v] + i;
            out[0] = sg[v][i];
            out[C] = sb[v][i];
        }
}

// ------------------------------------------------------------ few values
// dx, dg and db in one launch, where x and dy are so few that reading them twice costs
// less than a second launch: the first row_blocks workgroups have the rows' dx, NW waves
// to a row, the others the sums over all rows of `cols` columns each (16 to 64, a power of
// two, fewer of narrower rows), their threads a row apart, added in a fixed order.
constexpr int kFewThreads = 512;

template <int NW>
__global__ __launch_bounds__(kFewThreads) void layernorm_bwd_few(
    int R, int C, int row_blocks, int cols, const float* __restrict__ x, const float* __restrict__ g,
    const float* __restrict__ mean, const float* __restrict__ rstd, const float* __restrict__ dy,
    const float* dxin, float* dx, float* dg, float* db, int flags) {
    __shared__ float part[2][kFewThreads];
    const int t = threadIdx.x;
    if((int)blockIdx.x < row_blocks) {
        const int row = blockIdx.x * (kFewThreads / 64 / NW) + t / (64 * NW), at = t % (64 * NW);
        if(NW == 1 && row >= R) return;  // (of several waves each workgroup has one row)
        const float *xr = x + row * C, *dr = dy + row * C;
        const float m = mean[row], r = rstd[row];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll 2
        for(int c = at; c < C; c += 64 * NW) {
            const float v = g[c] * dr[c];
            s1 += v;
            s2 = fmaf(v, (xr[c] - m) * r, s2);
        }
        if constexpr(NW == 1) {
            s1 = pk::wave_sum(s1);
            s2 = pk::wave_sum(s2);
        } else {
            s1 = pk::block_sum<NW>(s1, part[0]);
            s2 = pk::block_sum<NW>(s2, part[1]);
        }
        s1 /= (float)C;
        s2 /= (float)C;
#pragma unroll 2
        for(int c = at; c < C; c += 64 * NW) {
            const float v = r * (g[c] * dr[c] - s1 - (xr[c] - m) * r * s2);
            dx[row * C + c] = dxin ? dxin[row * C + c] + v : v;
        }
        return;
    }
    const int c = ((int)blockIdx.x - row_blocks) * cols + t % cols;
    float sg = 0.0f, sb = 0.0f;
    if(c < C) {
#pragma unroll 4
        for(int row = t / cols; row < R; row += kFewThreads / cols) {
            const float d = dy[row * C + c];
            sg = fmaf(d, (x[row * C + c] - mean[row]) * rstd[row], sg);
            sb += d;
        }
    }
    part[0][t] = sg;
    part[1][t] = sb;
    for(int o = kFewThreads / 2; o >= cols; o /= 2) {
        __syncthreads();
        if(t < o) {
            part[0][t] += part[0][t + o];
            part[1][t] += part[1][t + o];
        }
    }
    if(t >= cols || c >= C) return;
    if(dg) dg[c] = (flags & PK_ACCUM2) ? dg[c] + part[0][t] : part[0][t];
    if(db) db[c] = (flags & PK_ACCUM3) ? db[c] + part[1][t] : part[1][t];
}

// ------------------------------------- rows of fewer than 4 or too many values
// a row to NW waves, read again for every sum
template <int NW>
__global__ __launch_bounds__(64 * NW) void layernorm_fwd_any(int64_t C, float eps,
                                                             const float* __restrict__ x,
                                                             const float* __restrict__ g,
                                                             const float* __restrict__ b,
                                                             float* __restrict__ y,
                                                             float* __restrict__ mean,
                                                             float* __restrict__ rstd) {
    __shared__ float red[NW];
    const int64_t row = blockIdx.x;
    const float* xr = x + row * C;
    float s = 0.0f;
    for(int64_t c = threadIdx.x; c < C; c += 64 * NW) s += xr[c];
    const float m = pk::block_sum<NW>(s, red) / (float)C;
    s = 0.0f;
    for(int64_t c = threadIdx.x; c < C; c += 64 * NW) s = fmaf(xr[c] - m, xr[c] - m, s);
    const float r = 1.0f / sqrtf(pk::block_sum<NW>(s, red) / (float)C + eps);
    if(threadIdx.x == 0) {
        if(mean) mean[row] = m;
        if(rstd) rstd[row] = r;
    }
    for(int64_t c = threadIdx.x; c < C; c += 64 * NW)
        y[row * C + c] = (xr[c] - m) * r * g[c] + (b ? b[c] : 0.0f);
}

template <int NW>
__global__ __launch_bounds__(64 * NW) void layernorm_dx_any(int64_t C, const float* __restrict__ x,
                                                            const float* __restrict__ g,
                                                            const float* __restrict__ mean,
                                                            const float* __restrict__ rstd,
                                                            const float* __restrict__ dy,
                                                            const float* dxin, float* dx) {
    __shared__ float red[2][NW];
    const int64_t row = blockIdx.x;
    const float* xr = x + row * C;
    const float* dr = dy + row * C;
    const float m = mean[row], r = rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for(int64_t c = threadIdx.x; c < C; c += 64 * NW) {
        const float t = g[c] * dr[c];
        s1 += t;
        s2 += t * ((xr[c] - m) * r);
    }
    s1 = pk::block_sum<NW>(s1, red[0]) / (float)C;
    s2 = pk::block_sum<NW>(s2, red[1]) / (float)C;
    for(int64_t c = threadIdx.x; c < C; c += 64 * NW) {
        const float v = r * (g[c] * dr[c] - s1 - (xr[c] - m) * r * s2);
        dx[row * C + c] = dxin ? dxin[row * C + c] + v : v;
    }
}

// the partial sums of dg and db over every gridDim.y-th row: ws [P][2][C]
__global__ __launch_bounds__(256) void layernorm_parts_any(int64_t R, int64_t C,
                                                           const float* __restrict__ x,
                                                           const float* __restrict__ mean,
                                                           const float* __restrict__ rstd,
                                                           const float* __restrict__ dy,
                                                           float* __restrict__ ws) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if(c >= C) return;
    float sg = 0.0f, sb = 0.0f;
    for(int64_t row = blockIdx.y; row < R; row += gridDim.y) {
        const float d = dy[row * C + c];
        sg += d * ((x[row * C + c] - mean[row]) * rstd[row]);
        sb += d;
    }
    float* out = ws + (int64_t)blockIdx.y * 2 * C;
    out[c] = sg;
    out[C + c] = sb;
}

// dg (+)= and db (+)= the sums of the P partials, in a fixed order: 64 columns of
// [2 C] per block, its 16 waves each summing every 16th partial
constexpr int kSumWaves = 16;
__global__ __launch_bounds__(64 * kSumWaves) void layernorm_sum(int64_t P, int64_t C,
                                                              const float* __restrict__ ws,
                                                              float* __restrict__ dg,
                                                              float* __restrict__ db, int flags) {
    __shared__ float part[kSumWaves][64];
    const int w = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    float acc = 0.0f;
    if(c < 2 * C) {
#pragma unroll 8
        for(int64_t p = w; p < P; p += kSumWaves) acc += ws[p * 2 * C + c];
    }
    part[w][lane] = acc;
    __syncthreads();
    if(w != 0 || c >= 2 * C) return;
    float s = part[0][lane];
#pragma unroll
    for(int i = 1; i < kSumWaves; ++i) s += part[i][lane];
    float* out = c < C ? dg : db;
    if(!out) return;
    float* o = out + (c < C ? c : c - C);
    *o = (flags & (c < C ? PK_ACCUM2 : PK_ACCUM3)) ? *o + s : s;
}

// f(NV, W, EXACT) for rows of C values, 4 <= C <= 16384: up to 4 vectors a lane, and as
// few waves as hold the row so (33.5 million values forward, us: C 512 2 vectors of one
// wave 41, 1 of two 55; 1024 4x1 41, 2x2 41, 1x4 55; 2048 4x2 41, 2x4 41, 2x8 62;
// 4096 4x4 40, 2x8 46).  The backward has two waves from C 769 on (1024 2x2 64.0, 4x1
// 66.4, with bounds 64.2 and 69.5; 768 3x1 65.5, 2x2 64.1).
template <bool BWD, class F>
void with_shape(int64_t C, F f) {
    auto shape = [&](auto nv, auto w) {
        constexpr int N = decltype(nv)::value, W = decltype(w)::value;
        if(C == 256 * N * W) f(nv, w, std::true_type());
        else f(nv, w, std::false_type());
    };
    using std::integral_constant;
    const int64_t v = (C + 255) / 256;  // vectors a lane of one wave would have
    if(v <= 1) shape(integral_constant<int, 1>(), integral_constant<int, 1>());
    else if(v <= 2) shape(integral_constant<int, 2>(), integral_constant<int, 1>());
    else if(v <= 3) shape(integral_constant<int, 3>(), integral_constant<int, 1>());
    else if(v <= 4) shape(integral_constant<int, BWD ? 2 : 4>(), integral_constant<int, BWD ? 2 : 1>());
    else if(v <= 6) shape(integral_constant<int, 3>(), integral_constant<int, 2>());
    else if(v <= 8) shape(integral_constant<int, 4>(), integral_constant<int, 2>());
    else if(v <= 12) shape(integral_constant<int, 3>(), integral_constant<int, 4>());
    else if(v <= 16) shape(integral_constant<int, 4>(), integral_constant<int, 4>());
    else if(v <= 24) shape(integral_constant<int, 3>(), integral_constant<int, 8>());
    else if(v <= 32) shape(integral_constant<int, 4>(), integral_constant<int, 8>());
    else shape(integral_constant<int, 8>(), integral_constant<int, 8>());
}

bool cached(int64_t C) { return C >= 4 && C <= 16384; }

// One launch for all the gradients of up to 16384 values, us in a graph, against partial
// sums and a launch that adds them: 1x64 2.5 and 3.6, 16x768 3.0 and 7.1, 64x128 3.0 and 5.8,
// 128x128 3.0 and 5.9, 1024x16 4.7 and 5.7, 4096x4 5.4 and 7.5, 2000x5 5.1 and 7.7; a launch
// less is 2 us less of the host's time as well.  It would gain up to 1024 rows of 2^19
// values (64x4096 4.6 and 9.4, 512x1024 5.0 and 7.2; 2048x64 7.3 and 6.6, 8192x8 12.1 and
// 8.0), but a row's dx has the same bits among any number of rows above this limit.
bool few(int64_t R, int64_t C) { return cached(C) && R * C <= 16384; }

// the workgroups of the backward of more, each of which leaves a partial sum: one on every
// CU at most (8192x4096 67 us, two 75; of short rows two: 65536x128 25, one 32)
int64_t parts_of(int64_t R, int64_t C) {
    if(few(R, C)) return 1;
    const int64_t rows = !cached(C) ? 1 : C <= 768 ? 8 : C <= 2048 ? 4 : C <= 4096 ? 2 : 1;
    const int64_t p = (R + rows - 1) / rows;
    const int64_t most = C <= 256 ? 512 : 256;
    return p < most ? p : most;
}

}  // namespace

extern "C" int pk_layernorm_fwd_f32(int64_t R, int64_t C, float eps, const float* x, const float* g,
                                    const float* b, float* y, float* mean, float* rstd,
                                    pk_stream_t stream) {
    if(R < 0 || C < 1) return pk::fail("pk_layernorm_fwd_f32: need R >= 0 and C >= 1");
    if(R > (int64_t)INT32_MAX || C > (int64_t)1 << 26)
        return pk::fail("pk_layernorm_fwd_f32: R above 2^31 - 1 or C above 2^26");
    if(R == 0) return PK_OK;
    if(!x || !g || !y) return pk::fail("pk_layernorm_fwd_f32: NULL pointer");
    hipStream_t st = pk::as_stream(stream);
    if(!cached(C)) {
        if(!pk::grid_fits(R, C < 4 ? 64 : 1024))
            return pk::fail("pk_layernorm_fwd_f32: too many rows of %lld values for one launch", (long long)C);
        if(C < 4) layernorm_fwd_any<1><<<(unsigned)R, 64, 0, st>>>(C, eps, x, g, b, y, mean, rstd);
        else layernorm_fwd_any<16><<<(unsigned)R, 1024, 0, st>>>(C, eps, x, g, b, y, mean, rstd);
        return pk::launch_status("pk_layernorm_fwd_f32");
    }
    with_shape<false>(C, [&](auto nv, auto w, auto exact) {
        constexpr int N = decltype(nv)::value, W = decltype(w)::value;
        constexpr bool EXACT = decltype(exact)::value;
        constexpr int rows = W > 4 ? 1 : 4 / W, threads = W > 4 ? 64 * W : 256;
        const int64_t blocks = (R + rows - 1) / rows;
        // workgroups walk the rows, the next one's loads under the present one's sums: four
        // on a CU (8192x1024 9.1 us, eight 10.6), eight of short rows (65536x128 18.5,
        // four 26.0)
        const int64_t most = C >= 512 ? 1024 : 2048;
        const unsigned grid = (unsigned)(blocks < most ? blocks : most);
        layernorm_fwd<N, W, EXACT><<<grid, threads, 0, st>>>((int)R, (int)C, eps, x, g, b, y, mean, rstd);
    });
    return pk::launch_status("pk_layernorm_fwd_f32");
}

extern "C" size_t pk_layernorm_bwd_workspace(int64_t R, int64_t C) {
    if(R <= 0 || C <= 0) return 0;
    return (size_t)parts_of(R, C) * 2 * (size_t)C * sizeof(float);
}

extern "C" int pk_layernorm_bwd_f32(int64_t R, int64_t C, const float* x, const float* g,
                                    const float* mean, const float* rstd, const float* dy,
                                    const float* dx_in, float* dx, float* dg, float* db, int flags,
                                    void* workspace, size_t workspace_bytes, pk_stream_t stream) {
    if(R < 0 || C < 1) return pk::fail("pk_layernorm_bwd_f32: need R >= 0 and C >= 1");
    if(R > (int64_t)INT32_MAX || C > (int64_t)1 << 26)
        return pk::fail("pk_layernorm_bwd_f32: R above 2^31 - 1 or C above 2^26");
    const bool sums = dg || db;
    if(R > 0) {
        if(!x || !g || !mean || !rstd || !dy)
            return pk::fail("pk_layernorm_bwd_f32: NULL input pointer");
        if(sums && (!workspace || workspace_bytes < pk_layernorm_bwd_workspace(R, C)))
            return pk::fail("pk_layernorm_bwd_f32: workspace needs %zu bytes",
                            pk_layernorm_bwd_workspace(R, C));
    }
    hipStream_t st = pk::as_stream(stream);
    float* ws = static_cast<float*>(workspace);
    const int64_t P = R > 0 ? parts_of(R, C) : 0;
    if(R > 0 && !dx && !sums) return PK_OK;
    if(R > 0 && few(R, C)) {
        int cols = 64;
        while(cols > 16 && kFewThreads / cols < R) cols /= 2;
        while(cols / 2 >= C) cols /= 2;
        const int rows = C <= 512 ? kFewThreads / 64 : 1, row_blocks = dx ? (int)((R + rows - 1) / rows) : 0;
        const unsigned grid = (unsigned)(row_blocks + (sums ? (C + cols - 1) / cols : 0));
        auto launch = [&](auto kernel) {
            kernel<<<grid, kFewThreads, 0, st>>>((int)R, (int)C, row_blocks, cols, x, g, mean, rstd, dy, dx_in, dx,
                                                 dg, db, flags);
        };
        if(rows > 1) launch(layernorm_bwd_few<1>);
        else launch(layernorm_bwd_few<kFewThreads / 64>);
        return pk::launch_status("pk_layernorm_bwd_f32");
    }
    if(R > 0 && cached(C)) {
        const int what = (dx ? kDx : 0) | (sums ? kSums : 0);
        with_shape<true>(C, [&](auto nv, auto w, auto exact) {
            constexpr int N = decltype(nv)::value, W = decltype(w)::value;
            constexpr bool EXACT = decltype(exact)::value;
            const size_t lds = kBwdWaves / W / 2 * 2 * (size_t)C * sizeof(float);
            if(dx && dx_in)
                layernorm_bwd<N, W, EXACT, true><<<(unsigned)P, 64 * kBwdWaves, lds, st>>>(
                    (int)R, (int)C, x, g, mean, rstd, dy, dx_in, dx, ws, what);
            else
                layernorm_bwd<N, W, EXACT, false><<<(unsigned)P, 64 * kBwdWaves, lds, st>>>(
                    (int)R, (int)C, x, g, mean, rstd, dy, nullptr, dx, ws, what);
        });
        if(sums)
            layernorm_sum<<<(unsigned)((2 * C + 63) / 64), 64 * kSumWaves, 0, st>>>(P, C, ws, dg, db, flags);
        return pk::launch_status("pk_layernorm_bwd_f32");
    }
    if(R > 0 && dx) {
        if(!pk::grid_fits(R, C < 4 ? 64 : 1024))
            return pk::fail("pk_layernorm_bwd_f32: too many rows of %lld values for one launch", (long long)C);
        if(C < 4) layernorm_dx_any<1><<<(unsigned)R, 64, 0, st>>>(C, x, g, mean, rstd, dy, dx_in, dx);
        else layernorm_dx_any<16><<<(unsigned)R, 1024, 0, st>>>(C, x, g, mean, rstd, dy, dx_in, dx);
    }
    if(sums) {
        if(R > 0)
            layernorm_parts_any<<<dim3((unsigned)((C + 255) / 256), (unsigned)P), 256, 0, st>>>(
                R, C, x, mean, rstd, dy, ws);
        layernorm_sum<<<(unsigned)((2 * C + 63) / 64), 64 * kSumWaves, 0, st>>>(P, C, ws, dg, db, flags);
    }
    return pk::launch_status("pk_layernorm_bwd_f32");
}
