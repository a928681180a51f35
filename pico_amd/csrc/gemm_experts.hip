// pico_amd/csrc/gemm_experts.hip -- matrix products grouped by expert: the launches
// of the fp32 (gemm_split.h), bf16 and split-bf16 (gemm_narrow.hip) tiles over
// groups of rows whose sizes only the device knows.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gemm_common.h"

namespace {

using namespace pkg;

constexpr int kMaxExperts = 1024;
// workgroups of a launch, at up to 1024 threads (fewer than 2^32 in all)
constexpr int64_t kMaxTiles = (int64_t)1 << 21;

int check(const char* who, int64_t n, int64_t M, int64_t N, int64_t E, const int32_t* offsets,
          int precision) {
    if(n < 0 || n > (int64_t)1 << 30 || M < 0 || N < 0 || E < 1 || E > kMaxExperts)
        return pk::fail("%s: need 0 <= n <= 2^30 rows, sizes >= 0 and 1 <= E <= %d experts", who, kMaxExperts);
    if(!offsets) return pk::fail("%s: NULL offsets", who);
    if(precision < 0 || precision > 2)
        return pk::fail("%s: precision %d is not 0 (fp32), 1 (bf16) or 2 (three bf16 products)", who, precision);
    return PK_OK;
}

int run(bool ta, bool tb, const ExpertParams& ep, int64_t grid, TileKind kind, bool full,
        int precision, hipStream_t st) {
    const dim3 g((unsigned)grid, (unsigned)ep.splits);
    if(precision == 0) return launch_split_experts(ta, tb, ep, g, kind, full, st);
    return launch_narrow_experts(ta, tb, precision, ep, g, kind, full, st);
}

// ------------------------------------------------ a few rows to an expert
// Y = X.W_e where every expert's weights are read for a handful of rows (tokens being
// generated): bound by W's bytes.  A workgroup takes 4 rows of an expert and 64 or
// 32 columns; its lanes lie 16 or 8 along the columns, the others along k, 4 k at a
// time, so W is read in runs of 256 or 128 bytes with two steps in flight, and each value is
// used 4 times in fp32 multiply-adds, which take less time than its bytes.  (bf16: operands
// rounded first, products exact.)  The partial sums meet across the lanes, then the
// waves, in a fixed order.
constexpr int kThinWaves = 8, kThinRows = 4;

template <int CL>
struct ThinTile {
    static constexpr int BM = kThinRows, BN = 4 * CL;
};

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

template <bool BF16>
__device__ __forceinline__ f32x4 rounded(f32x4 x) {
    if constexpr(BF16) {
        const bf16x4 b = __builtin_convertvector(x, bf16x4);
        return __builtin_convertvector(b, f32x4);
    }
    return x;
}

template <bool BF16>
__device__ __forceinline__ float rounded(float x) {
    return BF16 ? (float)(__bf16)x : x;
}

template <bool BF16, int CL>
__global__ __launch_bounds__(64 * kThinWaves) void experts_thin(ExpertParams p) {
    using T = ThinTile<CL>;
    constexpr int RM = kThinRows, KL = 64 / CL, STEP = 4 * KL * kThinWaves;  // k of a workgroup's step
    __shared__ alignas(16) float part[kThinWaves][RM][4 * CL];
    const TileJob j = tile_job<T>(p);
    if(j.skip) return;
    const int w = threadIdx.x / 64, lane = threadIdx.x % 64, cl = lane % CL;
    const int rows = (int)min(p.M - j.row0, (int64_t)RM);
    const int64_t col = j.col0 + 4 * cl, at = min(col, p.N - 4);
    const float* const wp = j.B + at;
    const int kl = lane / CL * 4;
    // a wave's x, [RM][4 KL], goes through LDS of its own: read by every lane it would
    // take as many cycles of the loads' path as W (4 experts [512, 512] 5.5 us, so 5.1; 2
    // [4096, 768] 13.2, 12.3; 64 [768, 768] of 8 rows 36, 32.5)
    constexpr int XV = KL / 4;
    __shared__ alignas(16) float xs[kThinWaves][RM][4 * KL];
    const int xr = lane / 16, xk = lane % 16 * XV;
    const float* const xp = j.A + (j.row0 + min(xr, rows - 1)) * p.lda + xk;
    f32x4 acc[RM];
#pragma unroll
    for(int r = 0; r < RM; ++r) acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    struct Step {
        f32x4 w[4];
        float x[XV];
    };
    auto load = [&](Step& s, int64_t k) {
#pragma unroll
        for(int v = 0; v < XV; ++v) s.x[v] = xp[k + v];
#pragma unroll
        for(int i = 0; i < 4; ++i) s.w[i] = *reinterpret_cast<const f32x4u*>(wp + (k + kl + i) * p.ldb);
        __builtin_amdgcn_sched_barrier(0);  // (not to be put off until they are needed)
    };
    auto add = [&](const Step& s) {
        f32x4 x[RM];
#pragma unroll
        for(int v = 0; v < XV; ++v) xs[w][xr][xk + v] = rounded<BF16>(s.x[v]);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for(int r = 0; r < RM; ++r) x[r] = *reinterpret_cast<const f32x4*>(&xs[w][r][kl]);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for(int i = 0; i < 4; ++i) {
            const f32x4 b = rounded<BF16>(s.w[i]);
#pragma unroll
            for(int r = 0; r < RM; ++r)
#pragma unroll
                for(int c = 0; c < 4; ++c) acc[r][c] = fmaf(x[r][i], b[c], acc[r][c]);
        }
    };
    // the steps that K fills, two in flight, without a branch around a load: the waits
    // would be for all of them
    int64_t k = 4 * w * KL;
    const int full = (int)(p.K / STEP);
    Step a, b;
    int left = full;
    if(left >= 2) {
        load(a, k);
        load(b, k + STEP);
        for(; left >= 4; left -= 2, k += 2 * STEP) {
            add(a);
            load(a, k + 2 * STEP);
            add(b);
            load(b, k + 3 * STEP);
        }
        add(a);
        if(left == 3) load(a, k + 2 * STEP);
        add(b);
        if(left == 3) add(a);
    } else if(left == 1) {
        load(a, k);
        add(a);
    }
    k = (int64_t)full * STEP + 4 * w * KL;
    if(k < p.K) {
        // a wave's last 4 KL k or fewer
#pragma unroll
        for(int v = 0; v < XV; ++v) a.x[v] = k + xk + v < p.K ? xp[k + v] : 0.0f;
#pragma unroll
        for(int i = 0; i < 4; ++i)
            a.w[i] = k + kl + i < p.K ? *reinterpret_cast<const f32x4u*>(wp + (k + kl + i) * p.ldb)
                                     : f32x4{0.f, 0.f, 0.f, 0.f};
        add(a);
    }
#pragma unroll
    for(int o = CL; o < 64; o <<= 1)
#pragma unroll
        for(int r = 0; r < RM; ++r)
#pragma unroll
            for(int c = 0; c < 4; ++c) acc[r][c] += __shfl_xor(acc[r][c], o, 64);
    if(lane < CL) {
#pragma unroll
        for(int r = 0; r < RM; ++r) *reinterpret_cast<f32x4*>(&part[w][r][4 * cl]) = acc[r];
    }
    __syncthreads();
    for(int i = threadIdx.x; i < rows * 4 * CL; i += 64 * kThinWaves) {
        const int r = i / (4 * CL), c = i % (4 * CL);
        float sum = part[0][r][c];
#pragma unroll
        for(int q = 1; q < kThinWaves; ++q) sum += part[q][r][c];
        // (a lane past N - 4 holds the row's last four)
        const int64_t n = j.col0 + c / 4 * 4, shift = max(n - (p.N - 4), (int64_t)0);
        if(c % 4 < shift) continue;
        float* const y = j.C + (j.row0 + r) * p.ldc + n - shift + c % 4;
        *y = j.beta != 0.0f ? *y + sum : sum;
    }
}

// Y = X.W_e^T of few rows, their input gradient: the sums run along W's rows.  A wave
// takes 4 rows and 8 outputs, its lanes lie along k, 4 k each, so that every load is a
// run of 1 KB; the lanes' sums meet at the end, each exchange halving the values a lane
// has.
constexpr int kThinOut = 8;

template <bool BF16>
__global__ __launch_bounds__(64 * kThinWaves) void experts_thin_t(ExpertParams p) {
    constexpr int RM = kThinRows, C = kThinOut, STEP = 256;
    using T = ThinTile<kThinWaves * C / 4>;
    const TileJob j = tile_job<T>(p);
    if(j.skip) return;
    const int w = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int rows = (int)min(p.M - j.row0, (int64_t)RM);
    const int64_t out = j.col0 + w * C;
    if(out >= p.N) return;
    const float *xp[RM], *wp[C];
#pragma unroll
    for(int r = 0; r < RM; ++r) xp[r] = j.A + (j.row0 + min(r, rows - 1)) * p.lda + 4 * lane;
#pragma unroll
    for(int c = 0; c < C; ++c) wp[c] = j.B + min(out + c, p.N - 1) * p.ldb + 4 * lane;
    float acc[RM * C];
#pragma unroll
    for(int i = 0; i < RM * C; ++i) acc[i] = 0.0f;
    struct Step {
        f32x4 x[RM], w[C];
    };
    auto load = [&](Step& s, int64_t k) {
#pragma unroll
        for(int r = 0; r < RM; ++r) s.x[r] = *reinterpret_cast<const f32x4u*>(xp[r] + k);
#pragma unroll
        for(int c = 0; c < C; ++c) s.w[c] = *reinterpret_cast<const f32x4u*>(wp[c] + k);
        __builtin_amdgcn_sched_barrier(0);  // (not to be put off until they are needed)
    };
    auto add = [&](const Step& s) {
        f32x4 x[RM];
#pragma unroll
        for(int r = 0; r < RM; ++r) x[r] = rounded<BF16>(s.x[r]);
#pragma unroll
        for(int c = 0; c < C; ++c) {
            const f32x4 b = rounded<BF16>(s.w[c]);
#pragma unroll
            for(int r = 0; r < RM; ++r)
#pragma unroll
                for(int i = 0; i < 4; ++i) acc[r * C + c] = fmaf(x[r][i], b[i], acc[r * C + c]);
        }
    };
    // whole steps, two in flight
    int left = (int)(p.K / STEP);
    int64_t k = 0;
    Step a, b;
    if(left > 0) {
        load(a, 0);
        for(; left > 2; left -= 2, k += 2 * STEP) {
            load(b, k + STEP);
            add(a);
            load(a, k + 2 * STEP);
            add(b);
        }
        if(left == 2) load(b, k + STEP);
        add(a);
        if(left == 2) add(b);
        k += left * STEP;
    }
    // the last 255 k or fewer: a lane's four, and the one lane's that has fewer
    const int64_t rest = p.K - k - 4 * lane;
    if(rest >= 4) {
        load(a, k);
        add(a);
    } else if(rest > 0) {
        for(int i = 0; i < (int)rest; ++i) {
            float x[RM];
#pragma unroll
            for(int r = 0; r < RM; ++r) x[r] = rounded<BF16>(xp[r][k + i]);
#pragma unroll
            for(int c = 0; c < C; ++c) {
                const float b = rounded<BF16>(wp[c][k + i]);
#pragma unroll
                for(int r = 0; r < RM; ++r) acc[r * C + c] = fmaf(x[r], b, acc[r * C + c]);
            }
        }
    }
    // lanes 2 i and 2 i + 1 end with value i
#pragma unroll
    for(int half = RM * C / 2; half > 0; half /= 2) {
        const int o = 2 * half;
        const bool up = lane & o;
#pragma unroll
        for(int i = 0; i < half; ++i) {
            const float give = up ? acc[i] : acc[i + half], keep = up ? acc[i + half] : acc[i];
            acc[i] = keep + __shfl_xor(give, o, 64);
        }
    }
    const float sum = acc[0] + __shfl_xor(acc[0], 1, 64);
    const int r = lane / 2 / C, c = lane / 2 % C;
    if(lane % 2 || r >= rows || out + c >= p.N) return;
    float* const y = j.C + (j.row0 + r) * p.ldc + out + c;
    *y = j.beta != 0.0f ? *y + sum : sum;
}

double thin_tiles(double groups, double m) { return groups * std::max(1.0, m / kThinRows + 0.5); }

// Microseconds: W once from memory, or once for every row tile from the caches, a start
// and one of every workgroup.  8 experts, rows each 1 / 4 / 8 / 16 / 24, us against those of matrix-core tiles:
// [768, 4096] 18 / 18 / 19 / 28 / 40 against 28 / 27 / 27 / 28 / 29 (in bf16 18 / 18 / 20 / 30 /
// 45 against 23 / 20 / 22 / 21 / 21), [2048, 768] 12 / 12 / 12 / 17 / 22 against 37 (96
// tiles, each all of K).  Small matrices have few tiles as well: 4 experts [512, 512] with
// 64 / 128 rows each 7 / 12 against 13.5, one of [419, 85] 5 against 13; 8 [333, 517] with
// 48 / 96 11 / 17 against 12, 17 [165, 641] with 48 20 against 11; in bf16 13 [152, 124] with 64 / 96 5.8 / 7.7 against 6.5.  Workgroups of 8 or 16 rows read W less often but are fewer
// and hold more: [768, 4096] with 4 rows each 24 and 31, when 4 took 22.
double thin_us(double groups, double m, int64_t N, int64_t K, int64_t tiles_n) {
    const double mb = (double)K * (double)N * 4e-6, tiles = thin_tiles(groups, m);
    return 3.0 + 0.003 * tiles * (double)tiles_n + mb * std::max(groups / 7.0, tiles / 20.0);
}

// Microseconds: W once from memory, or so many rounds of workgroups, one on a CU.  8
// experts, [N, K] with rows each 1 / 8 / 16 / 32 / 64, us against those of matrix-core
// tiles: [768, 4096] 20 / 22 / 34 / 50 / 96 against 66 (in bf16 22 / 23 / 40 / 61 / 119 against
// 51), [2048, 768] 12 / 15 / 25 / 44 / 85 against 18 / 18 / 18 / 19 / 24; 2 experts [93, 1464]
// up to 128 9 against 26.
double thin_t_us(double groups, double m, int64_t tiles_n, int64_t N, int64_t K, bool bf16) {
    const double wgs = thin_tiles(groups, m) * (double)tiles_n / 256.0;
    const double rounds = std::max(1.0, 0.5 * (wgs + std::ceil(wgs)));
    return std::max(4.0 + groups * (double)K * (double)N * 4e-6 / 6.5,
                    1.8 + rounds * (bf16 ? 3.0 + 0.0045 * (double)K : 2.2 + 0.0035 * (double)K));
}

// dW_e (+)= the sum of the S planes [S][E][K][N], in plane order
__global__ __launch_bounds__(256) void experts_dw_sum(int64_t E, int64_t K, int64_t N, int S,
                                                      const float* __restrict__ ws, float* dW,
                                                      int64_t ldw, int64_t sw, int accum) {
    const int64_t plane = E * K * N;
    for(int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < plane; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / N, e = r / K;
        float* const o = dW + e * sw + (r - e * K) * ldw + (i - r * N);
        float sum = 0.0f;
#pragma unroll 8
        for(int s = 0; s < S; ++s) sum += ws[s * plane + i];
        *o = accum ? *o + sum : sum;
    }
}

}  // namespace

extern "C" int pk_gemm_experts_f32(char tb, int64_t n, int64_t N, int64_t K, int64_t E,
                                   const int32_t* offsets, const float* X, int64_t ldx,
                                   const float* W, int64_t ldw, int64_t sw, float* Y, int64_t ldy,
                                   int flags, int precision, pk_stream_t stream) {
    const bool TB = tb == 'T' || tb == 't';
    if(!TB && tb != 'N' && tb != 'n')
        return pk::fail("pk_gemm_experts_f32: the transpose flag must be 'N' or 'T' (got '%c')", tb);
    if(int st = check("pk_gemm_experts_f32", n, N, K, E, offsets, precision)) return st;
    if(n == 0 || N == 0) return PK_OK;
    if(!Y || (K > 0 && (!X || !W))) return pk::fail("pk_gemm_experts_f32: NULL matrix");
    if(ldx < K || ldw < (TB ? K : N) || ldy < N || sw < 0)
        return pk::fail("pk_gemm_experts_f32: row stride too small, or a negative expert stride");
    // a tile's loads reach 32-bit byte offsets: 256 rows, or 32 rows of k
    const int64_t near_k = (int64_t)1 << 21, near_r = (int64_t)1 << 24;
    if(ldx > near_k || ldw > (TB ? near_k : near_r))
        return pk::fail("pk_gemm_experts_f32: row strides above 2^21 (W [K, N]: 2^24) are not built");
    ExpertParams ep = {};
    ep.A = X;
    ep.B = W;
    ep.C = Y;
    ep.M = n;
    ep.N = N;
    ep.K = K;
    ep.lda = ldx;
    ep.ldb = ldw;
    ep.ldc = ldy;
    ep.sBo = sw;
    ep.inner = 1;
    ep.alpha = 1.0f;
    ep.beta = (flags & PK_ACCUM) ? 1.0f : 0.0f;
    ep.splits = 1;
    ep.kchunk = K;
    ep.offsets = offsets;
    ep.experts = (int)E;
    ep.rows = kRows;
    const int64_t groups = E < n ? E : n;
    ExpertShape rest;
    const ExpertShape s = expert_rows_shape(precision, (double)groups, (double)n / groups, N, (double)K, &rest);
    // (the estimates are of up to 128 rows to an expert, 64 in bf16.  32 columns to a workgroup
    // where 64 would leave much of the chip idle, by the estimated tiles of 64; [K, N], rows
    // of each expert, us with 32 and 64, weights from memory, as in a model of several layers:
    // 96 tiles, 8 [2048, 768] of 1 14.2 and 17.3, 2 [4096, 2048] of 4 22.1 and 29.1; 128, 8
    // [768, 1024] of 1 8.7 and 8.9; 144, 8 [2048, 768] of 4 14.3 and 17.9, of 0 to 9 15.4 and
    // 17.3, 16 [1024, 384] of 4 8.6 and 10.1, 12 [2048, 768] of 1 19.7 and 19.5; 150, 3 [2048,
    // 1280] of 8 13.5 and 16.3; 154, 8 [2048, 704] of 5 16.3 and 15.0; 156, 13 [2048, 768] of 1
    // 22.6 and 20.2; 192, 8 [2048, 768] of 6 18.2 and 17.0.  Weights that are still in the
    // last-level cache differ less: 144 tiles, 8 [2048, 768] of 4 11.8 and 12.5, of 0 to 9
    // 11.9 and 11.5, 8 [768, 768] of 0 to 9 6.6 and 5.8)
    const int cl = thin_tiles((double)groups, (double)n / groups) * (double)((N + 63) / 64) <= 150.0 ? 8 : 16;
    const int64_t tiles_m = (n + kThinRows - 1) / kThinRows + groups + 1, tiles_n = (N + 4 * cl - 1) / (4 * cl);
    const int64_t tiles_t = (N + 63) / 64;
    if(TB && K > 0 && n <= 256 * groups && tiles_t <= kMaxTiles / tiles_m &&
       thin_t_us((double)groups, (double)n / groups, tiles_t, N, K, precision == 1) < s.us) {
        ep.tiles_m = (int)tiles_m;
        ep.tiles_n = (int)tiles_t;
        const unsigned grid = (unsigned)((tiles_m * ep.tiles_n + 7) / 8 * 8);
        hipStream_t st = pk::as_stream(stream);
        if(precision == 1) experts_thin_t<true><<<grid, 64 * kThinWaves, 0, st>>>(ep);
        else experts_thin_t<false><<<grid, 64 * kThinWaves, 0, st>>>(ep);
        return pk::launch_status("pk_gemm_experts_f32");
    }
    if(!TB && N >= 4 && K > 0 && n <= (precision == 0 ? 128 : 64) * groups && tiles_n <= kMaxTiles / tiles_m &&
       thin_us((double)groups, (double)n / groups, N, K, tiles_n) < s.us) {
        ep.tiles_m = (int)tiles_m;
        ep.tiles_n = (int)tiles_n;
        const unsigned grid = (unsigned)((tiles_m * tiles_n + 7) / 8 * 8);
        hipStream_t st = pk::as_stream(stream);
        auto launch = [&](auto cl) {
            constexpr int CL = decltype(cl)::value;
            if(precision == 1) experts_thin<true, CL><<<grid, 64 * kThinWaves, 0, st>>>(ep);
            else experts_thin<false, CL><<<grid, 64 * kThinWaves, 0, st>>>(ep);
        };
        if(cl == 16) launch(std::integral_constant<int, 16>());
        else launch(std::integral_constant<int, 8>());
        return pk::launch_status("pk_gemm_experts_f32");
    }
    // `most` row tiles at most
    auto tiles = [&](const ExpertShape& t, int64_t most, int which, bool full) {
        const int64_t tiles_n = (N + t.bn - 1) / t.bn;
        if(most > 0 && tiles_n > kMaxTiles / most)
            return pk::fail("pk_gemm_experts_f32: problem too large for one launch");
        ep.rows = which;
        ep.tiles_m = (int)most;
        ep.tiles_n = (int)tiles_n;
        return run(false, TB, ep, (most * tiles_n + 7) / 8 * 8, t.kind, full, precision, pk::as_stream(stream));
    };
    // every expert with rows, and the rows behind the last one's, end in a partial tile
    if(!rest.bm) return tiles(s, (n + s.bm - 1) / s.bm + groups + 1, kRows, false);
    if(int st = tiles(s, n / s.bm, kRowsWhole, N % s.bn == 0 && K % 32 == 0)) return st;
    // up to 255 rows of every expert
    return tiles(rest, groups * ((254 + rest.bm) / rest.bm) + kZeroTiles, kRowsRest, false);
}

extern "C" size_t pk_gemm_experts_dw_workspace(int64_t n, int64_t K, int64_t N, int64_t E) {
    if(n <= 0 || K <= 0 || N <= 0 || E < 1 || E > kMaxExperts) return 0;
    int most = 1;
    for(int precision = 0; precision < 3; ++precision) {
        int splits;
        expert_dw_shape(precision, E, K, N, n, true, &splits);
        if(splits > most) most = splits;
    }
    return most > 1 ? (size_t)most * (size_t)E * (size_t)K * (size_t)N * sizeof(float) : 0;
}

extern "C" int pk_gemm_experts_dw_f32(int64_t n, int64_t K, int64_t N, int64_t E,
                                      const int32_t* offsets, const float* X, int64_t ldx,
                                      const float* dY, int64_t ldy, float* dW, int64_t ldw, int64_t sw,
                                      int flags, int precision, void* workspace,
                                      size_t workspace_bytes, pk_stream_t stream) {
    if(int st = check("pk_gemm_experts_dw_f32", n, K, N, E, offsets, precision)) return st;
    if(K == 0 || N == 0) return PK_OK;
    if(!dW || (n > 0 && (!X || !dY))) return pk::fail("pk_gemm_experts_dw_f32: NULL matrix");
    if(ldx < K || ldy < N || ldw < N || (E > 1 && sw < (K - 1) * ldw + N))
        return pk::fail("pk_gemm_experts_dw_f32: row stride too small, or experts' gradients overlap");
    const int64_t near_r = (int64_t)1 << 24;
    if(ldx > near_r || ldy > near_r)
        return pk::fail("pk_gemm_experts_dw_f32: row strides above 2^24 are not built");
    ExpertParams ep = {};
    ep.A = X;
    ep.B = dY;
    ep.C = dW;
    ep.M = K;
    ep.N = N;
    ep.K = n;
    ep.lda = ldx;
    ep.ldb = ldy;
    ep.ldc = ldw;
    ep.sCo = sw;
    ep.inner = 1;
    ep.alpha = 1.0f;
    ep.beta = (flags & PK_ACCUM) ? 1.0f : 0.0f;
    ep.splits = 1;
    ep.kchunk = n;
    ep.offsets = offsets;
    ep.experts = (int)E;
    int splits;
    ExpertShape s = expert_dw_shape(precision, E, K, N, n, workspace != nullptr, &splits);
    if(workspace_bytes < (size_t)splits * (size_t)E * (size_t)K * (size_t)N * sizeof(float))
        s = expert_dw_shape(precision, E, K, N, n, false, &splits);
    ep.splits = splits;
    ep.ws = static_cast<float*>(workspace);
    const int64_t tiles_m = (K + s.bm - 1) / s.bm, tiles_n = (N + s.bn - 1) / s.bn;
    if(tiles_m > kMaxTiles || tiles_n > kMaxTiles || tiles_m * tiles_n > kMaxTiles / E)
        return pk::fail("pk_gemm_experts_dw_f32: problem too large for one launch");
    ep.tiles_m = (int)tiles_m;
    ep.tiles_n = (int)tiles_n;
    // (an expert's tiles in 8 runs, one to an XCD)
    hipStream_t st = pk::as_stream(stream);
    if(int rc = run(true, false, ep, (tiles_m * tiles_n + 7) / 8 * 8 * E, s.kind, false, precision, st)) return rc;
    if(splits == 1) return PK_OK;
    experts_dw_sum<<<pk::grid_for(E * K * N, 256), 256, 0, st>>>(E, K, N, splits, ep.ws, dW, ldw, sw,
                                                                flags & PK_ACCUM);
    return pk::launch_status("pk_gemm_experts_dw_f32");
}
