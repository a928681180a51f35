// pico_amd/csrc/gemm_experts.hip -- matrix products grouped by expert: the launches
// of the fp32 (gemm_split.h), bf16 and split-bf16 (gemm_narrow.hip) tiles over
// groups of rows whose sizes only the device knows.
#include "gemm_common.h"

namespace {

using namespace pkg;

constexpr int kMaxExperts = 1024;

int check(const char* who, int64_t n, int64_t M, int64_t N, int64_t E, const int32_t* offsets,
          int precision) {
    if(n < 0 || n > (int64_t)1 << 30 || M < 0 || N < 0 || E < 1 || E > kMaxExperts)
        return pk::fail("%s: need 0 <= n <= 2^30 rows, sizes >= 0 and 1 <= E <= %d experts", who, kMaxExperts);
    if(!offsets) return pk::fail("%s: NULL offsets", who);
    if(precision < 0 || precision > 2)
        return pk::fail("%s: precision %d is not 0 (fp32), 1 (bf16) or 2 (three bf16 products)", who, precision);
    return PK_OK;
}

int run(bool ta, bool tb, const ExpertParams& ep, int64_t grid, TileKind kind, int precision,
        hipStream_t st) {
    const dim3 g((unsigned)grid, (unsigned)ep.splits);
    if(precision == 0) return launch_split_experts(ta, tb, ep, g, kind, st);
    return launch_narrow_experts(ta, tb, precision, ep, g, kind, st);
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
    ep.rows = 1;
    const int64_t groups = E < n ? E : n;
    const ExpertShape s = expert_rows_shape(precision, (double)groups, (double)n / groups, N, (double)K);
    // every expert with rows, and the rows behind the last one's, end in a partial tile
    const int64_t tiles_m = (n + s.bm - 1) / s.bm + groups + 1, tiles_n = (N + s.bn - 1) / s.bn;
    if(tiles_m * tiles_n > (int64_t)1 << 30)
        return pk::fail("pk_gemm_experts_f32: problem too large for one launch");
    ep.tiles_m = (int)tiles_m;
    ep.tiles_n = (int)tiles_n;
    return run(false, TB, ep, (tiles_m * tiles_n + 7) / 8 * 8, s.kind, precision, pk::as_stream(stream));
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
    if(tiles_m > (int64_t)1 << 30 || tiles_n > (int64_t)1 << 30 || tiles_m * tiles_n * E > (int64_t)1 << 30)
        return pk::fail("pk_gemm_experts_dw_f32: problem too large for one launch");
    ep.tiles_m = (int)tiles_m;
    ep.tiles_n = (int)tiles_n;
    // (an expert's tiles in 8 runs, one to an XCD)
    hipStream_t st = pk::as_stream(stream);
    if(int rc = run(true, false, ep, (tiles_m * tiles_n + 7) / 8 * 8 * E, s.kind, precision, st)) return rc;
    if(splits == 1) return PK_OK;
    experts_dw_sum<<<pk::grid_for(E * K * N, 256), 256, 0, st>>>(E, K, N, splits, ep.ws, dW, ldw, sw,
                                                                flags & PK_ACCUM);
    return pk::launch_status("pk_gemm_experts_dw_f32");
}
