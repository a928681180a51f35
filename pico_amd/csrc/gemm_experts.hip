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
    if(precision == 0) return launch_split_experts(ta, tb, ep, (unsigned)grid, kind, st);
    return launch_narrow_experts(ta, tb, precision, ep, (unsigned)grid, kind, st);
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
    const ExpertShape s = expert_shape(precision, false, (double)groups, (double)n / groups, N, (double)K);
    // every expert with rows, and the rows behind the last one's, end in a partial tile
    const int64_t tiles_m = (n + s.bm - 1) / s.bm + groups + 1, tiles_n = (N + s.bn - 1) / s.bn;
    if(tiles_m * tiles_n > (int64_t)1 << 30)
        return pk::fail("pk_gemm_experts_f32: problem too large for one launch");
    ep.tiles_m = (int)tiles_m;
    ep.tiles_n = (int)tiles_n;
    return run(false, TB, ep, (tiles_m * tiles_n + 7) / 8 * 8, s.kind, precision, pk::as_stream(stream));
}

extern "C" size_t pk_gemm_experts_dw_workspace(int64_t n, int64_t K, int64_t N, int64_t E) {
    (void)n;
    (void)K;
    (void)N;
    (void)E;
    return 0;
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
    const ExpertShape s = expert_shape(precision, true, (double)E, (double)K, N, (double)n / E);
    const int64_t tiles_m = (K + s.bm - 1) / s.bm, tiles_n = (N + s.bn - 1) / s.bn;
    if(tiles_m > (int64_t)1 << 30 || tiles_n > (int64_t)1 << 30 || tiles_m * tiles_n * E > (int64_t)1 << 30)
        return pk::fail("pk_gemm_experts_dw_f32: problem too large for one launch");
    ep.tiles_m = (int)tiles_m;
    ep.tiles_n = (int)tiles_n;
    return run(true, false, ep, (tiles_m * tiles_n * E + 7) / 8 * 8, s.kind, precision, pk::as_stream(stream));
}
