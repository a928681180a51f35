// pico_amd/csrc/scan.hip -- a gated linear recurrence along the tokens of each
// sequence, channel by channel, and its gradients.
//
//   s_t = sigmoid(f_t),  h_t = s_t h_{t-1} + (1 - s_t) x_t,  h_0 given or zero
// and backwards, with the gradient u that a token hands to the one before it,
//   G_t = dh_t + u_{t+1},  u_t = s_t G_t
//   dx_t = (1 - s_t) G_t,  df_t = G_t (h_{t-1} - x_t) s_t (1 - s_t),  dh_0 = u_1
#include "pk_common.h"

namespace {

// s = sigmoid(f) and q = 1 - s = sigmoid(-f), each to its own last bits: the
// smaller one is not got by subtraction
__device__ __forceinline__ void gate(float f, float& s, float& q) {
    const float t = expf(-fabsf(f));  // (0, 1]; NaN stays NaN
    const float big = 1.0f / (1.0f + t), small = t * big;
    s = f >= 0.0f ? big : small;
    q = f >= 0.0f ? small : big;
}

__global__ __launch_bounds__(256) void scan_fwd_serial(int64_t B, int64_t T, int64_t C,
                                                       const float* __restrict__ f, int64_t ldf,
                                                       const float* __restrict__ x, int64_t ldx,
                                                       const float* __restrict__ h0,
                                                       float* __restrict__ h) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if(i >= B * C) return;
    const int64_t b = i / C, c = i % C;
    float p = h0 ? h0[i] : 0.0f;
    for(int64_t t = 0; t < T; ++t) {
        const int64_t row = b * T + t;
        float s, q;
        gate(f[row * ldf + c], s, q);
        p = s * p + q * x[row * ldx + c];
        h[row * C + c] = p;
    }
}

__global__ __launch_bounds__(256) void scan_bwd_serial(int64_t B, int64_t T, int64_t C,
                                                       const float* __restrict__ f, int64_t ldf,
                                                       const float* __restrict__ x, int64_t ldx,
                                                       const float* __restrict__ h0,
                                                       const float* __restrict__ h,
                                                       const float* __restrict__ dh, float* df,
                                                       int64_t lddf, float* dx, int64_t lddx,
                                                       float* dh0, int flags) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if(i >= B * C) return;
    const int64_t b = i / C, c = i % C;
    float u = 0.0f;
    for(int64_t t = T - 1; t >= 0; --t) {
        const int64_t row = b * T + t;
        float s, q;
        gate(f[row * ldf + c], s, q);
        const float G = dh[row * C + c] + u;
        const float before = t > 0 ? h[(row - 1) * C + c] : h0 ? h0[i] : 0.0f;
        if(df) {
            const float v = G * (before - x[row * ldx + c]) * (s * q);
            float* o = df + row * lddf + c;
            *o = (flags & PK_ACCUM) ? *o + v : v;
        }
        if(dx) {
            float* o = dx + row * lddx + c;
            *o = (flags & PK_ACCUM2) ? *o + q * G : q * G;
        }
        u = s * G;
    }
    if(dh0) dh0[i] = (flags & PK_ACCUM3) ? dh0[i] + u : u;
}

int check(const char* who, int64_t B, int64_t T, int64_t C, const float* f, int64_t ldf,
          const float* x, int64_t ldx) {
    if(B < 0 || T < 0 || C < 0) return pk::fail("%s: negative size", who);
    if(B > INT32_MAX || T > INT32_MAX || C > INT32_MAX || B * T > INT32_MAX ||
       B * C > (int64_t)INT32_MAX * 64)
        return pk::fail("%s: B*T rows or B*C channels too many for one call", who);
    if(B == 0 || T == 0 || C == 0) return PK_OK;
    if(!f || !x) return pk::fail("%s: NULL f or x", who);
    if(ldf < C || ldx < C) return pk::fail("%s: row stride < C", who);
    return PK_OK;
}

}  // namespace

extern "C" size_t pk_gated_scan_workspace(int64_t B, int64_t T, int64_t C) {
    (void)B;
    (void)T;
    (void)C;
    return 0;
}

extern "C" int pk_gated_scan_fwd_f32(int64_t B, int64_t T, int64_t C, const float* f, int64_t ldf,
                                     const float* x, int64_t ldx, const float* h0, float* h,
                                     void* workspace, size_t workspace_bytes, pk_stream_t stream) {
    if(int st = check("pk_gated_scan_fwd_f32", B, T, C, f, ldf, x, ldx)) return st;
    if(B == 0 || T == 0 || C == 0) return PK_OK;
    if(!h) return pk::fail("pk_gated_scan_fwd_f32: NULL h");
    scan_fwd_serial<<<(unsigned)((B * C + 255) / 256), 256, 0, pk::as_stream(stream)>>>(B, T, C, f, ldf, x,
                                                                                   ldx, h0, h);
    return pk::launch_status("pk_gated_scan_fwd_f32");
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
    scan_bwd_serial<<<(unsigned)((B * C + 255) / 256), 256, 0, pk::as_stream(stream)>>>(
        B, T, C, f, ldf, x, ldx, h0, h, dh, df, lddf, dx, lddx, dh0, flags);
    return pk::launch_status("pk_gated_scan_bwd_f32");
}
