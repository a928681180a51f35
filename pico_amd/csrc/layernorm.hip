// pico_amd/csrc/layernorm.hip -- layer norm over rows of [R, C] and its gradients.
//
//   y = (x - m) r g + b,  m = mean(x),  r = (mean((x - m)^2) + eps)^-1/2
//   xh = (x - m) r
//   dx = r (g dy - mean(g dy) - xh mean(g dy xh))
//   dg = sum over rows of dy xh,  db = sum over rows of dy
#include "pk_common.h"

namespace {

__global__ __launch_bounds__(256) void layernorm_fwd_any(int64_t R, int64_t C, float eps,
                                                         const float* __restrict__ x,
                                                         const float* __restrict__ g,
                                                         const float* __restrict__ b,
                                                         float* __restrict__ y,
                                                         float* __restrict__ mean,
                                                         float* __restrict__ rstd) {
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    const int lane = threadIdx.x % 64;
    if(row >= R) return;
    const float* xr = x + row * C;
    float s = 0.0f;
    for(int64_t c = lane; c < C; c += 64) s += xr[c];
    const float m = pk::wave_sum(s) / (float)C;
    s = 0.0f;
    for(int64_t c = lane; c < C; c += 64) s += (xr[c] - m) * (xr[c] - m);
    const float r = 1.0f / sqrtf(pk::wave_sum(s) / (float)C + eps);
    if(lane == 0) {
        if(mean) mean[row] = m;
        if(rstd) rstd[row] = r;
    }
    for(int64_t c = lane; c < C; c += 64)
        y[row * C + c] = (xr[c] - m) * r * g[c] + (b ? b[c] : 0.0f);
}

__global__ __launch_bounds__(256) void layernorm_dx_any(int64_t R, int64_t C,
                                                        const float* __restrict__ x,
                                                        const float* __restrict__ g,
                                                        const float* __restrict__ mean,
                                                        const float* __restrict__ rstd,
                                                        const float* __restrict__ dy,
                                                        const float* dxin, float* dx) {
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    const int lane = threadIdx.x % 64;
    if(row >= R) return;
    const float* xr = x + row * C;
    const float* dr = dy + row * C;
    const float m = mean[row], r = rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for(int64_t c = lane; c < C; c += 64) {
        const float t = g[c] * dr[c];
        s1 += t;
        s2 += t * ((xr[c] - m) * r);
    }
    s1 = pk::wave_sum(s1) / (float)C;
    s2 = pk::wave_sum(s2) / (float)C;
    for(int64_t c = lane; c < C; c += 64) {
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

int64_t parts_of(int64_t R) { return R < 256 ? R : 256; }

}  // namespace

extern "C" int pk_layernorm_fwd_f32(int64_t R, int64_t C, float eps, const float* x, const float* g,
                                    const float* b, float* y, float* mean, float* rstd,
                                    pk_stream_t stream) {
    if(R < 0 || C < 1) return pk::fail("pk_layernorm_fwd_f32: need R >= 0 and C >= 1");
    if(R > (int64_t)INT32_MAX) return pk::fail("pk_layernorm_fwd_f32: R above 2^31 - 1");
    if(R == 0) return PK_OK;
    if(!x || !g || !y) return pk::fail("pk_layernorm_fwd_f32: NULL pointer");
    layernorm_fwd_any<<<(unsigned)((R + 3) / 4), 256, 0, pk::as_stream(stream)>>>(R, C, eps, x, g, b, y,
                                                                             mean, rstd);
    return pk::launch_status("pk_layernorm_fwd_f32");
}

extern "C" size_t pk_layernorm_bwd_workspace(int64_t R, int64_t C) {
    if(R <= 0 || C <= 0) return 0;
    return (size_t)parts_of(R) * 2 * (size_t)C * sizeof(float);
}

extern "C" int pk_layernorm_bwd_f32(int64_t R, int64_t C, const float* x, const float* g,
                                    const float* mean, const float* rstd, const float* dy,
                                    const float* dx_in, float* dx, float* dg, float* db, int flags,
                                    void* workspace, size_t workspace_bytes, pk_stream_t stream) {
    if(R < 0 || C < 1) return pk::fail("pk_layernorm_bwd_f32: need R >= 0 and C >= 1");
    if(R > (int64_t)INT32_MAX) return pk::fail("pk_layernorm_bwd_f32: R above 2^31 - 1");
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
    const int64_t P = R > 0 ? parts_of(R) : 0;
    if(R > 0 && dx)
        layernorm_dx_any<<<(unsigned)((R + 3) / 4), 256, 0, st>>>(R, C, x, g, mean, rstd, dy, dx_in, dx);
    if(sums) {
        if(R > 0)
            layernorm_parts_any<<<dim3((unsigned)((C + 255) / 256), (unsigned)P), 256, 0, st>>>(
                R, C, x, mean, rstd, dy, ws);
        layernorm_sum<<<(unsigned)((2 * C + 63) / 64), 64 * kSumWaves, 0, st>>>(P, C, ws, dg, db, flags);
    }
    return pk::launch_status("pk_layernorm_bwd_f32");
}
