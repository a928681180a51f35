// pico_amd/csrc/experts.hip -- a mixture of experts around its products: the top-k
// router and its gradient, the grouping of the (token, choice) slots by expert,
// and the movement of rows into and out of expert order.
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "pk_common.h"

namespace {

// ---------------------------------------------------------------- the router
// G lanes to a token, N logits a lane (expert = lane + i G).  A logit becomes an
// integer that orders like it: NaN above all, -0 as 0, and 0 for -inf, which is
// never chosen.
__device__ __forceinline__ unsigned order_key(float v) {
    if(v != v) return 0xffffffffu;
    const unsigned b = __float_as_uint(v == 0.0f ? 0.0f : v);
    if(b == 0xff800000u) return 0;
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(unsigned k) {
    if(k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

template <int G, int N>
__global__ __launch_bounds__(256) void route_topk_kernel(int64_t R, int E, int k,
                                                         const float* __restrict__ z, int64_t ldz,
                                                         int32_t* __restrict__ experts,
                                                         float* __restrict__ gates) {
    const int64_t row = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const int lane = threadIdx.x % G;
    const bool on = row < R;  // (lanes of a last row stay for the exchanges)
    unsigned key[N];
#pragma unroll
    for(int i = 0; i < N; ++i) {
        const int e = lane + i * G;
        key[i] = on && e < E ? order_key(z[row * ldz + e]) : 0;
    }
    int mine = -1;
    float value = 0.0f;
    for(int j = 0; j < k; ++j) {
        unsigned best = key[0];
        int at = lane;
#pragma unroll
        for(int i = 1; i < N; ++i)
            if(key[i] > best) {
                best = key[i];
                at = lane + i * G;
            }
#pragma unroll
        for(int o = G / 2; o > 0; o >>= 1) {
            const unsigned other = __shfl_xor(best, o, G);
            const int there = __shfl_xor(at, o, G);
            if(other > best || (other == best && there < at)) {
                best = other;
                at = there;
            }
        }
#pragma unroll
        for(int i = 0; i < N; ++i)
            if(at == lane + i * G) key[i] = 0;
        if(lane == j) {
            mine = best ? at : -1;
            value = key_value(best);
        }
    }
    const float top = __shfl(value, 0, G);
    float w = mine < 0 ? 0.0f : expf(value - top);
    float sum = w;
#pragma unroll
    for(int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, G);
    if(on && lane < k) {
        experts[row * k + lane] = mine;
        gates[row * k + lane] = mine < 0 ? 0.0f : w / sum;
    }
}

// dz = g (dg - sum of g dg) on the chosen experts, 0 on the others
template <int G, int N>
__global__ __launch_bounds__(256) void route_topk_bwd_kernel(int64_t R, int E, int k,
                                                             const int32_t* __restrict__ experts,
                                                             const float* __restrict__ gates,
                                                             const float* __restrict__ dgates,
                                                             float* dz, int64_t ldd, int accum) {
    const int64_t row = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const int lane = threadIdx.x % G;
    const bool on = row < R, slot = on && lane < k;
    const int mine = slot ? experts[row * k + lane] : -1;
    // (a slot without an expert has no gradient, whatever dgates holds there)
    const float g = mine >= 0 ? gates[row * k + lane] : 0.0f;
    const float d = mine >= 0 ? dgates[row * k + lane] : 0.0f;
    float sum = g * d;
#pragma unroll
    for(int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, G);
    const float v = g * (d - sum);
    float out[N];
#pragma unroll
    for(int i = 0; i < N; ++i) out[i] = 0.0f;
    for(int j = 0; j < k; ++j) {
        const int e = __shfl(mine, j, G);
        const float x = __shfl(v, j, G);
#pragma unroll
        for(int i = 0; i < N; ++i)
            if(e == lane + i * G) out[i] += x;
    }
    if(!on) return;
#pragma unroll
    for(int i = 0; i < N; ++i) {
        const int e = lane + i * G;
        if(e >= E) continue;
        float* p = dz + row * ldd + e;
        *p = accum ? *p + out[i] : out[i];
    }
}

constexpr int kMaxExperts = 1024, kMaxTopk = 64;
// slots, at up to 64 lanes each (a launch has fewer than 2^32 threads)
constexpr int64_t kMaxSlots = (int64_t)1 << 25;

// f(G, N) as compile-time numbers: 4 logits a lane where that leaves at least 8 lanes
// to a token and k of them, so that a wave has several tokens and an exchange few
// steps (8192 tokens of 64 experts, 2 choices: 16 lanes 3.8 us, 64 lanes 6.0)
template <class F>
void with_router_shape(int E, int k, F f) {
    using std::integral_constant;
    int lanes = 8;
    while(lanes < 64 && (lanes < k || 4 * lanes < E)) lanes *= 2;
    auto logits = [&](auto g) {
        constexpr int G = decltype(g)::value;
        if(E <= G) f(g, integral_constant<int, 1>());
        else if(E <= 2 * G) f(g, integral_constant<int, 2>());
        else if(G < 64 || E <= 4 * G) f(g, integral_constant<int, 4>());
        else if(E <= 8 * G) f(integral_constant<int, 64>(), integral_constant<int, 8>());
        else f(integral_constant<int, 64>(), integral_constant<int, 16>());
    };
    if(lanes == 8) logits(integral_constant<int, 8>());
    else if(lanes == 16) logits(integral_constant<int, 16>());
    else if(lanes == 32) logits(integral_constant<int, 32>());
    else logits(integral_constant<int, 64>());
}

int check_route(const char* who, int64_t R, int64_t E, int64_t k) {
    if(R < 0 || E < 1 || E > kMaxExperts || k < 1 || k > E || k > kMaxTopk)
        return pk::fail("%s: need R >= 0, 1 <= E <= %d experts and 1 <= k <= min(E, %d) choices", who,
                        kMaxExperts, kMaxTopk);
    if(R > kMaxSlots || R * k > kMaxSlots) return pk::fail("%s: R*k above 2^25", who);
    return PK_OK;
}

// ------------------------------------------------- slots in expert order
// A stable counting sort of the n slots by expert.  Every block takes a chunk of
// consecutive slots; with more than one block a first launch counts each
// chunk's experts and the second one starts from those counts.
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

__device__ __forceinline__ int slot_expert(const int32_t* experts, int64_t i, int E) {
    const int e = experts[i];
    return e < 0 || e >= E ? E : e;  // E: dropped
}

__global__ __launch_bounds__(kPlanThreads) void plan_count(int64_t n, int64_t chunk, int E,
                                                        const int32_t* __restrict__ experts,
                                                        int32_t* __restrict__ counts) {
    __shared__ int hist[kMaxExperts + 1];
    for(int e = threadIdx.x; e <= E; e += kPlanThreads) hist[e] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * chunk, hi = lo + chunk < n ? lo + chunk : n;
    for(int64_t i = lo + threadIdx.x; i < hi; i += kPlanThreads)
        atomicAdd(&hist[slot_expert(experts, i, E)], 1);  // (whole numbers: any order)
    __syncthreads();
    for(int e = threadIdx.x; e <= E; e += kPlanThreads)
        counts[(int64_t)blockIdx.x * (E + 1) + e] = hist[e];
}

__global__ __launch_bounds__(kPlanThreads) void plan_place(int64_t n, int64_t chunk, int E, int bits,
                                                        const int32_t* __restrict__ experts,
                                                        const int32_t* __restrict__ counts,
                                                        int32_t* __restrict__ offsets,
                                                        int32_t* __restrict__ order,
                                                        int32_t* __restrict__ place) {
    __shared__ int next[kMaxExperts + 1];  // where this block's next slot of an expert goes
    __shared__ int cnt[kPlanWaves][kMaxExperts + 1];
    __shared__ int wave_total[kPlanWaves];
    const int w = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int64_t lo = (int64_t)blockIdx.x * chunk, hi = lo + chunk < n ? lo + chunk : n;
    for(int e = threadIdx.x; e <= E; e += kPlanThreads) {
        next[e] = 0;
#pragma unroll
        for(int i = 0; i < kPlanWaves; ++i) cnt[i][e] = 0;
    }
    __syncthreads();
    // totals of every expert, and of the blocks before this one
    int before[2] = {0, 0}, total[2] = {0, 0};  // experts threadIdx.x and threadIdx.x + 1024
    if(gridDim.x == 1) {
        for(int64_t i = lo + threadIdx.x; i < hi; i += kPlanThreads)
            atomicAdd(&next[slot_expert(experts, i, E)], 1);
        __syncthreads();
#pragma unroll
        for(int q = 0; q < 2; ++q) {
            const int e = threadIdx.x + q * kPlanThreads;
            if(e <= E) total[q] = next[e];
        }
    } else {
#pragma unroll
        for(int q = 0; q < 2; ++q) {
            const int e = threadIdx.x + q * kPlanThreads;
            if(e > E) continue;
#pragma unroll 8
            for(int b = 0; b < (int)gridDim.x; ++b) {
                const int c = counts[(int64_t)b * (E + 1) + e];
                total[q] += c;
                if(b < (int)blockIdx.x) before[q] += c;
            }
        }
    }
    // exclusive sums over the experts (only expert 1024 can be a thread's second)
    int s = total[0];
#pragma unroll
    for(int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(s, o, 64);
        if(lane >= o) s += t;
    }
    if(lane == 63) wave_total[w] = s;
    __syncthreads();
    int base = 0, all = 0;
#pragma unroll
    for(int i = 0; i < kPlanWaves; ++i) {
        if(i < w) base += wave_total[i];
        all += wave_total[i];
    }
    const int first[2] = {base + s - total[0], all};
#pragma unroll
    for(int q = 0; q < 2; ++q) {
        const int e = threadIdx.x + q * kPlanThreads;
        if(e > E) continue;
        next[e] = first[q] + before[q];
        if(blockIdx.x == 0) offsets[e] = first[q];
    }
    __syncthreads();
    for(int64_t at = lo; at < hi; at += kPlanThreads) {
        const int64_t i = at + threadIdx.x;
        const bool on = i < hi;
        const int e = on ? slot_expert(experts, i, E) : E + 1;
        // the wave's lanes with the same expert
        uint64_t same = ~0ull;
        for(int b = 0; b < bits; ++b) {
            const bool bit = (e >> b) & 1;
            const uint64_t m = __ballot(bit);
            same &= bit ? m : ~m;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        if(on && rank == 0) cnt[w][e] = __popcll(same);
        __syncthreads();
        if(on) {
            int p = next[e] + rank;
            for(int v = 0; v < w; ++v) p += cnt[v][e];
            order[p] = (int32_t)i;
            place[i] = e == E ? -1 : p;
        }
        __syncthreads();
        for(int q = threadIdx.x; q <= E; q += kPlanThreads) {
            int sum = 0;
#pragma unroll
            for(int v = 0; v < kPlanWaves; ++v) {
                sum += cnt[v][q];
                cnt[v][q] = 0;
            }
            next[q] += sum;
        }
        __syncthreads();
    }
}

// Up to 2048 slots are placed by one block (64 experts, us: 2048 5.6, two blocks and
// the launch that counts 6.0; 4096 8.7 against 7.0, 16384 27.5 against 6.8), more
// dealt to blocks of 1024, from 65536 of 2048 and so many that 256 do (262144
// 13.1, of 1024 17.6).
int64_t plan_chunk(int64_t n) {
    if(n <= 2048) return n > 0 ? n : 1;
    if(n <= 65536) return 1024;
    const int64_t c = (n + 255) / 256;
    return c <= 2048 ? 2048 : (c + kPlanThreads - 1) / kPlanThreads * kPlanThreads;
}

// ------------------------------------------------------------ rows
// V floats to a lane (1 or 4), L lanes to a row: a wave, or for a few rows a
// workgroup.  Bound by the rows' bytes (8192 tokens of 768, 2 choices, us: gather 17.5,
// combine 20, its backward 24.5, 5.0 to 6.1 TB/s); a few rows by the loads that wait
// for each other (a row's place, its values), which are issued together where they
// can be.
template <int V>
struct Row;
template <>
struct Row<1> {
    typedef float T;
    static __device__ __forceinline__ float dot(float a, float b) { return a * b; }
};
template <>
struct Row<4> {
    typedef f32x4 T;
    static __device__ __forceinline__ float dot(f32x4 a, f32x4 b) {
        return a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3];
    }
};

// out[r] = x[order[r] / k] for r < offsets[E]; zeros from there on
template <int V, int L>
__global__ __launch_bounds__(256) void expert_gather_kernel(int n, int64_t d, int k,
                                                            const int32_t* __restrict__ kept,
                                                            const int32_t* __restrict__ order,
                                                            const float* __restrict__ x, int64_t ldx,
                                                            float* __restrict__ out, int64_t ldo) {
    typedef typename Row<V>::T T;
    const int r = (int)(blockIdx.x * (256 / L) + threadIdx.x / L);
    if(r >= n) return;
    const int slot = order[r], count = *kept;
    const bool on = r < count && (unsigned)slot < (unsigned)n;
    const T* src = reinterpret_cast<const T*>(x + (int64_t)(on ? slot / k : 0) * ldx);
    T* dst = reinterpret_cast<T*>(out + (int64_t)r * ldo);
    const int m = (int)(d / V);
#pragma unroll 4
    for(int c = threadIdx.x % L; c < m; c += L) dst[c] = on ? src[c] : T{};
}

// out[t] = c[t] + sum over j of gates[t, j] ys[place[t, j]]  (gates NULL: 1)
template <int V, int L>
__global__ __launch_bounds__(256) void expert_combine_kernel(int R, int n, int64_t d, int k,
                                                             const int32_t* __restrict__ place,
                                                             const float* __restrict__ gates,
                                                             const float* __restrict__ ys, int64_t ldy,
                                                             const float* c, int64_t ldc, float* out,
                                                             int64_t ldo) {
    typedef typename Row<V>::T T;
    const int t = (int)(blockIdx.x * (256 / L) + threadIdx.x / L);
    if(t >= R) return;
    const int m = (int)(d / V);
    const int32_t* const pt = place + (int64_t)t * k;
    const float* const gt = gates ? gates + (int64_t)t * k : nullptr;
    for(int i = threadIdx.x % L; i < m; i += L) {
        const T base = c ? reinterpret_cast<const T*>(c + (int64_t)t * ldc)[i] : T{};
        T acc = T{};
        // four choices at a time, their rows in flight together
        for(int j = 0; j < k; j += 4) {
            T v[4];
            float g[4];
            bool on[4];
#pragma unroll
            for(int e = 0; e < 4; ++e) {
                const int q = j + e < k ? pt[j + e] : -1;
                on[e] = (unsigned)q < (unsigned)n;
                g[e] = gt && j + e < k ? gt[j + e] : 1.0f;
                v[e] = reinterpret_cast<const T*>(ys + (int64_t)(on[e] ? q : 0) * ldy)[i];
            }
#pragma unroll
            for(int e = 0; e < 4; ++e)
                if(on[e]) acc = acc + g[e] * v[e];
        }
        reinterpret_cast<T*>(out + (int64_t)t * ldo)[i] = c ? acc + base : acc;
    }
}

// dys[r] (+)= gates[slot] dout[slot / k], dgates[slot] (+)= dout[slot / k] . ys[r] for
// slot = order[r]; zeros for dropped slots
template <int V>
__global__ __launch_bounds__(256) void expert_combine_bwd_kernel(
    int n, int64_t d, int k, const int32_t* __restrict__ kept, const int32_t* __restrict__ order,
    const float* __restrict__ gates, const float* __restrict__ ys, int64_t ldy,
    const float* __restrict__ dout, int64_t ldo, float* dys, int64_t ldd, float* dgates, int flags) {
    typedef typename Row<V>::T T;
    const int r = (int)(blockIdx.x * 4 + threadIdx.x / 64);
    if(r >= n) return;
    const int lane = threadIdx.x % 64, m = (int)(d / V);
    const int slot = order[r], count = *kept;
    const bool known = (unsigned)slot < (unsigned)n, on = known && r < count;
    const float g = on ? gates[slot] : 0.0f;
    const T* up = reinterpret_cast<const T*>(dout + (int64_t)(on ? slot / k : 0) * ldo);
    const T* yr = reinterpret_cast<const T*>(ys + (int64_t)r * ldy);
    T* dr = reinterpret_cast<T*>(dys + (int64_t)r * ldd);
    float dot = 0.0f;
    for(int c = lane; c < m; c += 64) {
        const T u = on ? up[c] : T{};
        if(dys) {
            const T v = on ? g * u : T{};
            dr[c] = (flags & PK_ACCUM) ? dr[c] + v : v;
        }
        if(on && dgates) dot += Row<V>::dot(u, yr[c]);
    }
    if(!dgates || !known) return;
    dot = pk::wave_sum(dot);
    if(lane == 0) dgates[slot] = (flags & PK_ACCUM2) ? dgates[slot] + dot : dot;
}

// rows to which a workgroup each is better than a wave (d 768, 2 choices, us as
// workgroups and as waves: gather of 16 slots 2.4 and 2.6, 1024 2.8 and 3.0, 2048 3.6 and
// 3.5, 8192 9.0 and 8.5; combine of 8 tokens 2.6 and 3.9, 1024 3.4 and 4.5, 2048 4.5 and
// 6.1, 4096 9.7 and 9.9)
constexpr int64_t kFewSlots = 1024, kFewTokens = 2048;

bool vec4(int64_t d, std::initializer_list<std::pair<const void*, int64_t>> xs) {
    bool v = d % 4 == 0;
    for(auto& x : xs) v = v && (!x.first || (pk::aligned16(x.first) && x.second % 4 == 0));
    return v;
}

template <class F>
void with_rows(bool vec, bool workgroup, F f) {
    using std::integral_constant;
    if(vec && workgroup) f(integral_constant<int, 4>(), integral_constant<int, 256>());
    else if(vec) f(integral_constant<int, 4>(), integral_constant<int, 64>());
    else if(workgroup) f(integral_constant<int, 1>(), integral_constant<int, 256>());
    else f(integral_constant<int, 1>(), integral_constant<int, 64>());
}

int check_rows(const char* who, int64_t n, int64_t d, int64_t k) {
    if(n < 0 || n > kMaxSlots || d < 1 || d > (int64_t)1 << 30 || k < 1 || k > kMaxTopk)
        return pk::fail("%s: need 0 <= n <= 2^25 slots, 1 <= d <= 2^30 and 1 <= k <= %d", who, kMaxTopk);
    return PK_OK;
}

}  // namespace

extern "C" int pk_route_topk_f32(int64_t R, int64_t E, int64_t k, const float* logits, int64_t ldz,
                                 int32_t* experts, float* gates, pk_stream_t stream) {
    if(int st = check_route("pk_route_topk_f32", R, E, k)) return st;
    if(R == 0) return PK_OK;
    if(!logits || !experts || !gates || ldz < E)
        return pk::fail("pk_route_topk_f32: NULL pointer or row stride < E");
    with_router_shape((int)E, (int)k, [&](auto g, auto nn) {
        constexpr int G = decltype(g)::value, N = decltype(nn)::value;
        route_topk_kernel<G, N><<<(unsigned)((R * G + 255) / 256), 256, 0, pk::as_stream(stream)>>>(
            R, (int)E, (int)k, logits, ldz, experts, gates);
    });
    return pk::launch_status("pk_route_topk_f32");
}

extern "C" int pk_route_topk_bwd_f32(int64_t R, int64_t E, int64_t k, const int32_t* experts,
                                     const float* gates, const float* dgates, float* dlogits,
                                     int64_t ldd, int flags, pk_stream_t stream) {
    if(int st = check_route("pk_route_topk_bwd_f32", R, E, k)) return st;
    if(R == 0) return PK_OK;
    if(!experts || !gates || !dgates || !dlogits || ldd < E)
        return pk::fail("pk_route_topk_bwd_f32: NULL pointer or row stride < E");
    with_router_shape((int)E, (int)k, [&](auto g, auto nn) {
        constexpr int G = decltype(g)::value, N = decltype(nn)::value;
        route_topk_bwd_kernel<G, N><<<(unsigned)((R * G + 255) / 256), 256, 0, pk::as_stream(stream)>>>(
            R, (int)E, (int)k, experts, gates, dgates, dlogits, ldd, flags & PK_ACCUM);
    });
    return pk::launch_status("pk_route_topk_bwd_f32");
}

extern "C" size_t pk_expert_plan_workspace(int64_t n, int64_t E) {
    if(n <= 0 || n > INT32_MAX || E < 1 || E > kMaxExperts) return 0;
    const int64_t c = plan_chunk(n), blocks = (n + c - 1) / c;
    return blocks > 1 ? (size_t)blocks * (size_t)(E + 1) * sizeof(int32_t) : 0;
}

extern "C" int pk_expert_plan(int64_t n, int64_t E, const int32_t* experts, int32_t* offsets,
                              int32_t* order, int32_t* place, void* workspace,
                              size_t workspace_bytes, pk_stream_t stream) {
    if(n < 0 || n > INT32_MAX || E < 1 || E > kMaxExperts)
        return pk::fail("pk_expert_plan: need 0 <= n < 2^31 slots and 1 <= E <= %d experts", kMaxExperts);
    if(!offsets || (n > 0 && (!experts || !order || !place))) return pk::fail("pk_expert_plan: NULL pointer");
    const size_t need = pk_expert_plan_workspace(n, E);
    if(need && (!workspace || workspace_bytes < need))
        return pk::fail("pk_expert_plan: workspace needs %zu bytes", need);
    const int64_t chunk = plan_chunk(n);
    const unsigned blocks = n > 0 ? (unsigned)((n + chunk - 1) / chunk) : 1;
    int bits = 1;
    while((1 << bits) < E + 2) ++bits;  // (E + 1: a lane past the end)
    hipStream_t st = pk::as_stream(stream);
    int32_t* counts = static_cast<int32_t*>(workspace);
    if(blocks > 1) plan_count<<<blocks, kPlanThreads, 0, st>>>(n, chunk, (int)E, experts, counts);
    plan_place<<<blocks, kPlanThreads, 0, st>>>(n, chunk, (int)E, bits, experts, counts, offsets, order, place);
    return pk::launch_status("pk_expert_plan");
}

extern "C" int pk_expert_gather_f32(int64_t n, int64_t d, int64_t k, int64_t E, const int32_t* offsets,
                                    const int32_t* order, const float* x, int64_t ldx, float* out,
                                    int64_t ldo, pk_stream_t stream) {
    if(int st = check_rows("pk_expert_gather_f32", n, d, k)) return st;
    if(E < 1 || n % k) return pk::fail("pk_expert_gather_f32: need E >= 1 and n a multiple of k");
    if(n == 0) return PK_OK;
    if(!offsets || !order || !x || !out || ldx < d || ldo < d)
        return pk::fail("pk_expert_gather_f32: NULL pointer or row stride < d");
    with_rows(vec4(d, {{x, ldx}, {out, ldo}}), n <= kFewSlots, [&](auto v, auto l) {
        constexpr int V = decltype(v)::value, L = decltype(l)::value;
        expert_gather_kernel<V, L><<<(unsigned)((n * L + 255) / 256), 256, 0, pk::as_stream(stream)>>>(
            (int)n, d, (int)k, offsets + E, order, x, ldx, out, ldo);
    });
    return pk::launch_status("pk_expert_gather_f32");
}

extern "C" int pk_expert_combine_f32(int64_t R, int64_t d, int64_t k, const int32_t* place,
                                     const float* gates, const float* ys, int64_t ldy, const float* c,
                                     int64_t ldc, float* out, int64_t ldo, pk_stream_t stream) {
    if(R < 0 || R > kMaxSlots) return pk::fail("pk_expert_combine_f32: need 0 <= R <= 2^25");
    if(int st = check_rows("pk_expert_combine_f32", R * k, d, k)) return st;
    if(R == 0) return PK_OK;
    if(!place || !ys || !out || ldy < d || ldo < d || (c && ldc < d))
        return pk::fail("pk_expert_combine_f32: NULL pointer or row stride < d");
    with_rows(vec4(d, {{ys, ldy}, {c, ldc}, {out, ldo}}), R <= kFewTokens, [&](auto v, auto l) {
        constexpr int V = decltype(v)::value, L = decltype(l)::value;
        expert_combine_kernel<V, L><<<(unsigned)((R * L + 255) / 256), 256, 0, pk::as_stream(stream)>>>(
            (int)R, (int)(R * k), d, (int)k, place, gates, ys, ldy, c, ldc, out, ldo);
    });
    return pk::launch_status("pk_expert_combine_f32");
}

extern "C" int pk_expert_combine_bwd_f32(int64_t R, int64_t d, int64_t k, int64_t E,
                                         const int32_t* offsets, const int32_t* order,
                                         const float* gates, const float* ys, int64_t ldy,
                                         const float* dout, int64_t ldo, float* dys, int64_t ldd,
                                         float* dgates, int flags, pk_stream_t stream) {
    if(R < 0 || R > kMaxSlots) return pk::fail("pk_expert_combine_bwd_f32: need 0 <= R <= 2^25");
    if(int st = check_rows("pk_expert_combine_bwd_f32", R * k, d, k)) return st;
    if(E < 1) return pk::fail("pk_expert_combine_bwd_f32: need E >= 1");
    if(R == 0 || (!dys && !dgates)) return PK_OK;
    if(!offsets || !order || !gates || !dout || (dgates && !ys) || (ys && ldy < d) || ldo < d ||
       (dys && ldd < d))
        return pk::fail("pk_expert_combine_bwd_f32: NULL pointer or row stride < d");
    const int64_t n = R * k;
    const unsigned grid = (unsigned)((n + 3) / 4);
    if(vec4(d, {{ys, ldy}, {dout, ldo}, {dys, ldd}}))
        expert_combine_bwd_kernel<4><<<grid, 256, 0, pk::as_stream(stream)>>>(
            (int)n, d, (int)k, offsets + E, order, gates, ys, ldy, dout, ldo, dys, ldd, dgates, flags);
    else
        expert_combine_bwd_kernel<1><<<grid, 256, 0, pk::as_stream(stream)>>>(
            (int)n, d, (int)k, offsets + E, order, gates, ys, ldy, dout, ldo, dys, ldd, dgates, flags);
    return pk::launch_status("pk_expert_combine_bwd_f32");
}
