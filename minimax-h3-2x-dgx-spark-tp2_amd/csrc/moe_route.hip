// The router of an expert layer (gfx950): every token's k best experts, their weights, and the order of the (token, choice)
// pairs by expert that the products by expert take their rows in.
//
// Per token, x_e its logits:
//   score_e = exp(x_e - max x) / sum_e exp(x_e - max x)   or   1 / (1 + exp(-x_e))
//   chosen: k times the largest of x_e (both scores rise with it, so that no rounding decides), or with a bias of score_e +
//   bias_e in 64 bits; the lowest index among equals; an expert at -inf and a NaN are never chosen
//   weight = score (/ the sum of the chosen scores) * scale
// Pair p = t k + j; order = the pairs by expert, each expert's in ascending p, then those without an expert; place[p] = where p
// went; offsets[e] = the first place of expert e.
//
// A wave takes one token: lane l holds the logits V l .. V l + V - 1 as unsigned keys of the same order, so that a round is a
// maximum over the lanes (DPP) and the lowest lane that has it; a workgroup of 16 waves takes 128 tokens at a time, and
// ranks their pairs in LDS: the lanes of 64 consecutive pairs with the same expert by one ballot per bit of its number,
// then the 64s in turn.  Up to 128 tokens one workgroup does it all; past that a second launch adds up the counts of the
// workgroups before its own (at most 512) and moves the ranks to their places.
#include <algorithm>

#include "h3fp8_common.h"

namespace {

using namespace h3;

constexpr int TB = 128;                                   // tokens of a batch
constexpr int WAVES = 16;
constexpr int MAX_BLOCKS = 512;
constexpr int MAX_E = 512, MAX_K = 16;
constexpr int CHUNKS = TB * MAX_K / 64;                   // of 64 pairs, in a batch

struct RouteArgs {
    const void* logits;
    int64_t ld;
    int64_t T;
    int E, k;
    int renorm, sigmoid;
    float scale;
    const float* bias;
    float* weights;
    int* experts;
    int* offsets;
    int* order;
    int* place;
    int* counts;                                          // [blocks, E + 1]: pairs per expert (E: without one)
    int per;                                              // tokens per workgroup, a multiple of TB
};

// fp32 as an unsigned number of the same order, 0 for what is never chosen (-inf, NaN); +0 and -0 alike.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = f2u(x + 0.0f);
    return x > -__builtin_inff() ? u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u) : 0u;
}
__device__ __forceinline__ uint64_t key_of(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
    return x > -(double)__builtin_inff() ? u ^ ((u >> 63) ? ~0ull : 1ull << 63) : 0ull;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true); }

// The maximum over the wave, in a scalar.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, dpp<0xb1>(v));                             // lane ^ 1, lane ^ 2, the other four, the other eight of 16
    v = max(v, dpp<0x4e>(v));
    v = max(v, dpp<0x141>(v));
    v = max(v, dpp<0x140>(v));
    const uint32_t a = max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16));
    const uint32_t b = max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48));
    return max(a, b);
}

// Sums over the wave in one fixed order.
__device__ __forceinline__ float wave_sum(float v) {
    v += u2f(dpp<0xb1>(f2u(v)));
    v += u2f(dpp<0x4e>(f2u(v)));
    v += u2f(dpp<0x141>(f2u(v)));
    v += u2f(dpp<0x140>(f2u(v)));
    const float a = u2f(__builtin_amdgcn_readlane((int)f2u(v), 0)) + u2f(__builtin_amdgcn_readlane((int)f2u(v), 16));
    const float b = u2f(__builtin_amdgcn_readlane((int)f2u(v), 32)) + u2f(__builtin_amdgcn_readlane((int)f2u(v), 48));
    return a + b;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ int wave_prefix(int v) {       // inclusive
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}

template <int DT>
__device__ __forceinline__ float load_logit(const void* row, int i) {
    if (DT == H3FP8_DT_F32) return reinterpret_cast<const float*>(row)[i];
    const uint16_t h = reinterpret_cast<const uint16_t*>(row)[i];
    return DT == H3FP8_DT_FP16 ? fp16_to_f32(h) : bf16_to_f32(h);
}

// The logits of lane l, V l on; past E: -inf.
template <int DT, int V>
__device__ __forceinline__ void load_token(const RouteArgs& a, int64_t t, int lane, float (&x)[V]) {
    const char* row = reinterpret_cast<const char*>(a.logits) + t * a.ld * (DT == H3FP8_DT_F32 ? 4 : 2);
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = V * lane + v < a.E ? load_logit<DT>(row, V * lane + v) : -__builtin_inff();
}

// One token by one wave: lane j < k returns choice j (expert or -1, weight).
template <int V, bool BIAS>
__device__ __forceinline__ void pick(const RouteArgs& a, const float (&x)[V], int lane, int& expert, float& weight) {
    float top = x[0];
    bool nan = false;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        top = fmaxf(top, x[v]);
        nan = nan || x[v] != x[v];
    }
    const bool any_nan = __ballot(nan) != 0;
    const uint32_t top_key = wave_max(key_of(top));       // 0: every logit is masked
    const float xmax = top_key == 0 ? 0.0f : u2f((top_key >> 31) ? top_key ^ 0x80000000u : ~top_key);
    expert = -1;
    float mine = 0.0f, score = 0.0f;                      // lane j: the logit of choice j, its score
    double score64 = 0.0;
    if constexpr (BIAS) {
        double s[V], sum = 0.0;
        uint64_t key[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            s[v] = a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[v])) : exp((double)x[v] - (double)xmax);
            sum += s[v] == s[v] ? s[v] : 0.0;             // a NaN is not among those to choose from
        }
        if (!a.sigmoid) {
            sum = wave_sum(sum);
#pragma unroll
            for (int v = 0; v < V; ++v) s[v] = s[v] / sum;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int e = V * lane + v;
            // beside an infinite logit there are no scores: such a token's experts go by the bias
            const double base = s[v] == s[v] ? s[v] : 0.0;
            key[v] = e < a.E && x[v] > -__builtin_inff() ? key_of(base + (double)a.bias[e]) : 0ull;
        }
        for (int j = 0; j < a.k; ++j) {
            uint64_t best = key[0];
            double bs = s[0];
            int bv = 0;
#pragma unroll
            for (int v = 1; v < V; ++v)
                if (key[v] > best) best = key[v], bs = s[v], bv = v;
            const uint32_t hi = wave_max((uint32_t)(best >> 32));
            const uint32_t lo = wave_max((uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
            if ((hi | lo) == 0) break;
            const int win = __builtin_ctzll(__ballot(best == (((uint64_t)hi << 32) | lo)));
            const int e = __builtin_amdgcn_readlane(V * lane + bv, win);
            const double es = __shfl(bs, win, 64);
            if (lane == j) expert = e, score64 = es;
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (V * lane + v == e) key[v] = 0ull;
        }
        if (a.renorm) {
            const double total = wave_sum(lane < a.k ? score64 : 0.0);
            score64 = total == 0.0 ? 0.0 : score64 / total;
        }
        weight = (float)(score64 * (double)a.scale);
    } else {
        uint32_t key[V];
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            key[v] = key_of(x[v]);
            if (!a.sigmoid && !a.renorm) sum += expf(x[v] - xmax);
        }
        if (!a.sigmoid && !a.renorm) sum = wave_sum(sum);
        for (int j = 0; j < a.k; ++j) {
            uint32_t best = key[0];
            int bv = 0;
#pragma unroll
            for (int v = 1; v < V; ++v)
                if (key[v] > best) best = key[v], bv = v;
            const uint32_t m = wave_max(best);
            if (m == 0) break;
            const int win = __builtin_ctzll(__ballot(best == m));
            const int e = __builtin_amdgcn_readlane(V * lane + bv, win);
            if (lane == j) expert = e, mine = u2f((m >> 31) ? m ^ 0x80000000u : ~m);
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (V * lane + v == e) key[v] = 0u;
        }
        if (expert >= 0) {
            const float t = expf(a.sigmoid ? -fabsf(mine) : mine - xmax);
            score = a.sigmoid ? (mine >= 0.0f ? 1.0f : t) / (1.0f + t) : t;
        }
        if (a.renorm) sum = wave_sum(score);
        else if (a.sigmoid) sum = 1.0f;
        weight = sum == 0.0f ? 0.0f : score / sum * a.scale;
    }
    if (any_nan) weight = __builtin_nanf("");
    if (expert < 0) weight = 0.0f;
}

struct RouteLds {
    int expert[TB * MAX_K];                               // of the batch's pairs; E: none
    uint16_t count[CHUNKS * (MAX_E + 2)];                 // per 64 pairs and expert (rows of E + 1 rounded up to even), then what comes before them
    int run[MAX_E + 1];                                   // of the batches before
    int base[MAX_E + 1];
};

// The exclusive sums of total[0 .. E] into base, by one wave.
__device__ __forceinline__ void scan(const int* total, int* base, int E, int lane) {
    int carry = 0;
    for (int e0 = 0; e0 <= E; e0 += 64) {
        const int e = e0 + lane, n = e <= E ? total[e] : 0, s = wave_prefix(n);
        if (e <= E) base[e] = carry + s - n;
        carry += __builtin_amdgcn_readlane(s, 63);
    }
}

template <int DT, int V, bool BIAS>
__global__ void __launch_bounds__(WAVES * 64) moe_route_pick_kernel(RouteArgs a) {
    extern __shared__ __attribute__((aligned(16))) char route_lds[];
    RouteLds& s = *reinterpret_cast<RouteLds*>(route_lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int E = a.E, k = a.k, bits = 32 - __builtin_clz((unsigned)E);
    const int64_t first = (int64_t)blockIdx.x * a.per, last = min(first + a.per, a.T);
    const int row = (E + 2) & ~1;
    for (int e = threadIdx.x; e <= E; e += WAVES * 64) s.run[e] = 0;
    for (int64_t t0 = first; t0 < last; t0 += TB) {
        const int n = (int)min<int64_t>(TB, last - t0), pairs = n * k, chunks = (pairs + 63) / 64;
        for (int i = threadIdx.x; i < chunks * row / 2; i += WAVES * 64) reinterpret_cast<uint32_t*>(s.count)[i] = 0;
        float x[V], next[V];
        if (wave < n) load_token<DT, V>(a, t0 + wave, lane, x);
        for (int i = wave; i < n; i += WAVES) {
            if (i + WAVES < n) load_token<DT, V>(a, t0 + i + WAVES, lane, next);
            int expert;
            float weight;
            pick<V, BIAS>(a, x, lane, expert, weight);
            if (lane < k) {
                const int64_t p = (t0 + i) * k + lane;
                a.weights[p] = weight;
                a.experts[p] = expert;
                s.expert[i * k + lane] = expert < 0 ? E : expert;
            }
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = next[v];
        }
        __syncthreads();
        // ranks within 64 pairs
        int rank[CHUNKS / WAVES];
#pragma unroll
        for (int i = 0; i < CHUNKS / WAVES; ++i) {
            const int c = wave + i * WAVES, q = 64 * c + lane;
            if (c >= chunks) break;
            const bool in = q < pairs;
            const int e = in ? s.expert[q] : -1;
            uint64_t peers = __ballot(in);
            for (int b = 0; b < bits; ++b) {
                const bool bit = (e >> b) & 1;
                const uint64_t m = __ballot(bit);
                peers &= bit ? m : ~m;
            }
            rank[i] = __popcll(peers & ((1ull << lane) - 1));
            if (in && rank[i] == 0) s.count[c * row + e] = (uint16_t)__popcll(peers);
        }
        __syncthreads();
        for (int e = threadIdx.x; e <= E; e += WAVES * 64) {
            int sum = 0;
            for (int c = 0; c < chunks; ++c) {
                const int m = s.count[c * row + e];
                s.count[c * row + e] = (uint16_t)sum;
                sum += m;
            }
            s.base[e] = s.run[e];
            s.run[e] += sum;
        }
        __syncthreads();
        if (a.counts == nullptr) {                        // the only batch: s.run are the totals
            if (wave == 0) scan(s.run, s.base, E, lane);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < CHUNKS / WAVES; ++i) {
            const int c = wave + i * WAVES, q = 64 * c + lane;
            if (c >= chunks || q >= pairs) break;
            const int e = s.expert[q], at = s.base[e] + s.count[c * row + e] + rank[i];
            a.place[t0 * k + q] = at;                     // with more than one workgroup: within this one's, moved later
            if (a.counts == nullptr) a.order[at] = (int)(t0 * k) + q;
        }
        __syncthreads();
    }
    if (a.counts == nullptr) {
        if (first >= last) {
            for (int e = threadIdx.x; e <= E; e += WAVES * 64) a.offsets[e] = 0;
        } else {
            for (int e = threadIdx.x; e <= E; e += WAVES * 64) a.offsets[e] = s.base[e];
        }
    } else {
        for (int e = threadIdx.x; e <= E; e += WAVES * 64) a.counts[(int64_t)blockIdx.x * (E + 1) + e] = s.run[e];
    }
}

// The pairs of workgroup b of the first launch to their places: counts of the workgroups before it, and offsets.
__global__ void __launch_bounds__(WAVES * 64) moe_route_place_kernel(RouteArgs a, int blocks) {
    __shared__ int before[MAX_E + 1], total[MAX_E + 1], base[MAX_E + 1];
    const int lane = threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int n = a.E + 1;
    for (int e = threadIdx.x; e < n; e += WAVES * 64) before[e] = total[e] = 0;
    __syncthreads();
    // a thread sums one expert's counts of every parts-th workgroup; LDS adds of whole numbers, in any order
    const int parts = max(1, WAVES * 64 / n);
    for (int i = threadIdx.x; i < n * parts; i += WAVES * 64) {
        const int e = i % n;
        int lo = 0, all = 0;
        for (int b = i / n; b < blocks; b += parts) {
            const int c = a.counts[(int64_t)b * n + e];
            all += c;
            lo += b < (int)blockIdx.x ? c : 0;
        }
        atomicAdd(&before[e], lo);
        atomicAdd(&total[e], all);
    }
    __syncthreads();
    if (wave == 0) scan(total, base, a.E, lane);
    __syncthreads();
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e < n; e += WAVES * 64) a.offsets[e] = base[e];
    const int64_t first = (int64_t)blockIdx.x * a.per * a.k, last = min((int64_t)(blockIdx.x + 1) * a.per, a.T) * a.k;
    for (int64_t p = first + threadIdx.x; p < last; p += WAVES * 64) {
        const int x = a.experts[p], e = x < 0 ? a.E : x, at = base[e] + before[e] + a.place[p];
        a.place[p] = at;
        a.order[at] = (int)p;
    }
}

// Tokens per workgroup of the first launch.
int64_t per_block(int64_t T) { return TB * std::max<int64_t>(1, (T + (int64_t)TB * MAX_BLOCKS - 1) / ((int64_t)TB * MAX_BLOCKS)); }

template <int DT, int V>
int launch_pick(const RouteArgs& a, unsigned blocks, hipStream_t st) {
    if (a.bias) hipLaunchKernelGGL((moe_route_pick_kernel<DT, V, true>), dim3(blocks), dim3(WAVES * 64), sizeof(RouteLds), st, a);
    else hipLaunchKernelGGL((moe_route_pick_kernel<DT, V, false>), dim3(blocks), dim3(WAVES * 64), sizeof(RouteLds), st, a);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

template <int DT>
int launch_width(const RouteArgs& a, unsigned blocks, hipStream_t st) {
    if (a.E <= 64) return launch_pick<DT, 1>(a, blocks, st);
    if (a.E <= 128) return launch_pick<DT, 2>(a, blocks, st);
    if (a.E <= 256) return launch_pick<DT, 4>(a, blocks, st);
    return launch_pick<DT, 8>(a, blocks, st);
}

}  // namespace

extern "C" int64_t h3fp8_moe_route_workspace(int64_t T, int64_t E) {
    if (T <= TB || E < 0) return 0;
    return (T + per_block(T) - 1) / per_block(T) * (E + 1) * 4;
}

extern "C" int h3fp8_moe_route(const void* logits, int64_t ld, int dtype, int64_t T, int64_t E, int k, int scoring, int renorm,
                               float scale, const float* bias, float* weights, int32_t* experts, int32_t* offsets,
                               int32_t* order, int32_t* place, void* workspace, int64_t workspace_bytes, void* stream) {
    H3_REQUIRE(T >= 0 && E >= 1 && E <= MAX_E, "h3fp8_moe_route: %lld tokens, %lld experts (1 to %d)", (long long)T, (long long)E, MAX_E);
    H3_REQUIRE(k >= 1 && k <= MAX_K && k <= E, "h3fp8_moe_route: k = %d of %lld experts (1 to %d)", k, (long long)E, MAX_K);
    H3_REQUIRE(T <= 0x7fffffff / k, "h3fp8_moe_route: too many tokens");
    H3_REQUIRE(dtype == H3FP8_DT_BF16 || dtype == H3FP8_DT_FP16 || dtype == H3FP8_DT_F32, "h3fp8_moe_route: bad dtype %d", dtype);
    H3_REQUIRE(scoring == 0 || scoring == 1, "h3fp8_moe_route: bad scoring %d", scoring);
    H3_REQUIRE(offsets && (T == 0 || (logits && weights && experts && order && place)), "h3fp8_moe_route: null pointer");
    H3_REQUIRE(T <= 1 || ld >= 0, "h3fp8_moe_route: negative stride");
    const unsigned elem = dtype == H3FP8_DT_F32 ? 4 : 2;
    H3_REQUIRE((((uintptr_t)logits & (elem - 1)) | (((uintptr_t)bias | (uintptr_t)weights | (uintptr_t)experts | (uintptr_t)offsets |
                (uintptr_t)order | (uintptr_t)place | (uintptr_t)workspace) & 3)) == 0, "h3fp8_moe_route: misaligned pointer");
    const int64_t need = h3fp8_moe_route_workspace(T, E);
    H3_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "h3fp8_moe_route: the workspace needs %lld bytes", (long long)need);
    RouteArgs a{};
    a.logits = logits; a.ld = ld; a.T = T; a.E = (int)E; a.k = k; a.renorm = renorm != 0; a.sigmoid = scoring; a.scale = scale;
    a.bias = bias; a.weights = weights; a.experts = experts; a.offsets = offsets; a.order = order; a.place = place;
    a.counts = need ? (int*)workspace : nullptr;
    a.per = (int)per_block(T);
    const unsigned blocks = (unsigned)std::max<int64_t>(1, (T + a.per - 1) / a.per);
    hipStream_t st = (hipStream_t)stream;
    const int rc = dtype == H3FP8_DT_F32 ? launch_width<H3FP8_DT_F32>(a, blocks, st)
                   : dtype == H3FP8_DT_FP16 ? launch_width<H3FP8_DT_FP16>(a, blocks, st)
                                            : launch_width<H3FP8_DT_BF16>(a, blocks, st);
    if (rc || !need) return rc;
    hipLaunchKernelGGL(moe_route_place_kernel, dim3(blocks), dim3(WAVES * 64), 0, st, a, (int)blocks);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}
