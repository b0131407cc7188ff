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
// 16 lanes take a token, a wave four; a lane holds V of its logits (2 to 32: E / 16 or up to twice that).  The choice goes by one
// threshold and a ranking of what reaches it, 16 lanes against each other (DPP); rounds over all the logits only where that leaves
// more than 16 (see pick).  With a bias it goes by fp32 scores, and what could be among the k best by their error is scored and
// ranked again in 64 bits, a lane each; only where more than 16 are within that error, all are.
// A workgroup of 16 waves takes 64 tokens at a time, and ranks the pairs of 128 in LDS: the lanes of 64 consecutive pairs with the
// same expert by one ballot per bit of its number, then the 64s in turn.  Up to 128 tokens one workgroup does it all; past that
// a second launch adds up the counts of the workgroups before its own (at most 256) and moves the ranks to their places.
//
// us of the kernels: a token of 32 experts, k 4: 3.7; 64 tokens of 256, k 8, sigmoid with bias 10.4 (64-bit scores of all experts:
// 32, their registers in memory 27); 32768 tokens of 256, k 8, fp32: 15.2 + 8.5 (k rounds with one expert taken out in each 62 in
// all, k rounds of 16 lanes a token 29, by difference instead of by taking out 27), the logits' bytes alone 6.8.  What bounds it:
// a workgroup's way from load to places, 7 to 9 us, and past 64 tokens per CU the vector instructions (131072 tokens 41 us, bf16);
// the second launch its reads of all counts (256 rows of E + 1 from L2 in each workgroup).
#include <algorithm>

#include "h3fp8_common.h"

namespace {

using namespace h3;

constexpr int TB = 128;                                   // tokens of a batch; what one workgroup takes without a second launch
constexpr int WAVES = 16;                                 // of a workgroup; 8 where a lane holds 32 logits and 64-bit scores
constexpr int MAX_BLOCKS = 256;
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
    int* counts;                                          // [blocks, row]: pairs per expert (E: without one)
    int row;                                              // E + 1 rounded up to 4
    int vec;                                              // the logits' rows take 16-byte loads
    int vec_bias;                                         // so do four biases
    int per;                                              // tokens per workgroup
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

// Over the 16 lanes of a token, in all of them: lane ^ 1, lane ^ 2, the other four of eight, the other eight.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, dpp<0xb1>(v));
    v = max(v, dpp<0x4e>(v));
    v = max(v, dpp<0x141>(v));
    return max(v, dpp<0x140>(v));
}
__device__ __forceinline__ uint32_t min16(uint32_t v) {
    v = min(v, dpp<0xb1>(v));
    v = min(v, dpp<0x4e>(v));
    v = min(v, dpp<0x141>(v));
    return min(v, dpp<0x140>(v));
}
__device__ __forceinline__ float sum16(float v) {
    v += u2f(dpp<0xb1>(f2u(v)));
    v += u2f(dpp<0x4e>(f2u(v)));
    v += u2f(dpp<0x141>(f2u(v)));
    return v + u2f(dpp<0x140>(f2u(v)));
}
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)dpp<CTRL>((uint32_t)(u >> 32)) << 32 | dpp<CTRL>((uint32_t)u)));
}
__device__ __forceinline__ double sum16(double v) {
    v += dpp64<0xb1>(v);
    v += dpp64<0x4e>(v);
    v += dpp64<0x141>(v);
    return v + dpp64<0x140>(v);
}
// Exclusive prefix sums over the 16 lanes.
__device__ __forceinline__ int prefix16(int n) {
    int v = n;
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    return v - n;
}
// Lane `at` of each 16.
__device__ __forceinline__ int lane16(int v, int at, int lane) { return __shfl(v, (lane & ~15) + at, 64); }
__device__ __forceinline__ double lane16(double v, int at, int lane) { return __shfl(v, (lane & ~15) + at, 64); }

__device__ __forceinline__ int wave_prefix(int v) {       // inclusive
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}

// A lane's logits: element v is expert at(v) + W l16, so that 16 lanes read 16 W consecutive ones at once (W of them 16 bytes).
template <int DT, int V>
struct Lay {
    static constexpr int FULL = DT == H3FP8_DT_F32 ? 4 : 8, W = V < FULL ? V : FULL;
    __host__ __device__ static constexpr int at(int v) { return v / W * 16 * W + v % W; }
};

template <int DT>
__device__ __forceinline__ float load_logit(const void* row, int i) {
    if (DT == H3FP8_DT_F32) return reinterpret_cast<const float*>(row)[i];
    const uint16_t h = reinterpret_cast<const uint16_t*>(row)[i];
    return DT == H3FP8_DT_FP16 ? fp16_to_f32(h) : bf16_to_f32(h);
}

template <int DT, int V>
__device__ __forceinline__ void load_token(const RouteArgs& a, const char* row, bool live, int l16, float (&x)[V]) {
    using L = Lay<DT, V>;
    constexpr int SIZE = DT == H3FP8_DT_F32 ? 4 : 2;
    if (L::W == L::FULL && a.vec) {
#pragma unroll
        for (int v = 0; v < V; v += L::W) {
            const int e = L::at(v) + L::W * l16;
            const v4u u = live && e < a.E ? *reinterpret_cast<const v4u*>(row + e * SIZE) : v4u{0u, 0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < L::W; ++i) {
                const uint32_t h = SIZE == 4 ? u[i & 3] : (u[(i >> 1) & 3] >> (16 * (i & 1))) & 0xffffu;
                const float f = SIZE == 4 ? u2f(h) : DT == H3FP8_DT_FP16 ? fp16_to_f32(h) : bf16_to_f32(h);
                x[v + i] = live && e < a.E ? f : -__builtin_inff();
            }
        }
        return;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = L::at(v) + L::W * l16;
        x[v] = live && e < a.E ? load_logit<DT>(row, e) : -__builtin_inff();
    }
}

__device__ __forceinline__ float value_of(uint32_t key) { return u2f((key >> 31) ? key ^ 0x80000000u : ~key); }

// The largest of the lane's keys, over the 16 lanes; 0: none is left.
template <int V>
__device__ __forceinline__ uint32_t best16(const uint32_t (&key)[V]) {
    uint32_t m = key[0];
#pragma unroll
    for (int v = 1; v < V; ++v) m = max(m, key[v]);
    return max16(m);
}

// The largest key below m != 0, over the 16 lanes; 0: none.  m - 1 - key, as an unsigned number, is smallest for it: keys from m on
// wrap to 2^32 - 1 - (key - m), which is more than m - 1 - other for any other key, two keys being less than 2^32 apart.
template <int V>
__device__ __forceinline__ uint32_t next16(const uint32_t (&key)[V], uint32_t m) {
    uint32_t d = m - 1 - key[0];
#pragma unroll
    for (int v = 1; v < V; ++v) d = min(d, m - 1 - key[v]);
    const uint32_t next = m - 1 - min16(d);
    return next < m ? next : 0u;
}

// The lowest index whose key is m, which is taken out.
template <int DT, int V>
__device__ __forceinline__ int take16(uint32_t (&key)[V], uint32_t m, int l16) {
    using L = Lay<DT, V>;
    uint32_t c = 0xffff0000u;
#pragma unroll
    for (int v = V - 1; v >= 0; --v) c = key[v] == m ? (uint32_t)L::at(v) : c;
    const uint32_t e = min16(c + (uint32_t)(L::W * l16)), mine = e - (uint32_t)(L::W * l16);
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = mine == (uint32_t)L::at(v) ? 0u : key[v];
    return (int)e;
}

__device__ __forceinline__ double score64(const RouteArgs& a, double x, double top, double sum) {
    return a.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - top) / sum;
}

// The biases of a lane's experts, -inf past the last.
template <int DT, int V>
__device__ __forceinline__ void load_bias(const RouteArgs& a, int l16, float (&b)[V]) {
    using L = Lay<DT, V>;
    typedef float v4f __attribute__((ext_vector_type(4)));
    if (L::W >= 4 && a.vec_bias) {
#pragma unroll
        for (int v = 0; v < V; v += 4) {
            const int e = L::at(v) + L::W * l16;
            const v4f q = e < a.E ? *reinterpret_cast<const v4f*>(a.bias + e) : v4f{} - __builtin_inff();
#pragma unroll
            for (int u = 0; u < 4; ++u) b[(v + u) % V] = q[u];
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int e = L::at(v) + L::W * l16;
            b[v] = e < a.E ? a.bias[e] : -__builtin_inff();
        }
    }
}

// Whether lane `other` (rotated in) comes before this one: by key, then by index.
template <class K, int N>
__device__ __forceinline__ int rank_step(K key, int e) {
    constexpr int ROR = 0x120 + N;
    uint64_t o = dpp<ROR>((uint32_t)key);
    if constexpr (sizeof(K) == 8) o |= (uint64_t)dpp<ROR>((uint32_t)(key >> 32)) << 32;
    const int oe = (int)dpp<ROR>((uint32_t)e);
    return o > key || (o == key && oe < e) ? 1 : 0;
}
template <class K>
__device__ __forceinline__ int rank16(K key, int e) {
    return rank_step<K, 1>(key, e) + rank_step<K, 2>(key, e) + rank_step<K, 3>(key, e) + rank_step<K, 4>(key, e) + rank_step<K, 5>(key, e) +
           rank_step<K, 6>(key, e) + rank_step<K, 7>(key, e) + rank_step<K, 8>(key, e) + rank_step<K, 9>(key, e) + rank_step<K, 10>(key, e) +
           rank_step<K, 11>(key, e) + rank_step<K, 12>(key, e) + rank_step<K, 13>(key, e) + rank_step<K, 14>(key, e) + rank_step<K, 15>(key, e);
}

// How many of the other 15 lanes have a larger key.
template <int N = 1>
__device__ __forceinline__ int above16(uint32_t key) {
    const int more = dpp<0x120 + N>(key) > key ? 1 : 0;
    if constexpr (N < 15) return more + above16<N + 1>(key);
    return more;
}

// A wave's LDS accesses in order, for the compiler.
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Four tokens by a wave: lane j < k of each token's 16 returns choice j (expert or -1, weight).  token: the lane's row of logits.
//
// The k-th largest of the 16 lanes' own largest keys is one that the k best reach.  Where up to 16 experts reach it, as mostly with
// up to 8 choices (it takes 10.6 draws to meet 8 of 16 lanes), they get a lane each and are ranked.  Else k rounds, each the
// largest key below the last, leave the key of the k-th best, unless some are equal a later one.  With a bias both keys are lowered
// by what the fp32 scores may be off by.
template <int DT, int V, bool BIAS>
__device__ __forceinline__ void pick(const RouteArgs& a, const void* token, float (&x)[V], int lane, int* scratch, int& expert, float& weight) {
    using L = Lay<DT, V>;
    const int l16 = lane & 15;
    float top = x[0];
    bool nan = false;
#pragma unroll
    for (int v = 0; v < V; v += 2) {
        top = fmaxf(fmaxf(top, x[v]), x[v + 1]);
        nan = nan || __builtin_isunordered(x[v], x[v + 1]);
    }
    const bool any_nan = max16(nan ? 1u : 0u) != 0;
    const uint32_t top_key = max16(key_of(top));          // 0: every logit is masked
    const float xmax = top_key == 0 ? 0.0f : value_of(top_key);
    // the softmax's sum: terms by the hardware's exponential; those that count have small exponents
    float sum = 0.0f;
    if (!a.sigmoid && (BIAS || !a.renorm)) {
#pragma unroll
        for (int v = 0; v < V; ++v) sum += __builtin_amdgcn_exp2f((x[v] - xmax) * 1.4426950408889634f);
        sum = sum16(sum);
    }
    // what the rounds go by: the logit, or score + bias in fp32; beside an infinite logit there are no scores: those experts go by
    // the bias.  Two scores of a token, s and s', are off against each other
    //   - by their own exponentials, products and reciprocals (1 ulp each) and the rounding of the exponents' arguments (s |d| 2^-22.8,
    //     where s is at most exp(-|d|)): 2^-21 in all, a sigmoid's, both of which may be near 1, 2^-20;
    //   - with softmax by the sum: (V + 4) 2^-24 of it for the additions of a lane and between lanes, up to 2^-18.8, and 2^-20.8 for its
    //     terms.  That is one factor of all scores, so it takes |s - s'| <= 1 times as much from their difference;
    //   - by 2^-23 (1 + |sum|) for the two roundings of score + bias.
    // All together 0.85 (1 + |sum|) 2^-18 at most: the margin of 2^-18 (1 + |sum|) below keeps every expert that 64 bits could choose.
    if constexpr (BIAS) {
        float b[V];
        load_bias<DT, V>(a, l16, b);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float t = __builtin_amdgcn_exp2f((a.sigmoid ? -x[v] : x[v] - xmax) * 1.4426950408889634f);
            const float s = __builtin_amdgcn_rcpf(a.sigmoid ? 1.0f + t : sum) * (a.sigmoid ? 1.0f : t);
            x[v] = x[v] > -__builtin_inff() ? (s == s ? s : 0.0f) + b[v] : -__builtin_inff();
        }
    }
    // those from the value of `least` on (with a bias: less what the fp32 scores may be off by), the lane's place among them and
    // their number
    uint32_t in = 0;                                      // bit v: element v is one
    int at = 0, total = 0;
    bool flat = false;
    auto choose = [&](uint32_t least) {
        const float edge = value_of(least);
        flat = BIAS && (any_nan || !(fabsf(edge) < __builtin_inff()));
        const float lowest = -0x1.fffffep127f;
        const float from = least == 0 ? __builtin_nanf("") : BIAS ? fmaxf(edge - 0x1p-18f * (1.0f + fabsf(edge)), lowest) : edge;
        in = 0;
#pragma unroll
        for (int v = V - 1; v >= 0; --v) in = 2 * in + (x[v] >= from ? 1u : 0u);
        const int n = __popc(in);
        at = prefix16(n);
        total = lane16(at + n, 15, lane);
    };
    const bool some = top_key != 0;
    bool done = false;
    if (a.k <= 8) {
        if (BIAS) {
            top = x[0];
#pragma unroll
            for (int v = 1; v < V; ++v) top = fmaxf(top, x[v]);
        }
        const uint32_t m = key_of(top), least = min16(above16(m) < a.k ? m : 0xffffffffu);
        choose(least);
        done = __ballot(some && (least == 0 || total > 16)) == 0;
    }
    if (!done) {
        uint32_t key[V];
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = key_of(x[v]);
        uint32_t least = best16(key);
        for (int j = 1; j < a.k; ++j) {
            const uint32_t m = next16(key, least);
            if (__ballot(m != 0) == 0) break;
            least = m != 0 ? m : least;
        }
        choose(least);
    }
    double sum64 = 1.0;
    if (BIAS && !a.sigmoid) {
        sum64 = 0.0;
#pragma unroll 1
        for (int v = 0; v < V; ++v) {
            const int e = L::at(v) + L::W * l16;
            const double t = e < a.E ? exp((double)load_logit<DT>(token, e) - (double)xmax) : 0.0;
            sum64 += t == t ? t : 0.0;                    // a NaN is not among those to choose from
        }
        sum64 = sum16(sum64);
    }
    expert = -1;
    float mine = 0.0f;                                    // lane j: the logit of choice j, or
    double mine64 = 0.0;                                  // ... its score
    if (__ballot(some && (total > 16 || flat)) == 0) {
        int* list = scratch + (lane & ~15);
        while (__ballot(in != 0)) {
            if (in != 0) {
                const int v = __ffs((int)in) - 1;
                list[at++] = L::at(v) + L::W * l16;
                in &= in - 1;
            }
        }
        wave_order();
        const bool has = l16 < total;
        const int e = has ? list[l16] : 0xffff;
        const float f = has ? load_logit<DT>(token, e) : 0.0f;
        int rank;
        double s = 0.0;
        if constexpr (BIAS) {
            s = has ? score64(a, (double)f, (double)xmax, sum64) : 0.0;
            const uint64_t k64 = has ? key_of((s == s ? s : 0.0) + (double)a.bias[e]) : 0ull;
            rank = rank16(k64, e);
        } else {
            rank = rank16(has ? key_of(f) : 0u, e);
        }
        wave_order();
        if (has && rank < a.k) list[rank] = e | (l16 << 16);
        wave_order();
        const int got = l16 < min(total, a.k) ? list[l16] : l16 << 16, from = got >> 16;
        if (l16 < min(total, a.k)) expert = got & 0xffff;
        if constexpr (BIAS) mine64 = lane16(s, from, lane);
        else mine = u2f((uint32_t)lane16((int)f2u(f), from, lane));
    } else if constexpr (BIAS) {
        // all of them again in every round, from memory: few registers, and rarely
        uint64_t taken = 0;
#pragma unroll 1
        for (int j = 0; j < a.k; ++j) {
            uint64_t best = 0;
            double bs = 0.0;
            int bv = 0;
#pragma unroll 1
            for (int v = 0; v < V; ++v) {
                const int e = L::at(v) + L::W * l16;
                if (e >= a.E || ((taken >> v) & 1)) continue;
                const float f = load_logit<DT>(token, e);
                const double s = score64(a, (double)f, (double)xmax, sum64);
                const uint64_t o = f > -__builtin_inff() ? key_of((s == s ? s : 0.0) + (double)a.bias[e]) : 0ull;
                if (o > best) best = o, bs = s, bv = v;
            }
            const uint32_t hi = max16((uint32_t)(best >> 32)), lo = max16((uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
            const bool at_best = best != 0 && best == ((uint64_t)hi << 32 | lo);
            const uint32_t own = at_best ? (uint32_t)(L::at(bv) + L::W * l16) : 0xffff0000u, e = min16(own);
            const int by = (int)max16(own == e && at_best ? (uint32_t)l16 : 0u);
            const double s = lane16(bs, by, lane);
            if (own == e && at_best) taken |= 1ull << bv;
            if (l16 == j && e < 0xffff0000u) expert = (int)e, mine64 = s;
        }
    } else {
        // more than 16 reach it: equal ones, taken one by one, the lowest index first
        uint32_t key[V];
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = key_of(x[v]);
        for (int j = 0; j < a.k; ++j) {
            const uint32_t m = best16(key);
            const int e = take16<DT, V>(key, m, l16);
            if (l16 == j && m != 0) expert = e, mine = value_of(m);
        }
    }
    if constexpr (BIAS) {
        if (expert < 0) mine64 = 0.0;
        if (a.renorm) {
            const double all = sum16(mine64);
            mine64 = all == 0.0 ? 0.0 : mine64 / all;
        }
        weight = (float)(mine64 * (double)a.scale);
    } else {
        float score = 0.0f;
        if (a.sigmoid) {
            // over their sum the scores count by their quotients, which are ordinary numbers where fp32 cannot hold the scores
            // themselves (subnormal from -87, 0 from -104 on): as multiples of exp(the best logit) where that is below 1.  From where
            // float64 cannot hold one either, 1 + exp(-x) infinite, it is 0, as with a bias.
            const float low = a.renorm ? fminf(xmax, 0.0f) : 0.0f, t = expf(-fabsf(mine));
            const float up = mine >= 0.0f ? 1.0f : expf(mine - low);
            if (expert >= 0 && mine > -709.78271484375f) score = up / (1.0f + t);
        } else if (expert >= 0) {
            score = expf(mine - xmax);
        }
        if (a.renorm) sum = sum16(score);
        else if (a.sigmoid) sum = 1.0f;
        weight = sum == 0.0f ? 0.0f : score / sum * a.scale;
    }
    if (any_nan) weight = __builtin_nanf("");
    if (expert < 0) weight = 0.0f;
}

constexpr int pick_waves(int V, bool bias) { return V > 16 && bias ? WAVES / 2 : WAVES; }

struct RouteLds {
    int expert[TB * MAX_K];                               // of the batch's pairs; E: none
    uint16_t count[CHUNKS * (MAX_E + 2)];                 // per 64 pairs and expert (rows of E + 1 rounded up to even), then what comes before them
    int scratch[WAVES * 64];
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
__global__ void __launch_bounds__(pick_waves(V, BIAS) * 64) moe_route_pick_kernel(RouteArgs a) {
    constexpr int WAVES = pick_waves(V, BIAS);
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
        const int l16 = lane & 15;
        for (int i0 = 4 * wave; i0 < n; i0 += 4 * WAVES) {
            const int i = i0 + (lane >> 4);
            const char* token = reinterpret_cast<const char*>(a.logits) + (t0 + min(i, n - 1)) * a.ld * (DT == H3FP8_DT_F32 ? 4 : 2);
            float x[V];
            load_token<DT, V>(a, token, i < n, l16, x);
            int expert;
            float weight;
            pick<DT, V, BIAS>(a, token, x, lane, s.scratch + wave * 64, expert, weight);
            if (i < n && l16 < k) {
                const int64_t p = (t0 + i) * k + l16;
                a.weights[p] = weight;
                a.experts[p] = expert;
                s.expert[i * k + l16] = expert < 0 ? E : expert;
            }
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
        for (int e = threadIdx.x; e <= E; e += WAVES * 64) a.counts[(int64_t)blockIdx.x * a.row + e] = s.run[e];
    }
}

// The pairs of workgroup b of the first launch to their places: counts of the workgroups before it, and offsets.  (With a launch
// between the two that sums the counts once: 2048 tokens of 256, k 8 22 us against 14, 32768 27 against 26, 131072 59 against 55.)
__global__ void __launch_bounds__(WAVES * 64) moe_route_place_kernel(RouteArgs a, int blocks) {
    __shared__ int before[MAX_E + 4], total[MAX_E + 4], base[MAX_E + 1];
    const int lane = threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int n = a.E + 1, quads = a.row / 4;
    for (int e = threadIdx.x; e < a.row; e += WAVES * 64) before[e] = total[e] = 0;
    __syncthreads();
    // a thread sums four experts' counts of every parts-th workgroup, eight loads under way; LDS adds of whole numbers, in any order
    typedef int v4i __attribute__((ext_vector_type(4)));
    const int parts = WAVES * 64 / quads, q = threadIdx.x % quads, part = threadIdx.x / quads;
    if (part < parts) {
        v4i lo = {0, 0, 0, 0}, all = {0, 0, 0, 0};
        for (int b0 = part; b0 < blocks; b0 += 8 * parts) {
            v4i c[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int b = b0 + u * parts;
                c[u] = b < blocks ? *reinterpret_cast<const v4i*>(a.counts + (int64_t)b * a.row + 4 * q) : v4i{0, 0, 0, 0};
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                all += c[u];
                if (b0 + u * parts < (int)blockIdx.x) lo += c[u];
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (4 * q + u < n) {                          // the rows' last places hold nothing
                atomicAdd(&before[4 * q + u], lo[u]);
                atomicAdd(&total[4 * q + u], all[u]);
            }
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

// Tokens per workgroup of the first launch: as few 64s as keep the workgroups at 256, one per CU.  The second launch reads all their
// counts in each: 131072 tokens x 256 experts 70 us with 512 workgroups.
int64_t per_block(int64_t T) {
    return T <= TB ? TB : 64 * ((T + 64 * MAX_BLOCKS - 1) / (64 * MAX_BLOCKS));
}

template <int DT, int V>
int launch_pick(const RouteArgs& a, unsigned blocks, hipStream_t st) {
    if (a.bias) hipLaunchKernelGGL((moe_route_pick_kernel<DT, V, true>), dim3(blocks), dim3(pick_waves(V, true) * 64), sizeof(RouteLds), st, a);
    else hipLaunchKernelGGL((moe_route_pick_kernel<DT, V, false>), dim3(blocks), dim3(pick_waves(V, false) * 64), sizeof(RouteLds), st, a);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

template <int DT>
int launch_width(const RouteArgs& a, unsigned blocks, hipStream_t st) {
    if (a.E <= 32) return launch_pick<DT, 2>(a, blocks, st);
    if (a.E <= 64) return launch_pick<DT, 4>(a, blocks, st);
    if (a.E <= 128) return launch_pick<DT, 8>(a, blocks, st);
    if (a.E <= 256) return launch_pick<DT, 16>(a, blocks, st);
    return launch_pick<DT, 32>(a, blocks, st);
}

}  // namespace

extern "C" int64_t h3fp8_moe_route_workspace(int64_t T, int64_t E) {
    if (T <= TB || E < 0) return 0;
    return (T + per_block(T) - 1) / per_block(T) * ((E + 4) / 4 * 4) * 4;
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
                (uintptr_t)order | (uintptr_t)place) & 3) | ((uintptr_t)workspace & 15)) == 0, "h3fp8_moe_route: misaligned pointer");
    const int64_t need = h3fp8_moe_route_workspace(T, E);
    H3_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "h3fp8_moe_route: the workspace needs %lld bytes", (long long)need);
    RouteArgs a{};
    a.logits = logits; a.ld = ld; a.T = T; a.E = (int)E; a.k = k; a.renorm = renorm != 0; a.sigmoid = scoring; a.scale = scale;
    a.bias = bias; a.weights = weights; a.experts = experts; a.offsets = offsets; a.order = order; a.place = place;
    a.counts = need ? (int*)workspace : nullptr;
    a.per = (int)per_block(T);
    a.row = (int)(E + 4) / 4 * 4;
    a.vec = ((uintptr_t)logits & 15) == 0 && ld * elem % 16 == 0 && E * elem % 16 == 0;
    a.vec_bias = ((uintptr_t)bias & 15) == 0 && E % 4 == 0;
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
