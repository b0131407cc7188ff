// RMSNorm of queries and keys per head with the position rotation in the same pass (gfx950).
//
// Per token t and head, x of D dims (D = 64, 128 or 256), R of them rotated (half = R / 2 pairs):
//   n_d = x_d / sqrt(sum x^2 / D + eps) * w_d                                    (fp32)
//   half-split:   pair p = dims (p, p + half);   interleaved: pair p = dims (2p, 2p + 1)
//   (a, b) -> (a cos_p - b sin_p, b cos_p + a sin_p), cos | sin = table[pos], pos = positions[t] or t
// rounded once to the input's type: unlike the fused consumer of the two-pass product (consumers.hip), which reproduces a
// stock kernel that rounds n to bf16 before it rotates.
//
// HBM-bound: every head is read and written once.  A lane holds 8 consecutive dims (16-byte loads and stores), D / 8 lanes
// a head, so a wave holds 512 / D heads of one token at a time (a pass), all of them q's or all of them k's, UNROLL passes'
// loads in flight together.  cos and sin of the lane's dims are loaded once and take up the norm weights (the partner's for sin),
// so that a dim costs one fma and three products.  The sum of squares goes over the head's lanes by DPP.  The half-split partner
// of dim d is half = R / 2 away, a multiple of 8, so it is in another lane at the same place: the lanes exchange their packed
// inputs (4 words instead of 8 normalised values); the interleaved partner is in the lane.  With few tokens a token's passes
// are dealt over several waves, until every SIMD has two.
// 18 880 tokens x (56 + 56) heads of 128, bf16: 197 us, 5.5 TB/s (two passes in flight 200, eight 192, but 4000 tokens x (32 + 8)
// heads 17.1 / 16.8 / 18.0; with q's and k's heads in one wave, the addresses and weights selected lane by lane, 209 and 22.1);
// 8 tokens x (32 + 8) heads 5.3-5.8 us a call, 3.3 of them on the GPU.  In one run, 18 880 tokens: (56 + 56) heads of 128 half-split
// 202 us, interleaved 201; (56 + 56) of 64 97 either way (5.6 TB/s); (28 + 28) of 256 203 and 202.
#include <algorithm>

#include "h3fp8_common.h"

namespace {

using namespace h3;

struct QkRopeArgs {
    const uint16_t* q;
    const uint16_t* k;
    int64_t q_t, q_h, k_t, k_h;                 // strides (elements) of tokens and heads
    uint16_t* oq;
    uint16_t* ok;
    int64_t oq_t, oq_h, ok_t, ok_h;
    const uint16_t* wq;
    const uint16_t* wk;
    const void* table;                          // [P, R]: cos of the half pairs, then sin
    int64_t ld_table;
    const void* positions;                      // null: the token's own number
    int64_t pos_stride;
    int pos_bytes;
    int64_t P;
    int64_t T;
    int H, Hk, half;
    float eps;
    int vec;                                    // the table entries of a lane are aligned for vector loads
    int per;                                    // passes (512 / D heads each) a wave takes
    int q_chunks, k_chunks;                     // waves per token, for q's heads and for k's
};

template <bool FP16>
__device__ __forceinline__ void widen8(v4u v, float f[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = FP16 ? fp16_to_f32(v[i] & 0xffffu) : u2f(v[i] << 16);
        f[2 * i + 1] = FP16 ? fp16_to_f32(v[i] >> 16) : u2f(v[i] & 0xffff0000u);
    }
}

template <bool FP16>
__device__ __forceinline__ v4u narrow8(const float f[8]) {
    v4u v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = FP16 ? fp16_rne(f[2 * i]) | (fp16_rne(f[2 * i + 1]) << 16) : cvt_bf16x2(f[2 * i], f[2 * i + 1]);
    return v;
}

// Entries p .. p + N - 1 of a table row; VEC: 16-byte aligned there.
template <bool TF32, bool VEC, int N>
__device__ __forceinline__ void table_read(const char* row, int p, float f[N]) {
    if (VEC) {
        if (TF32) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const v4f v = *reinterpret_cast<const v4f*>(row + 4 * (p + i));
#pragma unroll
                for (int e = 0; e < 4; ++e) f[i + e] = v[e];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const uint2 v = *reinterpret_cast<const uint2*>(row + 2 * (p + i));
                f[i] = u2f(v.x << 16); f[i + 1] = u2f(v.x & 0xffff0000u); f[i + 2] = u2f(v.y << 16); f[i + 3] = u2f(v.y & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            f[i] = TF32 ? reinterpret_cast<const float*>(row)[p + i] : bf16_to_f32(reinterpret_cast<const uint16_t*>(row)[p + i]);
    }
}

// The sum over a head's LPH lanes.
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
    v += u2f((uint32_t)__builtin_amdgcn_mov_dpp((int)f2u(v), 0xb1, 0xf, 0xf, true));     // lane ^ 1
    v += u2f((uint32_t)__builtin_amdgcn_mov_dpp((int)f2u(v), 0x4e, 0xf, 0xf, true));     // lane ^ 2
    v += u2f((uint32_t)__builtin_amdgcn_mov_dpp((int)f2u(v), 0x141, 0xf, 0xf, true));    // the other four of a half row
    if (LPH >= 16) v += u2f((uint32_t)__builtin_amdgcn_mov_dpp((int)f2u(v), 0x140, 0xf, 0xf, true));   // the other half row
    if (LPH >= 32) v += __shfl_xor(v, 16, 64);
    return v;
}

// 1 / sqrt(v) by the hardware's rsq (1 ulp), which takes subnormal numbers for zero: those are scaled by 2^64 first.
__device__ __forceinline__ float rsqrt32(float v) {
    const bool tiny = v < 0x1p-100f;
    return __builtin_amdgcn_rsqf(tiny ? v * 0x1p64f : v) * (tiny ? 0x1p32f : 1.0f);
}

// A uniform value, in a scalar register from here on.
template <class V>
__device__ __forceinline__ V pinned(V v) {
    asm("" : "+s"(v));
    return v;
}

typedef v4u __attribute__((address_space(1))) GlobalV4;

constexpr int UNROLL = 4;

template <int D, bool FP16, bool TF32, bool INTER>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(QkRopeArgs a) {
    constexpr int LPH = D / 8, HPW = 64 / LPH;              // lanes per head, heads per pass
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const uint32_t unit = blockIdx.x * 4 + wave, chunks = (uint32_t)(a.q_chunks + a.k_chunks), token = unit / chunks;
    if (token >= a.T) return;
    const int64_t t = token;
    const int chunk = (int)(unit - token * chunks);
    const bool isq = chunk < a.q_chunks;                    // the wave's heads: some of q's or some of k's
    const int j = lane % LPH, sub = lane / LPH;             // the lane's 8 dims 8j .. 8j + 7 of head `sub` of a pass
    const int heads = isq ? a.H : a.Hk;
    const int pass0 = (isq ? chunk : chunk - a.q_chunks) * a.per, passes = min(pass0 + a.per, (heads + HPW - 1) / HPW);
    // its byte strides and addresses, those of head 0 of a pass; in scalar registers, not behind a pointer that is selected
    const int64_t ih = pinned(2 * (isq ? a.q_h : a.k_h)), oh = pinned(2 * (isq ? a.oq_h : a.ok_h));
    const int64_t in0 = pinned((int64_t)(uintptr_t)(isq ? a.q + t * a.q_t : a.k + t * a.k_t));
    const int64_t out0 = pinned((int64_t)(uintptr_t)(isq ? a.oq + t * a.oq_t : a.ok + t * a.ok_t));
    const int64_t in_lane = sub * ih + 16 * j, out_lane = sub * oh + 16 * j;
    const int half = a.half;
    const bool rotated = 8 * j < 2 * half;                  // half-split: half % 8 == 0, a lane is wholly in or out
    const int pj = INTER || !rotated ? j : 8 * j < half ? j + half / 8 : j - half / 8;     // the partner lane of the head
    auto load = [&](int ps) {
        const bool live = ps < passes && ps * HPW + sub < heads;
        return live ? __builtin_nontemporal_load((const GlobalV4*)(in0 + ps * (HPW * ih) + in_lane)) : v4u{0u, 0u, 0u, 0u};
    };
    int64_t pos = t;
    if (a.positions)
        pos = a.pos_bytes == 8 ? reinterpret_cast<const int64_t*>(a.positions)[t * a.pos_stride]
                               : (int64_t)reinterpret_cast<const int32_t*>(a.positions)[t * a.pos_stride];
    v4u v[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) v[i] = load(pass0 + i);
    // out_d = n_d cos + (the partner's n) sin with a sign, n = x r w: cs and sn take the weights of the dim and of its partner
    float cs[8], sn[8], g[8], pg[8];
    const uint16_t* w = isq ? a.wq : a.wk;
    widen8<FP16>(*reinterpret_cast<const v4u*>(w + 8 * j), g);
    if (INTER) {
#pragma unroll
        for (int e = 0; e < 8; ++e) pg[e] = g[e ^ 1];
    } else {
        widen8<FP16>(*reinterpret_cast<const v4u*>(w + 8 * pj), pg);
    }
    const bool known = pos >= 0 && pos < a.P;               // else the outputs are NaN and the table is not read
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e] = known ? 1.0f : __builtin_nanf(""), sn[e] = 0.0f;
    if (known && rotated) {
        const char* row = reinterpret_cast<const char*>(a.table) + pos * a.ld_table * (TF32 ? 4 : 2);
        if (INTER) {
            float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
            if (a.vec) {
                table_read<TF32, true, 4>(row, 4 * j, c);
                table_read<TF32, true, 4>(row, half + 4 * j, s);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (4 * j + e < half) {
                        table_read<TF32, false, 1>(row, 4 * j + e, c + e);
                        table_read<TF32, false, 1>(row, half + 4 * j + e, s + e);
                    }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) cs[e] = c[e >> 1], sn[e] = (e & 1) ? s[e >> 1] : -s[e >> 1];
        } else {
            const int p = 8 * j < half ? 8 * j : 8 * j - half;
            if (a.vec) {
                table_read<TF32, true, 8>(row, p, cs);
                table_read<TF32, true, 8>(row, half + p, sn);
            } else {
                table_read<TF32, false, 8>(row, p, cs);
                table_read<TF32, false, 8>(row, half + p, sn);
            }
            if (8 * j < half) {
#pragma unroll
                for (int e = 0; e < 8; ++e) sn[e] = -sn[e];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e] *= g[e], sn[e] = rotated ? sn[e] * pg[e] : 0.0f;
    for (int ps = pass0; ps < passes; ps += UNROLL) {
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) {
            if (ps + i >= passes) break;                    // uniform
            float x[8], p[8], y[8];
            widen8<FP16>(v[i], x);
            if (!INTER) {                                   // a lane past the rotated dims has itself as its partner, and sin 0
                v4u o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = (uint32_t)__shfl((int)v[i][e], lane - j + pj, 64);
                widen8<FP16>(o, p);
            }
            v[i] = load(ps + UNROLL + i);
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(x[e], x[e], ss);
            const float r = rsqrt32(__builtin_fmaf(head_sum<LPH>(ss), 1.0f / D, a.eps));
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= r;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                p[e] = INTER ? (8 * j + e < 2 * half ? x[e ^ 1] : 0.0f) : p[e] * r;
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = __builtin_fmaf(x[e], cs[e], p[e] * sn[e]);
            if ((ps + i) * HPW + sub < heads)
                __builtin_nontemporal_store(narrow8<FP16>(y), (GlobalV4*)(out0 + (ps + i) * (HPW * oh) + out_lane));
        }
    }
}

template <int D, bool FP16, bool TF32>
int launch_qk(const QkRopeArgs& a, bool interleaved, dim3 grid, hipStream_t st) {
    if (interleaved) hipLaunchKernelGGL((qk_norm_rope_kernel<D, FP16, TF32, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((qk_norm_rope_kernel<D, FP16, TF32, false>), grid, dim3(256), 0, st, a);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

template <int D>
int launch_head(QkRopeArgs a, bool fp16, bool tf32, bool interleaved, hipStream_t st) {
    constexpr int HPW = 512 / D;
    const int pq = (a.H + HPW - 1) / HPW, pk = (a.Hk + HPW - 1) / HPW;
    // two waves per SIMD while there are passes to deal, then all of q's or k's heads of a token
    const int64_t waves = 8LL * h3host::cu_count();
    a.per = (int)std::max<int64_t>(1, std::min<int64_t>(std::max(pq, pk), a.T * (pq + pk) / waves));
    a.q_chunks = (pq + a.per - 1) / a.per;
    a.k_chunks = (pk + a.per - 1) / a.per;
    const int64_t units = a.T * (a.q_chunks + a.k_chunks);
    H3_REQUIRE(units <= ((int64_t)1 << 26) - 4, "h3fp8_qk_norm_rope: too many tokens for one launch");   // 2^32 threads
    const dim3 grid((unsigned)((units + 3) / 4));
    if (fp16) return tf32 ? launch_qk<D, true, true>(a, interleaved, grid, st) : launch_qk<D, true, false>(a, interleaved, grid, st);
    return tf32 ? launch_qk<D, false, true>(a, interleaved, grid, st) : launch_qk<D, false, false>(a, interleaved, grid, st);
}

bool rows_ok(const void* p, int64_t st_t, int64_t st_h) {
    return ((uintptr_t)p & 15) == 0 && st_t >= 0 && st_h >= 0 && st_t % 8 == 0 && st_h % 8 == 0;
}

}  // namespace

extern "C" int h3fp8_qk_norm_rope(const void* q, int64_t q_t, int64_t q_h, const void* k, int64_t k_t, int64_t k_h, int dtype,
                                  int64_t T, int H, int Hk, int D, const void* q_weight, const void* k_weight,
                                  const void* table, int64_t ld_table, int table_dtype, int64_t P, int R, int interleaved,
                                  const void* positions, int64_t pos_stride, int pos_bytes, float eps, void* out_q,
                                  int64_t oq_t, int64_t oq_h, void* out_k, int64_t ok_t, int64_t ok_h, void* stream) {
    H3_REQUIRE(T >= 0 && H >= 0 && Hk >= 0 && P >= 0, "h3fp8_qk_norm_rope: negative size");
    H3_REQUIRE(D == 64 || D == 128 || D == 256, "h3fp8_qk_norm_rope: head size %d (64, 128 or 256)", D);
    H3_REQUIRE(R >= 0 && R <= D && R % (interleaved ? 2 : 16) == 0,
               "h3fp8_qk_norm_rope: %d rotated dims of %d (half-split: a multiple of 16, interleaved: of 2)", R, D);
    H3_REQUIRE(dtype == H3FP8_DT_BF16 || dtype == H3FP8_DT_FP16, "h3fp8_qk_norm_rope: bad dtype %d", dtype);
    H3_REQUIRE(table_dtype == H3FP8_DT_BF16 || table_dtype == H3FP8_DT_F32, "h3fp8_qk_norm_rope: the table is fp32 or bf16");
    if (T == 0 || (int64_t)H + Hk == 0) return H3FP8_OK;
    H3_REQUIRE(H <= (1 << 20) && Hk <= (1 << 20), "h3fp8_qk_norm_rope: too many heads");
    H3_REQUIRE((H == 0 || (q && out_q && q_weight)) && (Hk == 0 || (k && out_k && k_weight)) && (R == 0 || table),
               "h3fp8_qk_norm_rope: null pointer");
    H3_REQUIRE((H == 0 || (rows_ok(q, q_t, q_h) && rows_ok(out_q, oq_t, oq_h) && ((uintptr_t)q_weight & 15) == 0)) &&
                   (Hk == 0 || (rows_ok(k, k_t, k_h) && rows_ok(out_k, ok_t, ok_h) && ((uintptr_t)k_weight & 15) == 0)),
               "h3fp8_qk_norm_rope: q, k, their outputs and the weights need 16-byte alignment and token and head strides "
               "that are multiples of 8 elements");
    H3_REQUIRE(R == 0 || (ld_table >= R && ((uintptr_t)table & (table_dtype == H3FP8_DT_F32 ? 3 : 1)) == 0),
               "h3fp8_qk_norm_rope: the table's row stride must be >= %d", R);
    H3_REQUIRE(positions ? pos_bytes == 4 || pos_bytes == 8 : P >= T || R == 0,
               "h3fp8_qk_norm_rope: positions must be int32 or int64, and without them the table needs a row per token");
    QkRopeArgs a{};
    a.q = (const uint16_t*)q; a.q_t = q_t; a.q_h = q_h;
    a.k = (const uint16_t*)k; a.k_t = k_t; a.k_h = k_h;
    a.oq = (uint16_t*)out_q; a.oq_t = oq_t; a.oq_h = oq_h;
    a.ok = (uint16_t*)out_k; a.ok_t = ok_t; a.ok_h = ok_h;
    a.wq = (const uint16_t*)q_weight; a.wk = (const uint16_t*)k_weight;
    a.table = table; a.ld_table = ld_table; a.P = R ? P : T;
    a.positions = R ? positions : nullptr; a.pos_stride = pos_stride; a.pos_bytes = pos_bytes;
    a.T = T; a.H = H; a.Hk = Hk; a.half = R / 2; a.eps = eps;
    const int need = table_dtype == H3FP8_DT_F32 ? 16 : 8;      // bytes of four entries
    a.vec = R % 8 == 0 && ld_table % 4 == 0 && ((uintptr_t)table & (need - 1)) == 0;
    const bool fp16 = dtype == H3FP8_DT_FP16, tf32 = table_dtype == H3FP8_DT_F32;
    hipStream_t st = (hipStream_t)stream;
    if (D == 64) return launch_head<64>(a, fp16, tf32, interleaved != 0, st);
    if (D == 128) return launch_head<128>(a, fp16, tf32, interleaved != 0, st);
    return launch_head<256>(a, fp16, tf32, interleaved != 0, st);
}
