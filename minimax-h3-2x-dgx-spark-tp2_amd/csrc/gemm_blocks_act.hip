// The block-scaled FP8 product with bias, activation and residual in its epilogue (gfx950).
//
//   y[m, n] = round(residual[m, n] + act(sum_b sa[m, b] sw[n / 128, b] P_b[m, n] + bias[n]))
//
// The sums are those of gemm_blocks.hip, by the same tiles and k-steps (gemm_blocks_core.h) and the same rule on sizes; the
// epilogue works on them in fp32 and rounds once.  What it saves is the passes behind the product, two bytes read and two
// written per element each.  A lane has 4 or 8 consecutive channels of a token, the piece that it stores: it reads the residual
// in the same piece, so that the output may be the residual itself.
//
// us, here / the product alone with a bias, calls back to back: 1 x 5376 -> 21 504, gelu_tanh 20 / 20.4; 200 x 7168 -> 5376 fp16 onto
// a residual 20.4 (weights from HBM 25 / 25; the kernel traced 22); 4100 x 5376 -> 14 336, gelu 309 to 312 / 287 to 291 (the first
// ten calls behind a pause, while the clock settles, 374; traced 329 then); 18 880 x 14 336 -> 5376 onto a residual 1250 to 1257 (in
// one launch 1322 to 1332) / 1270 to 1276.  What bounds it is the product (gemm_blocks_core.h); the epilogue of the 256 x 256 tiles
// stands between two tiles of its workgroup.  us on top of the product in one launch, bias alone or relu / silu / gelu_tanh / gelu /
// residual: 4100 x 5376 -> 14 336 6 / 11 / 16 / 22 / 28, 18 880 x 14 336 -> 5376 16 / 40 / 50 / 55 / 58, 18 880 x 5376 -> 14 336
// 30 / 70 / 90 / 116 / 118 (541 MB of residual).  Its registers are the k-steps' own: a value that only they used, kept in memory
// during them, was loaded again in every k-step and waited for all the loads under way (1400 us in place of 1295 with a bias
// alone).  The activation's branch is taken per piece: with one for the whole tile the compiler moves its 128 sums through memory
// (248 bytes a lane).
//
// The activations take the hardware's exponential and reciprocal (1 ulp each; the exponent's argument, up to 64 in size where
// the result counts, is rounded to 2^-18): relative errors below 2^-17, a 64th of the smallest rounding behind them.  sigmoid:
// gemm_core.h.
//   silu y sigmoid(y); gelu_tanh 0.5 y (1 + tanh u) = y sigmoid(2u), u = sqrt(2 / pi) (y + 0.044715 y^3)
//   gelu y Phi(y): with a = |y|, Q(a) = erfc(a / sqrt 2) / 2 = 2^(-a^2 log2 e / 2) p(1 / (1 + 0.36 a)), p of degree 7 without
//     a constant, fitted to Q's other factor by least squares with weights moved towards the largest relative error (1e-6 on
//     0 .. 14.5, past which the exponential ends it); y (1 - Q(a)), or y Q(a) for y < 0.
#include "gemm_blocks_core.h"

namespace {

using namespace h3b;

struct ActParams {
    const uint16_t* residual;   // [M, N] in the output's type, row stride ldr (0: one row for all), or null
    int64_t ldr;
    int act;                    // H3FP8_ACT_*
};

__device__ __forceinline__ float gelu_tanh(float y) {
    const float u = y * __builtin_fmaf(0.044715f * y, y, 1.0f);
    return times_sigmoid(y, 1.5957691216057308f * u);     // 2 sqrt(2 / pi)
}

__device__ __forceinline__ float gelu_erf(float y) {
    const float a = __builtin_fabsf(y), t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.36f, a, 1.0f));
    float p = 0.04678725197f;
    p = __builtin_fmaf(p, t, -0.17884233615f);
    p = __builtin_fmaf(p, t, 0.17969809820f);
    p = __builtin_fmaf(p, t, 0.02741329712f);
    p = __builtin_fmaf(p, t, 0.13940465450f);
    p = __builtin_fmaf(p, t, 0.14182958544f);
    p = __builtin_fmaf(p, t, 0.14370902344f);
    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(a * -0.5f * LOG2E, a, 64.0f));
    const bool neg = y < 0.0f;
    return y * __builtin_fmaf(p * t * e, neg ? 0x1p-64f : -0x1p-64f, neg ? 0.0f : 1.0f);
}

template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
    switch (act) {
        case H3FP8_ACT_SILU:
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = times_sigmoid(v[e], v[e]);
            break;
        case H3FP8_ACT_GELU:
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = gelu_erf(v[e]);
            break;
        case H3FP8_ACT_GELU_TANH:
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = gelu_tanh(v[e]);
            break;
        case H3FP8_ACT_RELU:
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = v[e] < 0.0f ? 0.0f : v[e];
            break;
    }
}

template <class T, bool FP16>
struct ActStore {
    static constexpr bool REREAD = true;
    ActParams a;

    __device__ __forceinline__ void operator()(const BlocksParams& p, const TileRows& r, int tn, int wn, int wm, int lane,
                                               const v4f (&acc)[T::NI][T::NJ]) const {
        constexpr int N = T::PAIRS ? 8 : 4, Q = T::NI * 4 / N;      // channels of a piece, pieces of a token
        typedef unsigned int Piece __attribute__((ext_vector_type(N / 2)));
        const int c = lane & 15, g = lane >> 4;
        const __amdgpu_buffer_rsrc_t yr = make_rsrc(p.y + r.row0 * p.ldy, (uint32_t)(((r.rows - 1) * p.ldy + p.N) * 2));
        // without a residual or a bias: a buffer of no bytes, which reads as zeros
        const __amdgpu_buffer_rsrc_t rr = make_rsrc(a.residual ? a.residual + r.row0 * a.ldr : nullptr,
                                                    a.residual ? (uint32_t)(((r.rows - 1) * a.ldr + p.N) * 2) : 0u);
        const __amdgpu_buffer_rsrc_t br = make_rsrc(p.bias, p.bias ? (uint32_t)p.N * 2u : 0u);
        const int n0 = tn * T::TW + wn * 16 * T::NI + N * g;
        const uint32_t row = (uint32_t)(wm * 16 * T::NJ + c);
        auto read = [](__amdgpu_buffer_rsrc_t b, uint32_t off) {
            if constexpr (N == 8) return __builtin_bit_cast(Piece, __builtin_amdgcn_raw_buffer_load_b128(b, (int)off, 0, 0));
            else return __builtin_bit_cast(Piece, __builtin_amdgcn_raw_buffer_load_b64(b, (int)off, 0, 0));
        };
        auto half = [](const Piece& v, int e) {           // value e of a piece
            const uint32_t u = v[e >> 1];
            return FP16 ? fp16_to_f32(e & 1 ? u >> 16 : u & 0xffffu) : u2f(e & 1 ? u & 0xffff0000u : u << 16);
        };
        Piece res[2][T::NJ], bias[2];                     // one piece ahead
        auto load = [&](int q) {
            const int n = n0 + 4 * N * q;
            const uint32_t col = n < p.N ? (uint32_t)n * 2u : OOB;
            bias[q & 1] = read(br, col);
            // with one row for all, its bytes are there for rows past the last too, whose stores are dropped
#pragma unroll
            for (int j = 0; j < T::NJ; ++j) res[q & 1][j] = read(rr, n < p.N ? (row + 16 * j) * (uint32_t)a.ldr * 2u + col : OOB);
        };
        load(0);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int n = n0 + 4 * N * q;
            const bool in = n < p.N;
            if (q + 1 < Q) load(q + 1);
#pragma unroll
            for (int j = 0; j < T::NJ; ++j) {
                float v[N];
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] = acc[N == 8 ? 2 * q + (e >> 2) : q][j][e & 3] + half(bias[q & 1], e);
                activate<N>(v, a.act);
                Piece o;
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const float lo = v[e] + half(res[q & 1][j], e), hi = v[e + 1] + half(res[q & 1][j], e + 1);
                    o[e >> 1] = FP16 ? fp16_rne(lo) | (fp16_rne(hi) << 16) : cvt_bf16x2(lo, hi);
                }
                const uint32_t off = in ? (row + 16 * j) * (uint32_t)p.ldy * 2u + (uint32_t)n * 2u : OOB;
                if constexpr (N == 8) __builtin_amdgcn_raw_buffer_store_b128(o, yr, (int)off, 0, 0);
                else __builtin_amdgcn_raw_buffer_store_b64(o, yr, (int)off, 0, 0);
            }
        }
    }
};

template <class T, bool FP16>
__global__ void __launch_bounds__(T::WAVES * 64, 2) gemm_blocks_act_tile_kernel(BlocksParams p, ActParams a) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[tile_lds<T, false>()];
    tile_kernel<T, false>(p, lds, ActStore<T, FP16>{a});
}

extern __shared__ __attribute__((aligned(1024))) uint8_t small_lds[];

template <class T, bool FP16>
__global__ void __launch_bounds__(T::WAVES * 64) __attribute__((amdgpu_waves_per_eu(2)))
gemm_blocks_act_small_kernel(BlocksParams p, int tiles_n, int rt, ActParams a) {
    small_kernel<T, false>(p, small_lds, tiles_n, rt, ActStore<T, FP16>{a});
}

template <class T>
int launch_tile(const BlocksParams& p, const ActParams& a, const char* who, hipStream_t st) {
    const int64_t tiles = row_tiles(p, T::TT) * ((p.N + T::TW - 1) / T::TW);
    H3_REQUIRE(tiles > 0 && tiles < ((int64_t)1 << 31), "%s: %lld tiles for one launch", who, (long long)tiles);
    const dim3 grid((unsigned)std::min<int64_t>(tiles, h3host::cu_count())), block(T::WAVES * 64);
    if (p.fp16) hipLaunchKernelGGL((gemm_blocks_act_tile_kernel<T, true>), grid, block, 0, st, p, a);
    else hipLaunchKernelGGL((gemm_blocks_act_tile_kernel<T, false>), grid, block, 0, st, p, a);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

template <class T>
int launch_small(const BlocksParams& p, const ActParams& a, const char* who, hipStream_t st) {
    const int64_t tiles_n = (p.N + T::TW - 1) / T::TW, rt = row_tiles(p, T::TT), tiles = rt * tiles_n;
    H3_REQUIRE(tiles > 0 && tiles < ((int64_t)1 << 32) / (T::WAVES * 64), "%s: %lld tiles for one launch", who,
               (long long)tiles);                         // 2^32 threads
    const dim3 grid((unsigned)tiles), block(T::WAVES * 64);
    if (p.fp16) hipLaunchKernelGGL((gemm_blocks_act_small_kernel<T, true>), grid, block, T::LDS, st, p, (int)tiles_n, (int)rt, a);
    else hipLaunchKernelGGL((gemm_blocks_act_small_kernel<T, false>), grid, block, T::LDS, st, p, (int)tiles_n, (int)rt, a);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

// The rows that fill whole rounds of 256 x 256 tiles on G CUs, where what is left is up to half a round: a launch of smaller tiles
// (the same sums) takes it in less than the round that it would cost.  us with a bias, in one launch / split, tiles left of 256 in
// brackets: 6200 x 5376 x 7168 263 / 212 (21), 12 500 x 5376 x 5376 354 / 327 (21), 18 880 x 5376 x 14 336 1289 / 1228 (21), 18 880 x
// 14 336 x 5376 1259 / 1254 (56), 3800 x 5376 x 7168 170 / 141 (63), 16 740 x 9216 x 3328 487 / 485 (72), 4200 x 5376 x 7168 170 / 158
// (105).
// Where none is left over (the tiles fill their rounds, the last row tile full or not) it is one launch of all M rows: tiles that
// are left are at least a row tile, so that rt * 256 < M.
int64_t whole_rounds(int64_t M, int64_t N, int G) {
    const int64_t cols = (N + 255) / 256, tiles = (M + 255) / 256 * cols, rt = tiles / G * G / cols, left = tiles - rt * cols;
    return rt > 0 && left > 0 && 2 * left <= G ? rt * 256 : M;
}

// Rows of the first launch.
int64_t first_rows(int64_t M, int64_t N, int G) { return dense_form(M, N, G) == F_256x256 ? whole_rounds(M, N, G) : M; }

int run_form(const BlocksParams& p, const ActParams& a, int form, const char* who, hipStream_t st) {
    const bool nt = streams(p);
    switch (form) {
#define X(id, calls, per, ...)                                                                                         \
    case id:                                                                                                           \
        if constexpr (((calls) & DENSE) != 0) {                                                                        \
            if constexpr (((calls) & EXPERTS) != 0)                                                                    \
                if (nt) return launch_small<SmallTile<__VA_ARGS__, true>>(p, a, who, st);                              \
            return launch_small<SmallTile<__VA_ARGS__>>(p, a, who, st);                                                \
        }                                                                                                              \
        break;
        H3_SMALL_FORMS(X)
#undef X
        case F_256x128: return launch_tile<BigTile<2, 4, 8, 2, 3>>(p, a, who, st);
        case F_256x256: return launch_tile<BigTile<2, 4, 8, 4, 2>>(p, a, who, st);
    }
    H3_REQUIRE(false, "%s: no kernel for form %d", who, form);
    return H3FP8_OK;
}

int run(const BlocksParams& p, const ActParams& a, const char* who, hipStream_t st) {
    if (p.M == 0 || p.N == 0) return H3FP8_OK;
    const int G = h3host::cu_count(), form = dense_form(p.M, p.N, G);
    const int64_t rows = first_rows(p.M, p.N, G);
    if (rows == p.M) return run_form(p, a, form, who, st);
    BlocksParams head = p, rest = p;
    ActParams b = a;
    head.M = rows;
    rest.M = p.M - rows;
    rest.a += rows * p.lda;
    rest.sa += rows * p.sa_m;
    rest.y += rows * p.ldy;
    if (a.residual) b.residual += rows * a.ldr;
    const int rc = run_form(head, a, form, who, st);
    return rc ? rc : run_form(rest, b, dense_form(rest.M, p.N, G), who, st);
}

}  // namespace

namespace h3host {
// For the tests (host only): the rows of a call's first launch on G CUs; the others are a second one's.
int64_t gemm_blocks_act_rows(int64_t M, int64_t N, int G) { return first_rows(M, N, G); }
}  // namespace h3host

extern "C" int h3fp8_gemm_blocks_act(const void* a, int64_t lda, const void* w, int64_t ldw, const float* sa, int64_t sa_m,
                                     int64_t sa_k, const float* sw, int64_t sw_n, int64_t sw_k, const void* bias, int act,
                                     const void* residual, int64_t ldr, void* y, int64_t ldy, int out_dtype, int64_t M, int64_t N,
                                     int64_t K, void* stream) {
    const char* who = "h3fp8_gemm_blocks_act";
    BlocksParams p{};
    p.a = (const uint8_t*)a; p.w = (const uint8_t*)w; p.sa = sa; p.sw = sw; p.bias = bias; p.y = (uint16_t*)y;
    p.lda = lda; p.ldw = ldw; p.ldy = ldy;
    p.sa_m = sa_m; p.sa_k = sa_k; p.sw_n = sw_n; p.sw_k = sw_k;
    p.M = M; p.N = (int)N; p.K = (int)K; p.E = 1; p.fp16 = out_dtype == H3FP8_DT_FP16;
    const int rc = check(p, who, out_dtype, N, K, 1);
    if (rc) return rc;
    H3_REQUIRE(act >= H3FP8_ACT_NONE && act <= H3FP8_ACT_RELU, "%s: bad activation %d", who, act);
    H3_REQUIRE(((uintptr_t)bias & 15) == 0, "%s: the bias must be 16-byte aligned", who);
    H3_REQUIRE(!residual || (((uintptr_t)residual & 15) == 0 && (ldr == 0 || ldr >= N) && ldr % 8 == 0 &&
                             256 * ldr * 2 + 2 * N <= kMaxSpan),
               "%s: the residual must be 16-byte aligned, its row stride 0 or >= N and a multiple of 8", who);
    return run(p, ActParams{(const uint16_t*)residual, residual ? ldr : 0, act}, who, (hipStream_t)stream);
}
