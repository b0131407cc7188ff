// The FP8 product of block-scaled operands, dense and grouped by expert (gfx950).
//
//   y[m, n] = round(sum_b sa[m, b] * sw[n / 128, b] * P_b[m, n] (+ bias[n])),  P_b = sum over the 128 k of block b of
//   a[m, k] w[n, k];  grouped: row m of expert e (offsets[e] <= m < offsets[e + 1]) takes w[e], sw[e].
//
// One MFMA makes one P_b: v_mfma 16x16x128 on e4m3 from a zero accumulator, the weight rows as its A operand and the
// tokens as its B operand, so that lane l holds channels 4 (l >> 4) + r (r = 0 .. 3) of token l & 15 and the block's scale
// sa * sw is one number per lane: acc = fma(P_b, sa * sw, acc) in fp32, b ascending, and a zero sum is +0.  Every form below
// computes every element by this sequence, so all give the same bits.
#include "gemm_blocks_core.h"

namespace {

using namespace h3b;

template <class T, bool FP16, bool BIAS>
struct PlainStore {
    static constexpr bool REREAD = false;

    __device__ __forceinline__ void operator()(const BlocksParams& p, const TileRows& r, int tn, int wn, int wm, int lane,
                                               const v4f (&acc)[T::NI][T::NJ]) const {
        bstore<T, FP16, BIAS>(p, r, tn, wn, wm, lane, acc);
    }
};

template <class T, bool FP16, bool BIAS, bool GROUPED>
__global__ void __launch_bounds__(T::WAVES * 64, 2) gemm_blocks_tile_kernel(BlocksParams p) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[tile_lds<T, GROUPED>()];
    tile_kernel<T, GROUPED>(p, lds, PlainStore<T, FP16, BIAS>());
}

extern __shared__ __attribute__((aligned(1024))) uint8_t small_lds[];

template <class T, bool FP16, bool BIAS, bool GROUPED>
__global__ void __launch_bounds__(T::WAVES * 64) __attribute__((amdgpu_waves_per_eu(2))) gemm_blocks_small_kernel(BlocksParams p, int tiles_n, int rt) {
    small_kernel<T, GROUPED>(p, small_lds, tiles_n, rt, PlainStore<T, FP16, BIAS>());
}

template <class T, bool GROUPED>
int launch_tile(const BlocksParams& p, const char* who, hipStream_t st) {
    const int64_t tiles = row_tiles(p, T::TT) * ((p.N + T::TW - 1) / T::TW);
    H3_REQUIRE(tiles < ((int64_t)1 << 31), "%s: too many tiles for one launch", who);
    const dim3 grid((unsigned)std::min<int64_t>(tiles, h3host::cu_count())), block(T::WAVES * 64);
#define H3_B(FP16, BIAS) hipLaunchKernelGGL((gemm_blocks_tile_kernel<T, FP16, BIAS, GROUPED>), grid, block, 0, st, p)
    if constexpr (GROUPED) {                              // without a bias
        if (p.fp16) H3_B(true, false);
        else H3_B(false, false);
    } else if (p.fp16) {
        if (p.bias) H3_B(true, true);
        else H3_B(true, false);
    } else {
        if (p.bias) H3_B(false, true);
        else H3_B(false, false);
    }
#undef H3_B
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

template <class T, bool GROUPED>
int launch_small(const BlocksParams& p, const char* who, hipStream_t st) {
    const int64_t tiles_n = (p.N + T::TW - 1) / T::TW, rt = row_tiles(p, T::TT), tiles = rt * tiles_n;
    H3_REQUIRE(tiles < ((int64_t)1 << 32) / (T::WAVES * 64), "%s: too many tiles for one launch", who);      // 2^32 threads
    const dim3 grid((unsigned)tiles), block(T::WAVES * 64);
#define H3_B(FP16, BIAS) \
    hipLaunchKernelGGL((gemm_blocks_small_kernel<T, FP16, BIAS, GROUPED>), grid, block, T::LDS, st, p, (int)tiles_n, (int)rt)
    if constexpr (GROUPED) {
        if (p.fp16) H3_B(true, false);
        else H3_B(false, false);
    } else if (p.fp16) {
        if (p.bias) H3_B(true, true);
        else H3_B(true, false);
    } else {
        if (p.bias) H3_B(false, true);
        else H3_B(false, false);
    }
#undef H3_B
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

template <bool GROUPED>
int run(const BlocksParams& p, const char* who, hipStream_t st) {
    if (p.M == 0 || p.N == 0 || p.E == 0) return H3FP8_OK;
    const bool nt = streams(p);
    const int form = form_for(p.M, p.N, p.E, GROUPED, h3host::cu_count());
    switch (form) {
#define X(id, calls, per, ...)                                                                                         \
    case id:                                                                                                           \
        if constexpr (((calls) & (GROUPED ? EXPERTS : DENSE)) != 0) {                                                  \
            if constexpr (((calls) & EXPERTS) != 0)                                                                    \
                if (nt) return launch_small<SmallTile<__VA_ARGS__, true>, GROUPED>(p, who, st);                        \
            return launch_small<SmallTile<__VA_ARGS__>, GROUPED>(p, who, st);                                          \
        }                                                                                                              \
        break;
        H3_SMALL_FORMS(X)
#undef X
        case F_256x128:
            if constexpr (GROUPED)
                if (nt && once(p, 128)) return launch_tile<BigTile<2, 4, 8, 2, 3, true>, true>(p, who, st);
            return launch_tile<BigTile<2, 4, 8, 2, 3>, GROUPED>(p, who, st);
        case F_256x256:
            if constexpr (GROUPED)
                if (nt && once(p, 256)) return launch_tile<BigTile<2, 4, 8, 4, 2, true>, true>(p, who, st);
            return launch_tile<BigTile<2, 4, 8, 4, 2>, GROUPED>(p, who, st);
    }
    H3_REQUIRE(false, "%s: no kernel for form %d", who, form);
    return H3FP8_OK;
}

}  // namespace

namespace h3host {
// For the tests (host only): the tile, channels x tokens, that a call over M rows runs in on G CUs, and its place in the list of
// forms.
void gemm_blocks_plan(int64_t M, int64_t N, int64_t E, int grouped, int G, int* out) {
    const int f = form_for(M, N, E, grouped != 0, G);
    out[0] = kForms[f].tw;
    out[1] = kForms[f].tt;
    out[2] = f;
}
}  // namespace h3host

extern "C" {

int h3fp8_gemm_blocks(const void* a, int64_t lda, const void* w, int64_t ldw, const float* sa, int64_t sa_m, int64_t sa_k,
                      const float* sw, int64_t sw_n, int64_t sw_k, const void* bias, void* y, int64_t ldy, int out_dtype,
                      int64_t M, int64_t N, int64_t K, void* stream) {
    BlocksParams p{};
    p.a = (const uint8_t*)a; p.w = (const uint8_t*)w; p.sa = sa; p.sw = sw; p.bias = bias; p.y = (uint16_t*)y;
    p.lda = lda; p.ldw = ldw; p.ldy = ldy;
    p.sa_m = sa_m; p.sa_k = sa_k; p.sw_n = sw_n; p.sw_k = sw_k;
    p.M = M; p.N = (int)N; p.K = (int)K; p.E = 1; p.fp16 = out_dtype == H3FP8_DT_FP16;
    const int rc = check(p, "h3fp8_gemm_blocks", out_dtype, N, K, 1);
    return rc ? rc : run<false>(p, "h3fp8_gemm_blocks", (hipStream_t)stream);
}

int h3fp8_grouped_gemm_blocks(const void* a, int64_t lda, const void* w, int64_t w_e, int64_t ldw, const float* sa,
                              int64_t sa_m, int64_t sa_k, const float* sw, int64_t sw_e, int64_t sw_n, int64_t sw_k,
                              const void* offsets, int idx_bytes, void* y, int64_t ldy, int out_dtype, int64_t M, int64_t N,
                              int64_t K, int64_t E, void* stream) {
    BlocksParams p{};
    p.a = (const uint8_t*)a; p.w = (const uint8_t*)w; p.sa = sa; p.sw = sw; p.y = (uint16_t*)y;
    p.lda = lda; p.ldw = ldw; p.w_e = w_e; p.ldy = ldy;
    p.sa_m = sa_m; p.sa_k = sa_k; p.sw_e = sw_e; p.sw_n = sw_n; p.sw_k = sw_k;
    p.M = M; p.N = (int)N; p.K = (int)K; p.E = (int)E; p.fp16 = out_dtype == H3FP8_DT_FP16;
    p.offsets = offsets; p.idx_bytes = idx_bytes;
    const int rc = check(p, "h3fp8_grouped_gemm_blocks", out_dtype, N, K, E);
    if (rc) return rc;
    H3_REQUIRE(idx_bytes == 4 || idx_bytes == 8, "h3fp8_grouped_gemm_blocks: offsets must be int32 or int64");
    H3_REQUIRE(M == 0 || N == 0 || E == 0 || offsets, "h3fp8_grouped_gemm_blocks: null offsets");
    H3_REQUIRE((uintptr_t)offsets % (unsigned)idx_bytes == 0, "h3fp8_grouped_gemm_blocks: misaligned offsets");
    return run<true>(p, "h3fp8_grouped_gemm_blocks", (hipStream_t)stream);
}

}  // extern "C"
