// Product of 4-bit compact rows: C (M, N) = alpha A B^T + 1 bias^T on v_mfma_scale_f32_16x16x128_f8f6f4.
// Lane l of the instruction holds 32 codes of row (l & 15), block (l >> 4) of four: one compact block and its scale
// byte, so both operands go from memory to the matrix unit as they are stored.  E2M1 products times powers of two are
// exact and the sums are float (the E4M3 form of the instruction keeps only about 17 bits of a sum: 8-bit rows are not
// multiplied this way).
#include "vt_mx.h"

namespace {

struct MxNT {
    const uint8_t *ca, *sa, *cb, *sb;
    int64_t ldca, ldsa, ldcb, ldsb, M, N;
    int nb;                  // blocks of a row
    float alpha;
    const float* bias;
    void* C;
    int64_t ldc;
};

__device__ __forceinline__ i32x8 frag(const uint8_t* codes, int64_t ld, int64_t row, int kb, int nb) {
    i32x8 f = {0, 0, 0, 0, 0, 0, 0, 0};
    if (kb < nb) {
        const u32x4 w = *(const u32x4*)(codes + row * ld + (int64_t)kb * 16);
        f[0] = w[0], f[1] = w[1], f[2] = w[2], f[3] = w[3];
    }
    return f;
}
__device__ __forceinline__ int frag_scale(const uint8_t* scales, int64_t ld, int64_t row, int kb, int nb) {
    return kb < nb ? scales[row * ld + kb] : 127;
}

template <typename OutT>
__device__ __forceinline__ void mx_store(const MxNT& a, int64_t m, int64_t n, float v) {
    if (m < a.M && n < a.N) ((OutT*)a.C)[m * a.ldc + n] = (OutT)(a.alpha * v + (a.bias ? a.bias[n] : 0.0f));
}

// One wave a 32 x 32 tile of C, four waves a workgroup along N.
template <typename OutT>
__global__ __launch_bounds__(256) void k_mx_nt(MxNT a) {
    const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
    const int64_t m0 = (int64_t)blockIdx.y * 32, n0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 32;
    if (n0 >= a.N) return;
    f32x4 acc[2][2] = {};
    for (int kb0 = 0; kb0 < a.nb; kb0 += 4) {
        i32x8 fa[2], fb[2];
        int sa[2], sb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t ra = std::min<int64_t>(m0 + 16 * i + l, a.M - 1), rb = std::min<int64_t>(n0 + 16 * i + l, a.N - 1);
            fa[i] = frag(a.ca, a.ldca, ra, kb0 + q, a.nb);
            fb[i] = frag(a.cb, a.ldcb, rb, kb0 + q, a.nb);
            sa[i] = frag_scale(a.sa, a.ldsa, ra, kb0 + q, a.nb);
            sb[i] = frag_scale(a.sb, a.ldsb, rb, kb0 + q, a.nb);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fa[i], fb[j], acc[i][j], 4, 4, 0, sa[i], 0, sb[j]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx_store<OutT>(a, m0 + 16 * i + 4 * q + e, n0 + 16 * j + l, acc[i][j][e]);
}

}  // namespace

extern "C" size_t vt_mx_gemm_nt_workspace_bytes(int64_t M, int64_t N, int K) { return 0; }

extern "C" int vt_mx_gemm_nt(const void* ca, int64_t ldca, const void* sa, int64_t ldsa, int64_t M, const void* cb,
                             int64_t ldcb, const void* sb, int64_t ldsb, int64_t N, int K, float alpha, const float* bias,
                             int out_type, void* C, int64_t ldc, void* ws, size_t ws_bytes, void* stream) {
    if (!mx_rows_ok(VT_MX_FP4, ca, ldca, sa, ldsa, M, K) || !mx_rows_ok(VT_MX_FP4, cb, ldcb, sb, ldsb, N, K))
        return VT_ERR_BAD_ARG;
    if (out_type != VT_TYPE_F32 && out_type != VT_TYPE_BF16) return VT_ERR_BAD_ARG;
    if (M == 0 || N == 0) return VT_OK;
    if (!C || ldc < N) return VT_ERR_BAD_ARG;
    const int64_t gm = (M + 31) / 32, gn = (N + 127) / 128;
    if (gm > 65535 || gn > 0x7fffffff) return VT_ERR_UNSUPPORTED;
    MxNT a{(const uint8_t*)ca, (const uint8_t*)sa, (const uint8_t*)cb, (const uint8_t*)sb, ldca, ldsa, ldcb, ldsb, M, N,
           mx_blocks(K), alpha, bias, C, ldc};
    dim3 grid((unsigned)gn, (unsigned)gm);
    if (out_type == VT_TYPE_F32) hipLaunchKernelGGL(k_mx_nt<float>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(k_mx_nt<__bf16>, grid, dim3(256), 0, (hipStream_t)stream, a);
    return vt_launch_status();
}
