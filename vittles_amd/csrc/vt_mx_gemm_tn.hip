// Gradient of a linear layer's weights from stored activations: C (Da, Db) = alpha A^T diag(rowscale) B + 1 bias^T with
// compact rows A (N, Da) and float, bfloat16 or half rows B (N, Db).  The long axis N is cut into slabs; a slab's sums
// are float and the slabs are added in a fixed order.
#include "vt_mx.h"

namespace {

typedef _Float16 f16;
typedef __bf16 bf16;

constexpr int kTile = 64, kDepth = 16;

struct MxTN {
    const uint8_t *codes, *scales;
    int64_t ldc, lds, N, rows;      // rows: of a slab
    int Da, Db;
    const void* B;
    int64_t ldb;
    const double* rowscale;
    float* part;                    // [slabs][Da][Db]
};

template <int FMT>
__device__ __forceinline__ float mx_at(const MxTN& a, int64_t n, int c) {
    const float s = mx_scale(a.scales[n * a.lds + (c >> 5)]);
    const unsigned b = a.codes[n * a.ldc + (FMT == VT_MX_FP8 ? c : c >> 1)];
    return mx_pair<FMT, 0>(FMT == VT_MX_FP4 && (c & 1) ? b >> 4 : b, s)[0];
}

template <int FMT, typename T>
__global__ __launch_bounds__(256) void k_mx_tn(MxTN a) {
    __shared__ float sa[kDepth][kTile], sb[kDepth][kTile];
    const int d0 = blockIdx.x * kTile, k0 = blockIdx.y * kTile, tid = threadIdx.x, ti = tid >> 4, tj = tid & 15;
    const int64_t n_lo = (int64_t)blockIdx.z * a.rows, n_hi = std::min(a.N, n_lo + a.rows);
    float acc[4][4] = {};
    for (int64_t n0 = n_lo; n0 < n_hi; n0 += kDepth) {
        for (int i = tid; i < kDepth * kTile; i += 256) {
            const int64_t n = n0 + i / kTile;
            const int c = i % kTile;
            sa[i / kTile][c] = n < n_hi && d0 + c < a.Da ? mx_at<FMT>(a, n, d0 + c) : 0.0f;
            float b = 0.0f;
            if (n < n_hi && k0 + c < a.Db) {
                b = (float)((const T*)a.B)[n * a.ldb + k0 + c];
                if (a.rowscale) b = (float)(a.rowscale[n] * (double)b);
            }
            sb[i / kTile][c] = b;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kDepth; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[r][4 * ti + i], sb[r][4 * tj + j], acc[i][j]);
        __syncthreads();
    }
    float* out = a.part + (int64_t)blockIdx.z * a.Da * a.Db;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (d0 + 4 * ti + i < a.Da && k0 + 4 * tj + j < a.Db) out[(int64_t)(d0 + 4 * ti + i) * a.Db + k0 + 4 * tj + j] = acc[i][j];
}

__global__ __launch_bounds__(256) void k_mx_tn_join(const float* part, int slabs, int Da, int Db, float alpha, const float* bias,
                                                    float* C, int64_t ldo) {
    const int64_t total = (int64_t)Da * Db;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        float s = 0.0f;
        for (int p = 0; p < slabs; ++p) s += part[p * total + i];
        const int64_t d = i / Db;
        const int k = (int)(i - d * Db);
        C[d * ldo + k] = alpha * s + (bias ? bias[k] : 0.0f);
    }
}

int slabs(int64_t N, int Da, int Db) {
    const int64_t tiles = (int64_t)((Da + kTile - 1) / kTile) * ((Db + kTile - 1) / kTile);
    const int64_t want = std::max<int64_t>(1, 2 * vt_num_cu() / tiles), most = std::max<int64_t>(1, N / 256);
    return (int)std::min(want, most);
}

template <int FMT>
int launch(int type, const MxTN& a, int s, hipStream_t st) {
    dim3 grid((a.Da + kTile - 1) / kTile, (a.Db + kTile - 1) / kTile, s);
    if (type == VT_TYPE_F32) hipLaunchKernelGGL((k_mx_tn<FMT, float>), grid, dim3(256), 0, st, a);
    else if (type == VT_TYPE_BF16) hipLaunchKernelGGL((k_mx_tn<FMT, bf16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_mx_tn<FMT, f16>), grid, dim3(256), 0, st, a);
    return vt_launch_status();
}

}  // namespace

extern "C" size_t vt_mx_gemm_tn_workspace_bytes(int64_t N, int Da, int Db) {
    if (N < 0 || Da < 1 || Db < 1) return 0;
    return (size_t)slabs(N, Da, Db) * Da * Db * sizeof(float);
}

extern "C" int vt_mx_gemm_tn(int format, const void* codes, int64_t ldc, const void* scales, int64_t lds, int Da, int type,
                             const void* B, int64_t ldb, int Db, const double* rowscale, int64_t N, float alpha,
                             const float* bias, float* C, int64_t ldo, void* ws, size_t ws_bytes, void* stream) {
    if (!mx_rows_ok(format, codes, ldc, scales, lds, N, Da) || Db < 1 || !C || ldo < Db) return VT_ERR_BAD_ARG;
    if (type < VT_TYPE_F32 || type > VT_TYPE_F16 || (N > 0 && (!B || ldb < Db))) return VT_ERR_BAD_ARG;
    if (!ws || ws_bytes < vt_mx_gemm_tn_workspace_bytes(N, Da, Db)) return VT_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    const int s = slabs(N, Da, Db);
    if ((Db + kTile - 1) / kTile > 65535) return VT_ERR_UNSUPPORTED;
    MxTN a{(const uint8_t*)codes, (const uint8_t*)scales, ldc, lds, N, (N + s - 1) / s, Da, Db, B, ldb, rowscale, (float*)ws};
    if (int rc = format == VT_MX_FP8 ? launch<VT_MX_FP8>(type, a, s, st) : launch<VT_MX_FP4>(type, a, s, st)) return rc;
    const int64_t total = (int64_t)Da * Db;
    hipLaunchKernelGGL(k_mx_tn_join, dim3((unsigned)std::min<int64_t>((total + 255) / 256, 8 * vt_num_cu())), dim3(256), 0, st,
                       a.part, s, Da, Db, alpha, bias, C, ldo);
    return vt_launch_status();
}
