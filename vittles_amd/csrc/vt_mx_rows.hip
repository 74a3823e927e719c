// Row operators on compact rows: link, gradient, value, fused HVP, A v and A^T (u1 .* u2), with fp64 vectors and sums.
//     for every row n:  dot_n = x_n . v,  t_n = op(dot_n, per-row scalars) -> per-row outputs,  out += t_n x_n
// Two passes: one wave per row takes the dots and leaves t_n in the workspace; then every thread owns eight columns and
// walks a slab of rows.  Partial sums are combined in a fixed order (no atomics: the same bits every time).
#include "vt_mx.h"

namespace {

enum { OP_LINK, OP_GRAD, OP_VALUE, OP_HVP, OP_GEMV, OP_GEMVT };
template <int OP> constexpr bool kDot = OP != OP_GEMVT;
template <int OP> constexpr bool kCols = OP == OP_GRAD || OP == OP_HVP || OP == OP_GEMVT;

struct MxRows {
    const uint8_t* codes;
    const uint8_t* scales;
    int64_t ldc, lds, N;
    int D;
    const double *v;               // D-vector of the dot
    const double *y, *w, *offset;  // per-row inputs; GEMVT: y = u1, w = u2 (may be NULL); HVP: y = d
    double scale;
    int family;
    double *z, *r, *d;             // per-row outputs, each may be NULL
    double* t;                     // (N,) coefficients of the column pass; VALUE: the row's loss
    double* part;                  // [slabs][D]
};

// The row's coefficient in the column sum; writes the row's outputs.
template <int OP>
__device__ __forceinline__ double mx_row_op(const MxRows& a, int64_t n, double dot) {
    if constexpr (OP == OP_GEMVT) {
        return a.w ? a.y[n] * a.w[n] : a.y[n];
    } else if constexpr (OP == OP_HVP) {
        return a.y[n] * dot;
    } else if constexpr (OP == OP_GEMV) {
        a.z[n] = dot;
        return 0.0;
    } else {
        const double z = dot + (a.offset ? a.offset[n] : 0.0), w = a.w[n];
        if constexpr (OP == OP_VALUE) {
            return w * vt_loss(a.family, z, a.y[n]);
        } else {
            double l1, l2;
            vt_link(a.family, z, a.y[n], l1, l2);
            if (a.z) a.z[n] = z;
            if (a.r) a.r[n] = a.scale * l1;
            if (a.d) a.d[n] = a.scale * w * l2;
            return w * (a.scale * l1);
        }
    }
}

// Eight values of a row, columns 8 g .. 8 g + 7.
template <int FMT>
__device__ __forceinline__ void mx_load8(const MxRows& a, int64_t n, int g, float (&x)[8]) {
    const float s = mx_scale(a.scales[n * a.lds + (g >> 2)]);
    if constexpr (FMT == VT_MX_FP8) {
        const u32x2 w = *(const u32x2*)(a.codes + n * a.ldc + (int64_t)g * 8);
        float t[4];
        mx_word<FMT>(w[0], s, t);
        x[0] = t[0], x[1] = t[1], x[2] = t[2], x[3] = t[3];
        mx_word<FMT>(w[1], s, t);
        x[4] = t[0], x[5] = t[1], x[6] = t[2], x[7] = t[3];
    } else {
        mx_word<FMT>(*(const unsigned*)(a.codes + n * a.ldc + (int64_t)g * 4), s, x);
    }
}

template <int OP, int FMT>
__global__ __launch_bounds__(256) void k_mx_dots(MxRows a) {
    const int lane = threadIdx.x & 63;
    for (int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); n < a.N; n += (int64_t)gridDim.x * 4) {
        double dot = 0.0;
        if constexpr (kDot<OP>) {
            for (int g = lane; g * 8 < a.D; g += 64) {
                float x[8];
                mx_load8<FMT>(a, n, g, x);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (g * 8 + i < a.D) dot = fma((double)x[i], a.v[g * 8 + i], dot);
            }
            dot = vt_sum64(dot);
        }
        if (lane == 0) {
            const double t = mx_row_op<OP>(a, n, dot);
            if (a.t) a.t[n] = t;
        }
    }
}

template <int FMT>
__global__ __launch_bounds__(256) void k_mx_columns(MxRows a) {
    const int g = blockIdx.x * 256 + threadIdx.x;
    if (g * 8 >= a.D) return;
    double acc[8] = {};
    for (int64_t n = blockIdx.y; n < a.N; n += gridDim.y) {
        float x[8];
        mx_load8<FMT>(a, n, g, x);
        const double t = a.t[n];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = fma(t, (double)x[i], acc[i]);
    }
    double* out = a.part + (int64_t)blockIdx.y * a.D;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (g * 8 + i < a.D) out[g * 8 + i] = acc[i];
}

// out[c] = sum_p part[p][c] + beta[c] bvec[c], 32 columns a workgroup, 32 groups each summing every 32nd slab.
__global__ __launch_bounds__(1024) void k_mx_finalize(const double* part, int P, int D, const double* beta, const double* bvec,
                                                      double beta_scalar, double* out) {
    __shared__ double sh[32][33];
    const int cl = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + cl;
    double s = 0.0;
    if (c < D)
        for (int p = grp; p < P; p += 32) s += part[(int64_t)p * D + c];
    sh[grp][cl] = s;
    __syncthreads();
    if (grp == 0 && c < D) {
        double tot = 0.0;
#pragma unroll
        for (int q = 0; q < 32; ++q) tot += sh[q][cl];
        if (bvec) tot += (beta ? beta[c] : beta_scalar) * bvec[c];
        out[c] = tot;
    }
}

// value = scale * sum_n t_n, one workgroup.
__global__ __launch_bounds__(1024) void k_mx_sum(const double* t, int64_t N, double scale, double* out) {
    __shared__ double sh[16];
    double s = 0.0;
    for (int64_t n = threadIdx.x; n < N; n += 1024) s += t[n];
    s = vt_sum64(s);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double tot = 0.0;
        for (int i = 0; i < 16; ++i) tot += sh[i];
        out[0] = scale * tot;
    }
}

int col_tiles(int D) { return (D + 2047) / 2048; }
int64_t slabs(int64_t N, int D) { return std::max<int64_t>(1, std::min<int64_t>(N, std::max(1, 4 * vt_num_cu() / col_tiles(D)))); }

template <int OP, int FMT>
int run(MxRows a, int* nslabs, hipStream_t st) {
    const int grid = (int)std::min<int64_t>((a.N + 3) / 4, 8 * (int64_t)vt_num_cu());
    hipLaunchKernelGGL((k_mx_dots<OP, FMT>), dim3(grid), dim3(256), 0, st, a);
    if constexpr (kCols<OP>) {
        *nslabs = (int)slabs(a.N, a.D);
        hipLaunchKernelGGL((k_mx_columns<FMT>), dim3(col_tiles(a.D), *nslabs), dim3(256), 0, st, a);
    }
    return vt_launch_status();
}

template <int OP>
int run(int format, MxRows a, int* nslabs, hipStream_t st) {
    return format == VT_MX_FP8 ? run<OP, VT_MX_FP8>(a, nslabs, st) : run<OP, VT_MX_FP4>(a, nslabs, st);
}

int finalize(const double* part, int P, int D, const double* beta, const double* bvec, double beta_scalar, double* out,
             hipStream_t st) {
    hipLaunchKernelGGL(k_mx_finalize, dim3((D + 31) / 32), dim3(1024), 0, st, part, P, D, beta, bvec, beta_scalar, out);
    return vt_launch_status();
}

MxRows rows_of(const void* codes, int64_t ldc, const void* scales, int64_t lds, int64_t N, int D, void* ws) {
    MxRows a{};
    a.codes = (const uint8_t*)codes;
    a.scales = (const uint8_t*)scales;
    a.ldc = ldc, a.lds = lds, a.N = N, a.D = D;
    a.part = (double*)ws;
    a.t = a.part + slabs(N, D) * D;
    return a;
}

}  // namespace

extern "C" size_t vt_mx_rows_workspace_bytes(int64_t N, int D) {
    if (N < 0 || D < 1) return 0;
    return ((size_t)slabs(N, D) * D + (size_t)N) * sizeof(double);
}

#define VT_MX_ROWS_PROLOGUE                                                                  \
    if (!mx_rows_ok(format, codes, ldc, scales, lds, N, D)) return VT_ERR_BAD_ARG;           \
    if (!ws || ws_bytes < vt_mx_rows_workspace_bytes(N, D)) return VT_ERR_WORKSPACE;         \
    hipStream_t st = (hipStream_t)stream;                                                    \
    MxRows a = rows_of(codes, ldc, scales, lds, N, D, ws);

extern "C" int vt_mx_glm_link(int family, int format, const void* codes, int64_t ldc, const void* scales, int64_t lds,
                              const double* theta, const double* y, const double* w, const double* offset, double scale,
                              int64_t N, int D, double* z, double* r, double* d, void* ws, size_t ws_bytes, void* stream) {
    VT_MX_ROWS_PROLOGUE
    if (family < 0 || family > 2) return VT_ERR_BAD_ARG;
    if (N == 0) return VT_OK;
    if (!theta || !y || !w) return VT_ERR_BAD_ARG;
    a.v = theta, a.y = y, a.w = w, a.offset = offset, a.scale = scale, a.family = family;
    a.z = z, a.r = r, a.d = d, a.t = nullptr;
    return run<OP_LINK>(format, a, nullptr, st);
}

extern "C" int vt_mx_glm_grad(int family, int format, const void* codes, int64_t ldc, const void* scales, int64_t lds,
                              const double* theta, const double* y, const double* w, const double* offset, double scale,
                              const double* prior, int64_t N, int D, double* g, double* r, double* d, void* ws,
                              size_t ws_bytes, void* stream) {
    VT_MX_ROWS_PROLOGUE
    if (family < 0 || family > 2 || !theta || !g || (N > 0 && (!y || !w))) return VT_ERR_BAD_ARG;
    a.v = theta, a.y = y, a.w = w, a.offset = offset, a.scale = scale, a.family = family, a.r = r, a.d = d;
    int P = 0;
    if (N > 0)
        if (int rc = run<OP_GRAD>(format, a, &P, st)) return rc;
    return finalize(a.part, P, D, prior, prior ? theta : nullptr, 0.0, g, st);
}

extern "C" int vt_mx_glm_value(int family, int format, const void* codes, int64_t ldc, const void* scales, int64_t lds,
                               const double* theta, const double* y, const double* w, const double* offset, double scale,
                               int64_t N, int D, double* value, void* ws, size_t ws_bytes, void* stream) {
    VT_MX_ROWS_PROLOGUE
    if (family < 0 || family > 2 || !theta || !value || (N > 0 && (!y || !w))) return VT_ERR_BAD_ARG;
    a.v = theta, a.y = y, a.w = w, a.offset = offset, a.family = family;
    if (N > 0)
        if (int rc = run<OP_VALUE>(format, a, nullptr, st)) return rc;
    hipLaunchKernelGGL(k_mx_sum, dim3(1), dim3(1024), 0, st, a.t, N, scale, value);
    return vt_launch_status();
}

extern "C" int vt_mx_glm_hvp(int format, const void* codes, int64_t ldc, const void* scales, int64_t lds, const double* d,
                             const double* prior, double prior_scalar, const double* v, int64_t N, int D, double* out,
                             void* ws, size_t ws_bytes, void* stream) {
    VT_MX_ROWS_PROLOGUE
    if (!v || !out || (N > 0 && !d)) return VT_ERR_BAD_ARG;
    a.v = v, a.y = d;
    int P = 0;
    if (N > 0)
        if (int rc = run<OP_HVP>(format, a, &P, st)) return rc;
    return finalize(a.part, P, D, prior, prior || prior_scalar != 0.0 ? v : nullptr, prior_scalar, out, st);
}

extern "C" int vt_mx_gemv(int format, const void* codes, int64_t ldc, const void* scales, int64_t lds, const double* v,
                          int64_t N, int D, double* out, void* ws, size_t ws_bytes, void* stream) {
    VT_MX_ROWS_PROLOGUE
    if (N == 0) return VT_OK;
    if (!v || !out) return VT_ERR_BAD_ARG;
    a.v = v, a.z = out, a.t = nullptr;
    return run<OP_GEMV>(format, a, nullptr, st);
}

extern "C" int vt_mx_gemv_t(int format, const void* codes, int64_t ldc, const void* scales, int64_t lds, const double* u1,
                            const double* u2, int64_t N, int D, double* out, void* ws, size_t ws_bytes, void* stream) {
    VT_MX_ROWS_PROLOGUE
    if (!out || (N > 0 && !u1)) return VT_ERR_BAD_ARG;
    a.y = u1, a.w = u2;
    int P = 0;
    if (N > 0)
        if (int rc = run<OP_GEMVT>(format, a, &P, st)) return rc;
    return finalize(a.part, P, D, nullptr, nullptr, 0.0, out, st);
}
