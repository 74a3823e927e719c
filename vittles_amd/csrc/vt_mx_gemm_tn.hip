// Gradient of a linear layer's weights from stored activations: C (Da, Db) = alpha A^T diag(rowscale) B + 1 bias^T with
// compact rows A (N, Da) and float, bfloat16 or half rows B (N, Db), on v_mfma_f32_32x32x16_bf16.
// A code times its scale IS a bfloat16 (4 significant bits at most; v_cvt_scalef32_pk_bf16_fp8 / _fp4), so A enters the
// product exactly.  B is cut into bfloat16 parts that add up to it: one for bfloat16, two for half (11 bits), three for
// float (24 bits) and for anything times rowscale (rounded once to float).  Every product is exact; sums are float.
// Both operands are contracted along the rows, across which they lie in memory: a chunk of rows is staged as it lies and
// read with the transposing LDS read (ds_read_b64_tr_b16), 4 rows x 16 columns a quarter wave.
// The long axis N is cut into slabs; a slab's sums are float and the slabs are added in a fixed order.
#include "vt_mx.h"
#include <type_traits>

namespace {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

struct MxTN {
    const uint8_t *codes, *scales;
    int64_t ldc, lds, N, rows;      // rows: of a slab
    int Da, Db;
    const void* B;
    int64_t ldb;
    bool vec;                       // B's rows are 16-byte aligned
    const double* rowscale;
    float alpha;
    const float* bias;
    float* C;
    int64_t ldo;
    float* part;                    // [slabs][Da][Db], when there are several
};

// A workgroup of WM x WN waves, each MT x NT products of 32 x 32; kRows rows a chunk, two chunks in LDS.
template <int MT, int NT, int WM, int WN, int PARTS>
struct TnShape {
    static constexpr int kThreads = 64 * WM * WN, BM = 32 * MT * WM, BN = 32 * NT * WN, kRows = 32;
    // 64 bytes behind every row: the four rows of a transposing read lie in different banks
    static constexpr int kPitchA = 2 * BM + 64, kPitchB = 2 * BN + 64;
    static constexpr int kA = kRows * kPitchA, kB = kRows * kPitchB, kBuf = kA + PARTS * kB, kLds = 2 * kBuf;
    static constexpr int kLoadsA = kRows * BM / 8 / kThreads, kLoadsB = kRows * BN / 8 / kThreads;      // 8 columns each
    static_assert(kRows * BM / 8 % kThreads == 0 && kRows * BN / 8 % kThreads == 0, "even shares");
};

template <typename T, bool SCALED> constexpr int kParts = SCALED || std::is_same<T, float>::value ? 3 : std::is_same<T, f16>::value ? 2 : 1;

// x = parts[0] + parts[1] + ...: the leading 8 bits, the next 8, the rest.  An infinity or NaN is its first part alone.
template <int PARTS>
__device__ __forceinline__ void split(float x, unsigned (&p)[PARTS]) {
    unsigned u = __builtin_bit_cast(unsigned, x);
    p[0] = u >> 16;
    if constexpr (PARTS > 1) {
        const bool fine = (u & 0x7f800000u) != 0x7f800000u;
        if (x != x) p[0] |= 0x40u;          // a NaN whose payload lay in the bits that are cut stays one
#pragma unroll
        for (int i = 1; i < PARTS; ++i) {
            x = fine ? x - __builtin_bit_cast(float, u & 0xffff0000u) : 0.0f;
            u = __builtin_bit_cast(unsigned, x);
            p[i] = u >> 16;
        }
    }
}

__device__ __forceinline__ s16x8 read_tr(const uint8_t* p, int next4) {
    typedef __attribute__((address_space(3))) s16x4* ptr;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)p), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(p + next4));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <int FMT, typename T, bool SCALED, int MT, int NT, int WM, int WN, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_mx_tn(MxTN a) {
    constexpr int PARTS = kParts<T, SCALED>;
    using S = TnShape<MT, NT, WM, WN, PARTS>;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int d0 = blockIdx.x * S::BM, k0 = blockIdx.y * S::BN;
    const int64_t n_lo = (int64_t)blockIdx.z * a.rows, n_hi = std::min(a.N, n_lo + a.rows);
    const int width = mx_blocks(a.Da) * kMxBlock;

    u32x2 ca[S::kLoadsA];
    unsigned sc[S::kLoadsA];
    T cb[S::kLoadsB][8];
    double rs[S::kLoadsB];
    auto fetch = [&](int64_t n0) {
#pragma unroll
        for (int i = 0; i < S::kLoadsA; ++i) {
            const int e = tid + S::kThreads * i, c = d0 + e % (S::BM / 8) * 8;
            const int64_t n = n0 + e / (S::BM / 8);
            ca[i] = u32x2{0, 0};
            sc[i] = 127;
            if (n < n_hi && c < width) {
                if constexpr (FMT == VT_MX_FP8) ca[i] = *(const u32x2*)(a.codes + n * a.ldc + c);
                else ca[i][0] = *(const unsigned*)(a.codes + n * a.ldc + c / 2);
                sc[i] = a.scales[n * a.lds + c / kMxBlock];
            }
        }
#pragma unroll
        for (int i = 0; i < S::kLoadsB; ++i) {
            const int e = tid + S::kThreads * i, c = k0 + e % (S::BN / 8) * 8;
            const int64_t n = n0 + e / (S::BN / 8);
            const T* p = (const T*)a.B + n * a.ldb + c;
            if (n < n_hi && a.vec && c + 8 <= a.Db) {
                constexpr int W = (int)sizeof(T) / 2;
                u32x4 t[W];
#pragma unroll
                for (int j = 0; j < W; ++j) t[j] = ((const u32x4*)p)[j];
                __builtin_memcpy(cb[i], t, sizeof(t));
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) cb[i][j] = n < n_hi && c + j < a.Db ? p[j] : (T)0.0f;
            }
            if constexpr (SCALED) rs[i] = n < n_hi ? a.rowscale[n] : 0.0;
        }
    };
    auto put = [&](uint8_t* base) {
#pragma unroll
        for (int i = 0; i < S::kLoadsA; ++i) {
            const int e = tid + S::kThreads * i;
            const float s = mx_scale(sc[i]);
            bf16x2 v[4];
            if constexpr (FMT == VT_MX_FP8) {
                v[0] = mx_pair_bf16<FMT, 0>(ca[i][0], s), v[1] = mx_pair_bf16<FMT, 1>(ca[i][0], s);
                v[2] = mx_pair_bf16<FMT, 0>(ca[i][1], s), v[3] = mx_pair_bf16<FMT, 1>(ca[i][1], s);
            } else {
                v[0] = mx_pair_bf16<FMT, 0>(ca[i][0], s), v[1] = mx_pair_bf16<FMT, 1>(ca[i][0], s);
                v[2] = mx_pair_bf16<FMT, 2>(ca[i][0], s), v[3] = mx_pair_bf16<FMT, 3>(ca[i][0], s);
            }
            *(u32x4*)(base + e / (S::BM / 8) * S::kPitchA + e % (S::BM / 8) * 16) =
                u32x4{__builtin_bit_cast(unsigned, v[0]), __builtin_bit_cast(unsigned, v[1]), __builtin_bit_cast(unsigned, v[2]),
                      __builtin_bit_cast(unsigned, v[3])};
        }
#pragma unroll
        for (int i = 0; i < S::kLoadsB; ++i) {
            const int e = tid + S::kThreads * i;
            uint8_t* p = base + S::kA + e / (S::BN / 8) * S::kPitchB + e % (S::BN / 8) * 16;
            if constexpr (PARTS == 1) {
                u32x4 t;
                __builtin_memcpy(&t, cb[i], 16);
                *(u32x4*)p = t;
            } else {
                u32x4 w[PARTS];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    unsigned x[2][PARTS];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float b = (float)cb[i][2 * j + h];
                        if constexpr (SCALED) b = (float)(rs[i] * (double)b);
                        split<PARTS>(b, x[h]);
                    }
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) w[q][j] = x[0][q] | x[1][q] << 16;
                }
#pragma unroll
                for (int q = 0; q < PARTS; ++q) *(u32x4*)(p + q * S::kB) = w[q];
            }
        }
    };

    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    // a lane's part of a transposing read: row (lane % 16) / 4 of the quarter wave's four, columns 4 (lane % 4); the
    // quarters: columns 0 - 15 and 16 - 31 of rows 0 .., then of rows 8 ..
    const int qr = 8 * (lane >> 5) + (lane & 15) / 4, qc = 2 * (16 * (lane >> 4 & 1) + 4 * (lane & 3));
    const int oa = qr * S::kPitchA + qc + 2 * 32 * MT * wm, ob = S::kA + qr * S::kPitchB + qc + 2 * 32 * NT * wn;
    auto multiply = [&](const uint8_t* base) {
#pragma unroll
        for (int s = 0; s < S::kRows / 16; ++s) {
            s16x8 fa[MT], fb[PARTS][NT];
#pragma unroll
            for (int i = 0; i < MT; ++i) fa[i] = read_tr(base + oa + 16 * s * S::kPitchA + 64 * i, 4 * S::kPitchA);
#pragma unroll
            for (int q = 0; q < PARTS; ++q)
#pragma unroll
                for (int j = 0; j < NT; ++j) fb[q][j] = read_tr(base + ob + q * S::kB + 16 * s * S::kPitchB + 64 * j, 4 * S::kPitchB);
#pragma unroll
            for (int q = 0; q < PARTS; ++q)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fa[i]), __builtin_bit_cast(bf16x8, fb[q][j]),
                                                                           acc[i][j], 0, 0, 0);
        }
    };

    int buf = 0;
    if (n_lo < n_hi) {
        fetch(n_lo);
        put(lds);
    }
    for (int64_t n0 = n_lo; n0 < n_hi; n0 += S::kRows, buf ^= 1) {
        const bool more = n0 + S::kRows < n_hi;
        vt_lds_barrier();           // the chunk is written, and the other place is read
        if (more) fetch(n0 + S::kRows);
        multiply(lds + buf * S::kBuf);
        if (more) put(lds + (buf ^ 1) * S::kBuf);
    }

    // lane, element e of a 32 x 32 result: row 8 (e / 4) + 4 (lane / 32) + e % 4, column lane % 32
    const int l = lane & 31, h = lane >> 5;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int k = k0 + 32 * (wn * NT + j) + l;
            if (k < a.Db) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int d = d0 + 32 * (wm * MT + i) + 8 * (e / 4) + 4 * h + e % 4;
                    if (d < a.Da) {
                        if constexpr (SPLIT) a.part[((int64_t)blockIdx.z * a.Da + d) * a.Db + k] = acc[i][j][e];
                        else a.C[(int64_t)d * a.ldo + k] = a.alpha * acc[i][j][e] + (a.bias ? a.bias[k] : 0.0f);
                    }
                }
            }
        }
}

__global__ __launch_bounds__(256) void k_mx_tn_join(MxTN a, int slabs) {
    const int64_t total = (int64_t)a.Da * a.Db;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        float s = 0.0f;
        for (int p = 0; p < slabs; ++p) s += a.part[p * total + i];
        const int64_t d = i / a.Db;
        const int k = (int)(i - d * a.Db);
        a.C[d * a.ldo + k] = a.alpha * s + (a.bias ? a.bias[k] : 0.0f);
    }
}

struct TnPlan {
    int bm, bn, slabs;
    int64_t rows;
};

TnPlan plan(int64_t N, int Da, int Db) {
    TnPlan p;
    if (Db > 64) p.bm = 256, p.bn = 128;
    else p.bm = 128, p.bn = 64;
    const int64_t tiles = (int64_t)((Da + p.bm - 1) / p.bm) * ((Db + p.bn - 1) / p.bn);
    const int64_t want = std::max<int64_t>(1, 2 * vt_num_cu() / tiles), most = std::max<int64_t>(1, N / 128);
    p.slabs = (int)std::min(want, most);
    p.rows = (std::max<int64_t>(1, (N + p.slabs - 1) / p.slabs) + 31) / 32 * 32;
    p.slabs = (int)std::max<int64_t>(1, (N + p.rows - 1) / p.rows);
    return p;
}

template <int FMT, typename T, bool SCALED, int MT, int NT, int WM, int WN>
int launch(const MxTN& a, const TnPlan& p, hipStream_t st) {
    using S = TnShape<MT, NT, WM, WN, kParts<T, SCALED>>;
    const dim3 grid((a.Da + S::BM - 1) / S::BM, (a.Db + S::BN - 1) / S::BN, p.slabs);
    static VtLdsAttr attr_split, attr_whole;
    if (p.slabs > 1) {
        if (vt_allow_big_lds((const void*)k_mx_tn<FMT, T, SCALED, MT, NT, WM, WN, true>, attr_split, S::kLds) != VT_OK) return VT_ERR_HIP;
        hipLaunchKernelGGL((k_mx_tn<FMT, T, SCALED, MT, NT, WM, WN, true>), grid, dim3(S::kThreads), S::kLds, st, a);
        const int64_t total = (int64_t)a.Da * a.Db;
        hipLaunchKernelGGL(k_mx_tn_join, dim3((unsigned)std::min<int64_t>((total + 255) / 256, 8 * vt_num_cu())), dim3(256), 0, st, a, p.slabs);
    } else {
        if (vt_allow_big_lds((const void*)k_mx_tn<FMT, T, SCALED, MT, NT, WM, WN, false>, attr_whole, S::kLds) != VT_OK) return VT_ERR_HIP;
        hipLaunchKernelGGL((k_mx_tn<FMT, T, SCALED, MT, NT, WM, WN, false>), grid, dim3(S::kThreads), S::kLds, st, a);
    }
    return vt_launch_status();
}

template <int FMT, typename T, bool SCALED>
int launch(const MxTN& a, const TnPlan& p, hipStream_t st) {
    return p.bm == 256 ? launch<FMT, T, SCALED, 4, 2, 2, 2>(a, p, st) : launch<FMT, T, SCALED, 2, 1, 2, 2>(a, p, st);
}

template <int FMT, typename T>
int launch(const MxTN& a, const TnPlan& p, hipStream_t st) {
    return a.rowscale ? launch<FMT, T, true>(a, p, st) : launch<FMT, T, false>(a, p, st);
}

template <int FMT>
int launch(int type, const MxTN& a, const TnPlan& p, hipStream_t st) {
    return type == VT_TYPE_F32 ? launch<FMT, float>(a, p, st) : type == VT_TYPE_BF16 ? launch<FMT, bf16>(a, p, st) : launch<FMT, f16>(a, p, st);
}

}  // namespace

extern "C" size_t vt_mx_gemm_tn_workspace_bytes(int64_t N, int Da, int Db) {
    if (N < 0 || Da < 1 || Db < 1) return 0;
    return (size_t)plan(N, Da, Db).slabs * Da * Db * sizeof(float);
}

extern "C" int vt_mx_gemm_tn(int format, const void* codes, int64_t ldc, const void* scales, int64_t lds, int Da, int type,
                             const void* B, int64_t ldb, int Db, const double* rowscale, int64_t N, float alpha,
                             const float* bias, float* C, int64_t ldo, void* ws, size_t ws_bytes, void* stream) {
    if (!mx_rows_ok(format, codes, ldc, scales, lds, N, Da) || Db < 1 || !C || ldo < Db) return VT_ERR_BAD_ARG;
    if (type < VT_TYPE_F32 || type > VT_TYPE_F16 || (N > 0 && (!B || ldb < Db))) return VT_ERR_BAD_ARG;
    const TnPlan p = plan(N, Da, Db);
    if (!ws || ws_bytes < vt_mx_gemm_tn_workspace_bytes(N, Da, Db)) return VT_ERR_WORKSPACE;
    if ((Db + p.bn - 1) / p.bn > 65535) return VT_ERR_UNSUPPORTED;
    const int64_t es = type == VT_TYPE_F32 ? 4 : 2;
    const bool vec = (uintptr_t)B % 16 == 0 && ldb * es % 16 == 0;
    MxTN a{(const uint8_t*)codes, (const uint8_t*)scales, ldc, lds, N, p.rows, Da, Db, B, ldb, vec, rowscale, alpha, bias, C, ldo, (float*)ws};
    return format == VT_MX_FP8 ? launch<VT_MX_FP8>(type, a, p, (hipStream_t)stream) : launch<VT_MX_FP4>(type, a, p, (hipStream_t)stream);
}
