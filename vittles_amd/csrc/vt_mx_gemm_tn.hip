// Gradient of a linear layer's weights from stored activations: C (Da, Db) = alpha A^T diag(rowscale) B + 1 bias^T with
// compact rows A (N, Da) and float, bfloat16 or half rows B (N, Db), on v_mfma_f32_32x32x16_bf16.
// A code times its scale has 4 significant bits at most and is a bfloat16 (v_cvt_scalef32_pk_bf16_fp8 / _fp4) down to that
// type's smallest step, 2^-133: A enters the product exactly, but for the finest codes of E4M3 blocks with scale bytes 0 to
// 2 (largest magnitude below 2^-116), which are rounded to that step.  B is cut into bfloat16 parts that add up to it: one
// for bfloat16, two for half (11 bits), three for float (24 bits) and for anything times rowscale (rounded once to float);
// the parts of a float below 2^-110 end at 2^-133 too, what is finer is cut off.  Products are exact; sums are float.
// Both operands are contracted along the rows, across which they lie in memory: a chunk of rows is staged as it lies and
// read with the transposing LDS read (ds_read_b64_tr_b16), 4 rows x 16 columns a quarter wave.
// The long axis N is cut into slabs; a slab's sums are float and the slabs are added in a fixed order.
// What bounds it: 8192 x 4096 x 4096 takes 235 us in bfloat16 (1.17 PFLOP/s; a library product of 8192^3 reaches 1.36), 470
// in half, 670 in float and 715 weighted.  With one part it is LDS: a chunk of 64 rows costs 48 transposing reads of 512
// bytes in each of 8 waves, 2730 cycles at 72 bytes a cycle, 512 for the writes and 260 of conflicts, against 2048 of MFMA;
// measured at 16384 x 4096 x 1000: 4280 cycles a chunk, the matrix unit busy in 48 %.  For 16 rows two parts come to 910
// cycles of reads and 1024 of MFMA, three to 1138 and 1536.  Two VALU instructions go with an MFMA (conversion, the way to
// LDS).  Reading operands a step ahead, spreading the writes to LDS over the steps, or fixing the order of the two
// took the same time within 2 %; eight rows of a column side by side in LDS, read with ds_read_b128 at twice the rate of
// the transposing read (133 against 72 bytes a cycle) and put there by v_perm, 3 to 8 % longer; one chunk ahead instead of
// two 8 to 18 % longer.  16384 x 4096 x 1000 takes 140 to 150 us, 15 of them the slabs' way out and back, and 120
// if B is zeros: the clock that the power leaves (2.0 GHz) has its share.  Odd rows of B cost 0 (float) to 25 % (bfloat16,
// 16384 x 4096 x 1001: 179 us).  129 to 255 tiles of 256 x 256 go as one slab and leave CUs idle: 16384 x 4096 x 2304, 144
// tiles, takes 373 us in bfloat16 (0.83 PFLOP/s).
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
    const double* rowscale;
    float alpha;
    const float* bias;
    float* C;
    int64_t ldo;
    float* part;                    // [slabs][Da][Db], when there are several
};

// A workgroup of WM x WN waves, each MT x NT products of 32 x 32; kRows rows a chunk, two chunks in LDS (64 rows, where
// they fit, halve the barriers: 16384 x 4096 x 1000 in bfloat16 165 -> 151 us).
template <int MT, int NT, int WM, int WN, int PARTS>
struct TnShape {
    static constexpr int kThreads = 64 * WM * WN, BM = 32 * MT * WM, BN = 32 * NT * WN, kRows = PARTS == 1 && BN == 256 ? 64 : 32;
    // 64 bytes behind every row: the four rows of a transposing read lie in different banks
    static constexpr int kPitchA = 2 * BM + 64, kPitchB = 2 * BN + 64;
    static constexpr int kA = kRows * kPitchA, kB = kRows * kPitchB, kBuf = kA + PARTS * kB, kLds = 2 * kBuf;
    static constexpr int kLoadsA = kRows * BM / 16 / kThreads, kLoadsB = kRows * BN / 8 / kThreads;      // 16 and 8 columns each
    static_assert(kRows * BM / 16 % kThreads == 0 && kRows * BN / 8 % kThreads == 0, "even shares");
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

template <int FMT, typename T, bool SCALED, int MT, int NT, int WM, int WN, bool VEC, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_mx_tn(MxTN a, int tiles_d, int tiles_k) {
    constexpr int PARTS = kParts<T, SCALED>;
    using S = TnShape<MT, NT, WM, WN, PARTS>;
    using W = typename std::conditional<FMT == VT_MX_FP8, u32x4, u32x2>::type;      // 16 codes
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    // workgroups go to the 8 XCDs in turn: each gets a run of tiles, slab by slab, which share the slab's rows in its L2
    const int tiles = tiles_d * tiles_k, per_xcd = gridDim.x >> 3;
    const int t = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3), slab = t / tiles, tile = t - slab * tiles;
    const int64_t n_lo = slab * a.rows, n_hi = std::min(a.N, n_lo + a.rows);
    if (slab * a.rows >= std::max<int64_t>(a.N, 1)) return;
    const int d0 = tile / tiles_k * S::BM, k0 = tile % tiles_k * S::BN;
    const int width = mx_blocks(a.Da) * kMxBlock;

    // VEC: B's rows begin on 4 bytes (B's last column may bring the 2 bytes behind it, never another 4).  Else, in 16-bit
    // types: the aligned words around a piece, shifted into place when it goes to LDS (a row's parity is the same in every
    // chunk).
    const unsigned odd_base = VEC ? 0 : (unsigned)(uintptr_t)a.B & 2;
    unsigned va[S::kLoadsA], vs[S::kLoadsA], vb[S::kLoadsB];
#pragma unroll
    for (int i = 0; i < S::kLoadsA; ++i) {
        const int e = tid + S::kThreads * i, c = d0 + e % (S::BM / 16) * 16;
        const unsigned r = e / (S::BM / 16);
        va[i] = c < width ? r * (unsigned)a.ldc + (FMT == VT_MX_FP8 ? c : c / 2) : kNowhere;
        vs[i] = c < width ? r * (unsigned)a.lds + c / kMxBlock : kNowhere;
    }
#pragma unroll
    for (int i = 0; i < S::kLoadsB; ++i) {
        const int e = tid + S::kThreads * i, c = k0 + e % (S::BN / 8) * 8;
        vb[i] = c < a.Db ? odd_base + (e / (S::BN / 8) * (unsigned)a.ldb + c) * (unsigned)sizeof(T) : kNowhere;
    }
    struct Chunk {
        W ca[S::kLoadsA];
        unsigned sc[S::kLoadsA];
        u32x4 cb[S::kLoadsB][sizeof(T) / 2];
        unsigned tail[VEC ? 1 : S::kLoadsB];
        double rs[SCALED ? S::kLoadsB : 1];
    };
    // rows behind the slab's end come as 0; columns of a piece behind the last one are the next row's and end in columns
    // of the tile that are not stored
    auto fetch = [&](int64_t n0, Chunk& x) {
        const int64_t left = n_hi - n0;
        const auto ra = mx_rsrc(a.codes + n0 * a.ldc, left > 0 ? (left - 1) * a.ldc + (FMT == VT_MX_FP8 ? width : width / 2) : 0);
        const auto rs = mx_rsrc(a.scales + n0 * a.lds, left > 0 ? (left - 1) * a.lds + width / kMxBlock : 0);
        const auto rb = mx_rsrc((const uint8_t*)a.B - odd_base + n0 * a.ldb * (int64_t)sizeof(T),
                                left > 0 ? (odd_base + ((left - 1) * a.ldb + a.Db) * (int64_t)sizeof(T) + 3) / 4 * 4 : 0);
#pragma unroll
        for (int i = 0; i < S::kLoadsA; ++i) {
            if constexpr (FMT == VT_MX_FP8) x.ca[i] = __builtin_bit_cast(W, __builtin_amdgcn_raw_buffer_load_b128(ra, va[i], 0, 0));
            else x.ca[i] = __builtin_bit_cast(W, __builtin_amdgcn_raw_buffer_load_b64(ra, va[i], 0, 0));
            x.sc[i] = __builtin_amdgcn_raw_buffer_load_b8(rs, vs[i], 0, 0);
        }
#pragma unroll
        for (int i = 0; i < S::kLoadsB; ++i) {
            if constexpr (VEC) {
#pragma unroll
                for (int j = 0; j < (int)sizeof(T) / 2; ++j)
                    x.cb[i][j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rb, vb[i] + 16 * j, 0, 0));
            } else {
                // (a row behind the last one shares a word with it)
                const unsigned off = (tid + S::kThreads * i) / (S::BN / 8) < left ? vb[i] & ~3u : kNowhere;
                x.cb[i][0] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rb, off, 0, 0));
                x.tail[i] = __builtin_amdgcn_raw_buffer_load_b32(rb, off + 16, 0, 0);
            }
            if constexpr (SCALED) {
                const int64_t n = n0 + (tid + S::kThreads * i) / (S::BN / 8);
                x.rs[i] = n < n_hi ? a.rowscale[n] : 0.0;
            }
        }
    };
    auto put = [&](const Chunk& x, uint8_t* base) {
#pragma unroll
        for (int i = 0; i < S::kLoadsA; ++i) {
            const int e = tid + S::kThreads * i;
            const float s = mx_scale(x.sc[i]);
            u32x4 v[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                bf16x2 q[4];
                if constexpr (FMT == VT_MX_FP8) {
                    q[0] = mx_pair_bf16<FMT, 0>(x.ca[i][2 * h], s), q[1] = mx_pair_bf16<FMT, 1>(x.ca[i][2 * h], s);
                    q[2] = mx_pair_bf16<FMT, 0>(x.ca[i][2 * h + 1], s), q[3] = mx_pair_bf16<FMT, 1>(x.ca[i][2 * h + 1], s);
                } else {
                    q[0] = mx_pair_bf16<FMT, 0>(x.ca[i][h], s), q[1] = mx_pair_bf16<FMT, 1>(x.ca[i][h], s);
                    q[2] = mx_pair_bf16<FMT, 2>(x.ca[i][h], s), q[3] = mx_pair_bf16<FMT, 3>(x.ca[i][h], s);
                }
                v[h] = u32x4{__builtin_bit_cast(unsigned, q[0]), __builtin_bit_cast(unsigned, q[1]), __builtin_bit_cast(unsigned, q[2]),
                             __builtin_bit_cast(unsigned, q[3])};
            }
            // eight lanes write the first halves of their 32 bytes while the next eight write the second: all banks
            uint8_t* p = base + e / (S::BM / 16) * S::kPitchA + e % (S::BM / 16) * 32;
            const bool odd = lane & 8;
            *(u32x4*)(p + (odd ? 16 : 0)) = odd ? v[1] : v[0];
            *(u32x4*)(p + (odd ? 0 : 16)) = odd ? v[0] : v[1];
        }
#pragma unroll
        for (int i = 0; i < S::kLoadsB; ++i) {
            const int e = tid + S::kThreads * i;
            uint8_t* p = base + S::kA + e / (S::BN / 8) * S::kPitchB + e % (S::BN / 8) * 16;
            u32x4 b8[sizeof(T) / 2];
            __builtin_memcpy(b8, x.cb[i], sizeof(b8));
            if constexpr (!VEC) {
                const unsigned by = (vb[i] & 2) * 8;
#pragma unroll
                for (int j = 0; j < 4; ++j) b8[0][j] = __builtin_amdgcn_alignbit(j < 3 ? b8[0][j + 1] : x.tail[i], b8[0][j], by);
            }
            if constexpr (PARTS == 1) {
                *(u32x4*)p = b8[0];
            } else {
                T c[8];
                __builtin_memcpy(c, b8, sizeof(c));
                u32x4 w[PARTS];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    unsigned y[2][PARTS];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float b = (float)c[2 * j + h];
                        if constexpr (SCALED) b = (float)(x.rs[i] * (double)b);
                        split<PARTS>(b, y[h]);
                    }
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) w[q][j] = y[0][q] | y[1][q] << 16;
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

    // two chunks ahead in registers, one in LDS; chunks behind the end are zeros and add nothing
    Chunk even, odd;
    fetch(n_lo, even);
    fetch(n_lo + S::kRows, odd);
    put(even, lds);
    for (int64_t n0 = n_lo; n0 < n_hi; n0 += 2 * S::kRows) {
        vt_lds_barrier();           // the chunk is written, and the other place is read
        fetch(n0 + 2 * S::kRows, even);
        multiply(lds);
        put(odd, lds + S::kBuf);
        vt_lds_barrier();
        fetch(n0 + 3 * S::kRows, odd);
        multiply(lds + S::kBuf);
        put(even, lds);
    }

    // lane, element e of a 32 x 32 result: row 8 (e / 4) + 4 (lane / 32) + e % 4, column lane % 32; rows and columns past
    // the end fall outside the descriptor
    const int l = lane & 31, h = lane >> 5;
    const int64_t ld = SPLIT ? a.Db : a.ldo;
    float* const out = SPLIT ? a.part + (int64_t)slab * a.Da * a.Db : a.C;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int d = d0 + 32 * (wm * MT + i);
        const auto rc = mx_rsrc(out + d * ld + k0, d < a.Da ? ((a.Da - 1 - d) * ld + a.Db - k0) * (int64_t)sizeof(float) : 0);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int k = 32 * (wn * NT + j) + l;
            const bool in = k0 + k < a.Db;
            const float bias = !SPLIT && a.bias && in ? a.bias[k0 + k] : 0.0f;
            const unsigned at = in ? 4 * (4 * h * (unsigned)ld + k) : kNowhere;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, SPLIT ? acc[i][j][e] : a.alpha * acc[i][j][e] + bias), rc,
                                                      at + 4 * (8 * (e / 4) + e % 4) * (unsigned)ld, 0, 0);
        }
    }
}

// The slabs' sums in a fixed order: 32 elements a workgroup, G groups of threads that each take every G-th slab.
template <int G>
__global__ __launch_bounds__(32 * G) void k_mx_tn_join(MxTN a, int slabs) {
    __shared__ float sh[G][33];
    const int x = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int64_t total = (int64_t)a.Da * a.Db, i = (int64_t)blockIdx.x * 32 + x;
    float s = 0.0f;
    if (i < total)
        for (int p = g; p < slabs; p += G) s += a.part[p * total + i];
    sh[g][x] = s;
    __syncthreads();
    if (g == 0 && i < total) {
#pragma unroll
        for (int q = 1; q < G; ++q) s += sh[q][x];
        const int64_t d = i / a.Db;
        const int k = (int)(i - d * a.Db);
        a.C[d * a.ldo + k] = a.alpha * s + (a.bias ? a.bias[k] : 0.0f);
    }
}

// The same for few slabs: a thread an element.
__global__ __launch_bounds__(256) void k_mx_tn_join_few(MxTN a, int slabs) {
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
    // 128 x 64 tiles where a round or two of them with 128 rows each is the whole product: the way in and out of a tile of
    // 256 x 256 alone takes longer (35 x 1156 x 217 in float: 7 us, 28 in tiles of 256 x 256)
    const int64_t small = (int64_t)((Da + 127) / 128) * ((Db + 63) / 64) * ((N + 127) / 128);
    if (Db <= 64 || small <= 4 * vt_num_cu()) p.bm = 128, p.bn = 64;
    else p.bm = 256, p.bn = Db > 128 ? 256 : 128;
    const int64_t tiles = (int64_t)((Da + p.bm - 1) / p.bm) * ((Db + p.bn - 1) / p.bn);
    const int64_t want = std::max<int64_t>(1, (p.bn == 256 ? 1 : 2) * vt_num_cu() / tiles), most = std::max<int64_t>(1, N / 128);
    p.slabs = (int)std::min(want, most);
    p.rows = (std::max<int64_t>(1, (N + p.slabs - 1) / p.slabs) + 127) / 128 * 128;
    p.slabs = (int)std::max<int64_t>(1, (N + p.rows - 1) / p.rows);
    return p;
}

template <int FMT, typename T, bool SCALED, int MT, int NT, int WM, int WN, bool VEC>
int launch(const MxTN& a, const TnPlan& p, hipStream_t st) {
    using S = TnShape<MT, NT, WM, WN, kParts<T, SCALED>>;
    const int td = (a.Da + S::BM - 1) / S::BM, tk = (a.Db + S::BN - 1) / S::BN;
    const dim3 grid((unsigned)(((int64_t)td * tk * p.slabs + 7) / 8 * 8));
    static VtLdsAttr attr_split, attr_whole;
    if (p.slabs > 1) {
        if (vt_allow_big_lds((const void*)k_mx_tn<FMT, T, SCALED, MT, NT, WM, WN, VEC, true>, attr_split, S::kLds) != VT_OK) return VT_ERR_HIP;
        hipLaunchKernelGGL((k_mx_tn<FMT, T, SCALED, MT, NT, WM, WN, VEC, true>), grid, dim3(S::kThreads), S::kLds, st, a, td, tk);
        const int64_t total = (int64_t)a.Da * a.Db;
        if (p.slabs <= 8)
            hipLaunchKernelGGL(k_mx_tn_join_few, dim3((unsigned)std::min<int64_t>((total + 255) / 256, 8 * vt_num_cu())), dim3(256), 0, st, a, p.slabs);
        else
            hipLaunchKernelGGL(k_mx_tn_join<16>, dim3((unsigned)((total + 31) / 32)), dim3(512), 0, st, a, p.slabs);
    } else {
        if (vt_allow_big_lds((const void*)k_mx_tn<FMT, T, SCALED, MT, NT, WM, WN, VEC, false>, attr_whole, S::kLds) != VT_OK) return VT_ERR_HIP;
        hipLaunchKernelGGL((k_mx_tn<FMT, T, SCALED, MT, NT, WM, WN, VEC, false>), grid, dim3(S::kThreads), S::kLds, st, a, td, tk);
    }
    return vt_launch_status();
}

template <int FMT, typename T, bool SCALED, bool VEC>
int launch(const MxTN& a, const TnPlan& p, hipStream_t st) {
    if (p.bn == 256) return launch<FMT, T, SCALED, 4, 2, 2, 4, VEC>(a, p, st);
    if (p.bm == 256) return launch<FMT, T, SCALED, 4, 2, 2, 2, VEC>(a, p, st);
    return launch<FMT, T, SCALED, 2, 1, 2, 2, VEC>(a, p, st);
}

template <int FMT, typename T, bool SCALED>
int launch(const MxTN& a, const TnPlan& p, hipStream_t st) {
    if constexpr (sizeof(T) == 2)
        if ((uintptr_t)a.B % 4 != 0 || a.ldb % 2 != 0) return launch<FMT, T, SCALED, false>(a, p, st);
    return launch<FMT, T, SCALED, true>(a, p, st);
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
    // one slab goes straight to C; a float all the same, so that what a caller allocates has an address
    const int slabs = plan(N, Da, Db).slabs;
    return slabs > 1 ? (size_t)slabs * Da * Db * sizeof(float) : sizeof(float);
}

extern "C" int vt_mx_gemm_tn(int format, const void* codes, int64_t ldc, const void* scales, int64_t lds, int Da, int type,
                             const void* B, int64_t ldb, int Db, const double* rowscale, int64_t N, float alpha,
                             const float* bias, float* C, int64_t ldo, void* ws, size_t ws_bytes, void* stream) {
    if (!mx_rows_ok(format, codes, ldc, scales, lds, N, Da) || Db < 1 || !C || ldo < Db) return VT_ERR_BAD_ARG;
    if (type < VT_TYPE_F32 || type > VT_TYPE_F16 || (N > 0 && (!B || ldb < Db))) return VT_ERR_BAD_ARG;
    if ((uintptr_t)B % (type == VT_TYPE_F32 ? 4 : 2)) return VT_ERR_BAD_ARG;
    const TnPlan p = plan(N, Da, Db);
    if (!ws || ws_bytes < vt_mx_gemm_tn_workspace_bytes(N, Da, Db)) return VT_ERR_WORKSPACE;
    if (N <= 1) ldb = (Db + 7) / 8 * 8;      // a single row has no stride
    // 32-bit offsets inside a chunk of 64 rows, tile numbers in 31 bits
    if (ldc >= 1 << 25 || lds >= 1 << 25 || (N > 1 && ldb >= 1 << 23) || ldo >= 1 << 24) return VT_ERR_UNSUPPORTED;
    if ((int64_t)((Da + p.bm - 1) / p.bm) * ((Db + p.bn - 1) / p.bn) * p.slabs > 0x7ffffff0) return VT_ERR_UNSUPPORTED;
    MxTN a{(const uint8_t*)codes, (const uint8_t*)scales, ldc, lds, N, p.rows, Da, Db, B, ldb, rowscale, alpha, bias, C, ldo, (float*)ws};
    return format == VT_MX_FP8 ? launch<VT_MX_FP8>(type, a, p, (hipStream_t)stream) : launch<VT_MX_FP4>(type, a, p, (hipStream_t)stream);
}
