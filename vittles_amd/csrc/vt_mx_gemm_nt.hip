// Product of 4-bit compact rows: C (M, N) = alpha A B^T + 1 bias^T on the scaled MFMA.
// A lane of v_mfma_scale_f32_32x32x64_f8f6f4 (16x16x128) holds 32 codes of row (lane mod 32 (16)), block lane / 32 (16)
// of the step's two (four): one compact block and its scale byte, so both operands go from memory to the matrix unit as
// they are stored.  E2M1 products times powers of two are exact and the sums are float (the E4M3 form of the instruction
// keeps only about 17 bits of a sum: 8-bit rows are not multiplied this way).
#include "vt_mx.h"
#include <type_traits>

namespace {

constexpr int kFp4 = 4;                 // the instruction's format code

struct MxNT {
    const uint8_t *ca, *sa, *cb, *sb;
    int64_t ldca, ldsa, ldcb, ldsb, M, N;
    int nb, step;                       // blocks of a row; of a slice of the split axis
    float alpha;
    const float* bias;
    void* C;
    int64_t ldc;
    bool lines;                         // C's rows begin on cache lines
    float* part;                        // [slices][M][N] sums, when the axis is split
};

// The instruction reads four registers of E2M1 codes; the builtin's other four stay undefined.
__device__ __forceinline__ i32x8 nt_operand(u32x4 w) {
    return __builtin_bit_cast(i32x8, __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1));
}

template <typename OutT>
__device__ __forceinline__ void mx_store(const MxNT& a, int64_t m, int64_t n, float v) {
    ((OutT*)a.C)[m * a.ldc + n] = (OutT)(a.alpha * v + (a.bias ? a.bias[n] : 0.0f));
}

// ---- tiles ----------------------------------------------------------------------------------------------------------
// A workgroup of WM x WN waves computes a (32 MT WM) x (32 NT WN) tile of C, each wave MT x NT products of 32 x 32.  The
// axis goes by in chunks of 8 blocks (256 columns, 128 bytes a row: whole cache lines; chunks of 64 bytes with four
// places in LDS took 18 % longer, their lines come from L2 twice).  LDS holds two chunks: the next one is on its way
// (LDS-DMA, 16 bytes a lane for codes, 4 for scales) while this one is multiplied.
// LDS: 16-byte slot j of row r holds block j ^ ((r >> 1) & 7), so the sixteen rows that are read at a time lie in
// different banks.  The DMA writes slots in lane order; the permutation is in the lanes' addresses.
// Measured at 8192^3: 295 us from a graph, 315 among other kernels (3.7 and 3.5 PFLOP/s, medians; bfloat16 result 274);
// 4096^2 x 8192: 79 us, 3.5.  The codes' way from L2 alone takes 225 (2.1 GB at the ~10 TB/s that two chunks in flight
// draw), products and operand reads alone 214, writing C 50: the first two overlap, the last does not, a tile's workgroup
// fills its CU.  Reading operands a step ahead, with the barrier under the last step's products, took the same time.
constexpr int kChunk = 8, kRow = 16 * kChunk, kRowsPerLoad = 1024 / kRow;
__device__ __forceinline__ int nt_slot(int block, int row) { return 16 * (block ^ ((row >> 1) & 7)); }

typedef __attribute__((address_space(3))) void* mx_ldsptr;

template <int MT, int NT, int WM, int WN>
struct NtShape {
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves, BM = 32 * MT * WM, BN = 32 * NT * WN;
    static constexpr int kCodes = (BM + BN) * 16 * kChunk, kBuf = kCodes + (BM + BN) * kChunk, kLds = 2 * kBuf;
    static constexpr int kLoadsA = BM / (kRowsPerLoad * kWaves), kLoadsB = BN / (kRowsPerLoad * kWaves),
                         kLoadsS = (BM + BN) * (kChunk / 4) / kThreads;      // of a wave for one chunk
    static_assert(BM % (kRowsPerLoad * kWaves) == 0 && BN % (kRowsPerLoad * kWaves) == 0 && BM + BN == kThreads, "even shares, one row of scales a thread");
};

// DMA: the scales' rows all begin on 4 bytes and their words come by DMA too; else through registers (10 % slower).
template <int MT, int NT, int WM, int WN, bool DMA, typename OutT, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN) void k_mx_nt_tile(MxNT a, int tiles_m, int tiles_n) {
    using S = NtShape<MT, NT, WM, WN>;
    constexpr int kLoadsA = S::kLoadsA, kLoadsB = S::kLoadsB, kLoads = kLoadsA + kLoadsB + (DMA ? S::kLoadsS : 0), kWords = kChunk / 4, kScaleRows = 64 / kWords;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    // workgroups go to the 8 XCDs in turn: each XCD gets a run of tiles, walked in bands of 8 tiles along M, so that the
    // tiles in flight on an XCD share rows of A and of B in its L2
    const int total = tiles_m * tiles_n, per_xcd = gridDim.x >> 3;
    const int t = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (t >= total) return;
    const int band = t / (8 * tiles_n), in_band = t - band * 8 * tiles_n, width = std::min(8, tiles_m - band * 8);
    const int64_t m0 = (int64_t)(band * 8 + in_band % width) * S::BM, n0 = (int64_t)(in_band / width) * S::BN;
    const int kb_lo = blockIdx.y * a.step, kb_hi = std::min(a.nb, kb_lo + a.step);
    const int chunks = (kb_hi - kb_lo + kChunk - 1) / kChunk;

    const int rows_a = (int)std::min<int64_t>(S::BM, a.M - m0), rows_b = (int)std::min<int64_t>(S::BN, a.N - n0);
    // rows past the end read 0; blocks past a row's end are the next row's, and are masked in the last chunk
    const auto ra = mx_rsrc(a.ca + m0 * a.ldca, (rows_a - 1) * a.ldca + 16 * (int64_t)a.nb);
    const auto rb = mx_rsrc(a.cb + n0 * a.ldcb, (rows_b - 1) * a.ldcb + 16 * (int64_t)a.nb);
    const int rl = lane / kChunk, piece = nt_slot(lane % kChunk, rl + kRowsPerLoad * wave);     // (kWaves is even)
    const unsigned va = rl * (unsigned)a.ldca + piece, vb = rl * (unsigned)a.ldcb + piece;
    // (a scale word that holds a row's last scale may reach up to three bytes behind it, never out of its own 4 bytes)
    const auto rsa = mx_rsrc(a.sa + m0 * a.ldsa, (rows_a - 1) * a.ldsa + (a.nb + 3) / 4 * 4);
    const auto rsb = mx_rsrc(a.sb + n0 * a.ldsb, (rows_b - 1) * a.ldsb + (a.nb + 3) / 4 * 4);
    const unsigned vsa = lane / kWords * (unsigned)a.ldsa + 4 * (lane % kWords), vsb = lane / kWords * (unsigned)a.ldsb + 4 * (lane % kWords);
    // not DMA: this thread's row of scales; rows past the end repeat the last one
    const uint8_t* const ps = tid < S::BM ? a.sa + (m0 + std::min(tid, rows_a - 1)) * a.ldsa : a.sb + (n0 + std::min(tid - S::BM, rows_b - 1)) * a.ldsb;

    // load number i of this wave for the chunk at block kb
    auto fetch = [&](int kb, uint8_t* base, int i) {
        if (i < kLoadsA) {
            const int row = kRowsPerLoad * (wave + S::kWaves * i);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (mx_ldsptr)(base + row * kRow), 16, va + row * (unsigned)a.ldca + 16u * kb, 0, 0, 0);
        } else if (i < kLoadsA + kLoadsB) {
            const int row = kRowsPerLoad * (wave + S::kWaves * (i - kLoadsA));
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (mx_ldsptr)(base + (S::BM + row) * kRow), 16, vb + row * (unsigned)a.ldcb + 16u * kb, 0, 0, 0);
        } else {
            const int row = kScaleRows * (wave + S::kWaves * (i - kLoadsA - kLoadsB));
            const bool first = row < S::BM;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(first ? rsa : rsb, (mx_ldsptr)(base + S::kCodes + row * kChunk), 4,
                                                     (first ? vsa + row * (unsigned)a.ldsa : vsb + (row - S::BM) * (unsigned)a.ldsb) + kb, 0, 0, 0);
        }
    };
    // the eight scale bytes of its chunk, at whatever address they lie; blocks past the row's end count as 1
    auto scales = [&](int kb) -> u32x2 {
        typedef unsigned u32x2u __attribute__((ext_vector_type(2), aligned(1)));
        if (kb + kChunk <= a.nb) return *(const u32x2u*)(ps + kb);
        uint64_t v = 0;
#pragma unroll 1
        for (int j = 0; j < kChunk; ++j) v |= (uint64_t)(kb + j < a.nb ? ps[kb + j] : 127) << (8 * j);
        return __builtin_bit_cast(u32x2, v);
    };

    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    const int l = lane & 31, h = lane >> 5;
    // the chunk at `base`, with the loads of the chunk at block kb (if `more`) into `next` between the products
    auto multiply = [&](const uint8_t* base, bool more, int kb, uint8_t* next) {
        const uint8_t* pa = base + (wm * 32 * MT + l) * kRow;
        const uint8_t* pb = base + (S::BM + wn * 32 * NT + l) * kRow;
        const uint8_t* sc = base + S::kCodes;
        // bytes 0 and 2 of a word: the scales of its two steps for this half of the wave
        unsigned sa[MT][kWords], sb[NT][kWords];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int w = 0; w < kWords; ++w) sa[i][w] = *(const unsigned*)(sc + (wm * 32 * MT + 32 * i + l) * kChunk + 4 * w) >> (8 * h);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int w = 0; w < kWords; ++w) sb[j][w] = *(const unsigned*)(sc + (S::BM + wn * 32 * NT + 32 * j + l) * kChunk + 4 * w) >> (8 * h);
#pragma unroll
        for (int s = 0; s < kChunk / 2; ++s) {
            const int slot = nt_slot(2 * s + h, l);
            i32x8 fa[MT], fb[NT];
#pragma unroll
            for (int i = 0; i < MT; ++i) fa[i] = nt_operand(*(const u32x4*)(pa + 32 * kRow * i + slot));
#pragma unroll
            for (int j = 0; j < NT; ++j) fb[j] = nt_operand(*(const u32x4*)(pb + 32 * kRow * j + slot));
            if (more) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i)
                    if (i * 2 / kLoads == s) fetch(kb, next, i);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[i][j] = s % 2 == 0 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa[i], fb[j], acc[i][j], kFp4, kFp4, 0, (int)sa[i][s / 2], 0, (int)sb[j][s / 2])
                                           : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa[i], fb[j], acc[i][j], kFp4, kFp4, 2, (int)sa[i][s / 2], 2, (int)sb[j][s / 2]);
        }
    };
    auto barrier = [] {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    uint8_t* const scale_slot = lds + S::kCodes + tid * kChunk;
    if constexpr (!DMA) *(u32x2*)scale_slot = scales(kb_lo);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) fetch(kb_lo, lds, i);
    for (int c = 0; c < chunks; ++c) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // this wave's part of chunk c has landed
        barrier();          // everybody's has, and chunk c - 1 has been read: its place is free
        uint8_t* base = lds + (c & 1) * S::kBuf;
        const int kb = kb_lo + kChunk * c;
        if (kb + kChunk > a.nb) {
            // the row ends inside this chunk: codes of A behind the end become 0 and scales 1, so that what was
            // fetched there (the next row's) counts for nothing
            if constexpr (DMA)
                for (int i = tid; i < (S::BM + S::BN) * kChunk; i += S::kThreads)
                    if (kb + i % kChunk >= a.nb) base[S::kCodes + i] = 127;
            for (int i = tid; i < S::BM * kChunk; i += S::kThreads) {
                const int row = i / kChunk, j = i % kChunk;
                if (kb + j >= a.nb) *(u32x4*)(base + row * kRow + nt_slot(j, row)) = u32x4{0, 0, 0, 0};
            }
            barrier();
        }
        u32x2 next = {0, 0};
        if constexpr (!DMA)
            if (c + 1 < chunks) next = scales(kb + kChunk);
        multiply(base, c + 1 < chunks, kb + kChunk, lds + (~c & 1) * S::kBuf);
        if (!DMA && c + 1 < chunks) *(u32x2*)(scale_slot + (~c & 1) * S::kBuf) = next;
    }

    // lane, element e of a 32 x 32 result: row 8 (e / 4) + 4 (lane / 32) + e % 4, column lane % 32; rows and columns past
    // the end fall outside the descriptor
    using T = typename std::conditional<SPLIT, float, OutT>::type;
    const int64_t ld = SPLIT ? a.N : a.ldc;
    T* const out = SPLIT ? (T*)(a.part + (int64_t)blockIdx.y * a.M * a.N) : (T*)a.C;
    auto write = [&](auto aux) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int64_t m = m0 + 32 * (wm * MT + i);
            const auto rc = mx_rsrc(out + m * ld + n0, m < a.M ? ((a.M - 1 - m) * ld + a.N - n0) * (int64_t)sizeof(T) : 0);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int n = 32 * (wn * NT + j) + l;
                const float bias = !SPLIT && a.bias && n < rows_b ? a.bias[n0 + n] : 0.0f;
                const unsigned at = n < rows_b ? (unsigned)sizeof(T) * (4 * h * (unsigned)ld + n) : kNowhere;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const T c = (T)(SPLIT ? acc[i][j][e] : a.alpha * acc[i][j][e] + bias);
                    const unsigned off = at + (unsigned)sizeof(T) * (8 * (e / 4) + e % 4) * (unsigned)ld;
                    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, c), rc, off, 0, decltype(aux)::value);
                    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, c), rc, off, 0, decltype(aux)::value);
                }
            }
        }
    };
    // whole lines go past the caches, C is not read again here (2048 x 4096 x 4096: 35.1 -> 32.5 us); parts of lines have
    // to meet in L2 first (8192 x 8191 x 512: 202 us past it, 93 through it)
    if (!SPLIT && a.lines) write(std::integral_constant<int, 2>());
    else write(std::integral_constant<int, 0>());
}

template <typename OutT>
__global__ __launch_bounds__(256) void k_mx_nt_join(MxNT a, int slices) {
    const int64_t total = a.M * a.N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        float s = 0.0f;
        for (int p = 0; p < slices; ++p) s += a.part[p * total + i];
        const int64_t m = i / a.N;
        mx_store<OutT>(a, m, i - m * a.N, s);
    }
}

// ---- few rows -------------------------------------------------------------------------------------------------------
// Blocks of at most 16 MT rows of the shorter side ("few", F): each workgroup streams 16 rows of the other side ("many")
// straight from memory into v_mfma_scale_f32_16x16x128, its four waves on interleaved chunks of the axis, joined through
// LDS.  For up to 64 rows reading the many rows once is the whole cost; for small products with more it saves the tiles'
// long way in and out (151 x 219 x 563: 6.3 us, 13.5 in tiles).  SWAP: the few rows are B's.
struct MxFew {
    const uint8_t *cm, *sm, *cf, *sf;      // many, few
    int64_t ldcm, ldsm, ldcf, ldsf, many, few;
};

__device__ __forceinline__ i32x8 few_frag(const uint8_t* p, bool in) { return nt_operand(in ? *(const u32x4*)p : u32x4{0, 0, 0, 0}); }

template <int MT, bool SWAP, typename OutT>
__global__ __launch_bounds__(256) void k_mx_nt_few(MxNT a, MxFew f) {
    constexpr int U = 4;                   // steps of 4 blocks a wave takes at once: 256 bytes a row
    __shared__ f32x4 sh[3][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, q = lane >> 4;
    const int64_t r0 = (int64_t)blockIdx.x * 16, f0 = (int64_t)blockIdx.y * 16 * MT;
    const int64_t rm = std::min(r0 + l, f.many - 1);
    const uint8_t *pm = f.cm + rm * f.ldcm, *ps = f.sm + rm * f.ldsm;
    const uint8_t *pf[MT], *pfs[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t r = std::min<int64_t>(f0 + 16 * i + l, f.few - 1);
        pf[i] = f.cf + r * f.ldcf;
        pfs[i] = f.sf + r * f.ldsf;
    }
    f32x4 acc[MT] = {};
    for (int kb0 = wave * 4 * U; kb0 < a.nb; kb0 += 4 * 4 * U) {
        i32x8 fm[U], ff[U][MT];
        int sm[U], sf[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kb = kb0 + 4 * u + q;
            const bool in = kb < a.nb;
            fm[u] = few_frag(pm + (int64_t)kb * 16, in);
            sm[u] = in ? ps[kb] : 127;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                ff[u][i] = few_frag(pf[i] + (int64_t)kb * 16, in);
                sf[u][i] = in ? pfs[i][kb] : 127;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i)
                acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fm[u], ff[u][i], acc[i], kFp4, kFp4, 0, sm[u], 0, sf[u][i]);
    }
    if (wave > 0)
#pragma unroll
        for (int i = 0; i < MT; ++i) sh[wave - 1][i][lane] = acc[i];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        f32x4 v = acc[i];
#pragma unroll
        for (int w = 0; w < 3; ++w) {
            const f32x4 o = sh[w][i][lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += o[e];
        }
        // element e: many row 4 q + e, few row l
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t m = r0 + 4 * q + e, k = f0 + 16 * i + l;
            if (m < f.many && k < f.few) mx_store<OutT>(a, SWAP ? m : k, SWAP ? k : m, v[e]);
        }
    }
}

// A launch holds fewer than 2^32 threads: 2^27 of the many rows are 2^31 of them, more rows go in several launches.
constexpr int64_t kManyRows = 1 << 27;

template <int MT, typename OutT>
int launch_few(const MxNT& whole, hipStream_t st) {
    const bool swap = whole.N < whole.M;
    MxNT a = whole;
    MxFew f = swap ? MxFew{a.ca, a.sa, a.cb, a.sb, a.ldca, a.ldsa, a.ldcb, a.ldsb, a.M, a.N}
                   : MxFew{a.cb, a.sb, a.ca, a.sa, a.ldcb, a.ldsb, a.ldca, a.ldsa, a.N, a.M};
    for (int64_t left = f.many; left > 0; left -= kManyRows) {
        f.many = std::min(left, kManyRows);
        const dim3 grid((unsigned)((f.many + 15) / 16), (unsigned)((f.few + 16 * MT - 1) / (16 * MT)));
        if (swap) hipLaunchKernelGGL((k_mx_nt_few<MT, true, OutT>), grid, dim3(256), 0, st, a, f);
        else hipLaunchKernelGGL((k_mx_nt_few<MT, false, OutT>), grid, dim3(256), 0, st, a, f);
        if (int rc = vt_launch_status()) return rc;
        f.cm += f.many * f.ldcm, f.sm += f.many * f.ldsm;
        a.C = (OutT*)a.C + f.many * (swap ? a.ldc : 1);
        if (!swap && a.bias) a.bias += f.many;
    }
    return VT_OK;
}

struct NtPlan {
    int few;             // > 0: rows on the short side, in 16s
    int shape;           // tile: 0 = 256 x 256 (8 waves), 1 = 128 x 128 (4 waves)
    int slices, step;
};

int64_t tiles(int64_t M, int64_t N, int bm, int bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); }

NtPlan plan(int64_t M, int64_t N, int K, bool far) {
    const int nb = mx_blocks(K);
    NtPlan p{0, 1, 1, (nb + kChunk - 1) / kChunk * kChunk};
    const int64_t less = std::min(M, N), more = std::max(M, N);
    // a few rows' workgroup reads its few rows again for every 16 of the many: up to 48 MB of that from L2 it is the faster
    const double again = 0.5 * K * ((double)((more + 15) / 16) * less + (double)((less + 63) / 64) * more);
    if (less <= 64 || again <= 48e6 || far) {
        p.few = less <= 64 ? (int)((less + 15) / 16) : 4;
        return p;
    }
    // Tiles: 256 x 256, one to a CU: every round takes 17 + 1.75 us a chunk, the writing of C hides behind nothing.
    // 128 x 128, two to a CU: 6 us once and 5 + 1.2 a chunk for a round, one writes while the other multiplies.  Measured, us
    // (256 / 128): 4096^2 x 4096 46 / 53, 8192^2 x 8192 299 / 359, x 2048 118 / 120, x 256 77 / 56, 6000^2 x 1024 47 / 43,
    // 2048 x 4096 x 4096 34 / 29, 3000 x 4000 x 2048 24 / 26.  Tiles of 256 x 128, one
    // to a CU, were no better anywhere: 4096^2 x 4096 59, 8192^3 379, 2048 x 4096 x 4096 30.
    const int cu = vt_num_cu();
    const int chunks = (nb + kChunk - 1) / kChunk;
    const int64_t t = tiles(M, N, 128, 128);
    const double big = (double)((tiles(M, N, 256, 256) + cu - 1) / cu) * (17.0 + 1.75 * chunks);
    const double small = 6.0 + (double)((t + 2 * cu - 1) / (2 * cu)) * (5.0 + 1.2 * chunks);
    p.shape = big < small ? 0 : 1;
    // few tiles and a long axis: slices of at least 8 chunks, joined by a second pass (512 x 512 x 8192: 24 us whole, 14
    // in four slices; 512 x 4096 x 4096, 128 tiles: two slices took 4 us more than the whole)
    const int s = p.shape == 0 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(cu / (2 * t), chunks / 8), 16));
    p.step = (chunks + s - 1) / s * kChunk;
    p.slices = (nb + p.step - 1) / p.step;
    return p;
}

bool scale_words(const void* s, int64_t ld) { return (uintptr_t)s % 4 == 0 && ld % 4 == 0 && ld < 1 << 23; }

template <int MT, int NT, int WM, int WN, bool DMA, typename OutT>
int launch_tile(const MxNT& a, const NtPlan& p, hipStream_t st) {
    using S = NtShape<MT, NT, WM, WN>;
    const int tm = (int)((a.M + S::BM - 1) / S::BM), tn = (int)((a.N + S::BN - 1) / S::BN);
    const int64_t wgs = ((int64_t)tm * tn + 7) / 8 * 8;
    const dim3 grid((unsigned)wgs, p.slices);
    static VtLdsAttr attr_split, attr_whole;
    if (p.slices > 1) {
        if (vt_allow_big_lds((const void*)k_mx_nt_tile<MT, NT, WM, WN, DMA, OutT, true>, attr_split, S::kLds) != VT_OK) return VT_ERR_HIP;
        hipLaunchKernelGGL((k_mx_nt_tile<MT, NT, WM, WN, DMA, OutT, true>), grid, dim3(S::kThreads), S::kLds, st, a, tm, tn);
        hipLaunchKernelGGL((k_mx_nt_join<OutT>), dim3((unsigned)std::min<int64_t>((a.M * a.N + 255) / 256, 8 * vt_num_cu())),
                           dim3(256), 0, st, a, p.slices);
    } else {
        if (vt_allow_big_lds((const void*)k_mx_nt_tile<MT, NT, WM, WN, DMA, OutT, false>, attr_whole, S::kLds) != VT_OK) return VT_ERR_HIP;
        hipLaunchKernelGGL((k_mx_nt_tile<MT, NT, WM, WN, DMA, OutT, false>), grid, dim3(S::kThreads), S::kLds, st, a, tm, tn);
    }
    return vt_launch_status();
}

template <typename OutT>
int launch(const MxNT& a, const NtPlan& p, hipStream_t st) {
    switch (p.few) {
        case 0: break;
        case 1: return launch_few<1, OutT>(a, st);
        case 2: return launch_few<2, OutT>(a, st);
        case 3: return launch_few<3, OutT>(a, st);
        default: return launch_few<4, OutT>(a, st);
    }
    const bool dma = scale_words(a.sa, a.ldsa) && scale_words(a.sb, a.ldsb);
    if (p.shape == 0) return dma ? launch_tile<4, 2, 2, 4, true, OutT>(a, p, st) : launch_tile<4, 2, 2, 4, false, OutT>(a, p, st);
    return dma ? launch_tile<2, 2, 2, 2, true, OutT>(a, p, st) : launch_tile<2, 2, 2, 2, false, OutT>(a, p, st);
}

}  // namespace

extern "C" size_t vt_mx_gemm_nt_workspace_bytes(int64_t M, int64_t N, int K) {
    if (M < 1 || N < 1 || K < 1) return 0;
    const NtPlan p = plan(M, N, K, false);
    return p.few == 0 && p.slices > 1 ? (size_t)p.slices * M * N * sizeof(float) : 0;
}

extern "C" int vt_mx_gemm_nt(const void* ca, int64_t ldca, const void* sa, int64_t ldsa, int64_t M, const void* cb,
                             int64_t ldcb, const void* sb, int64_t ldsb, int64_t N, int K, float alpha, const float* bias,
                             int out_type, void* C, int64_t ldc, void* ws, size_t ws_bytes, void* stream) {
    if (!mx_rows_ok(VT_MX_FP4, ca, ldca, sa, ldsa, M, K) || !mx_rows_ok(VT_MX_FP4, cb, ldcb, sb, ldsb, N, K))
        return VT_ERR_BAD_ARG;
    if (out_type != VT_TYPE_F32 && out_type != VT_TYPE_BF16) return VT_ERR_BAD_ARG;
    if (M == 0 || N == 0) return VT_OK;
    if (!C || ldc < N) return VT_ERR_BAD_ARG;
    if (tiles(M, N, 16, 64) > 0x7ffffff0) return VT_ERR_UNSUPPORTED;
    if (ws_bytes < vt_mx_gemm_nt_workspace_bytes(M, N, K) || (!ws && vt_mx_gemm_nt_workspace_bytes(M, N, K))) return VT_ERR_WORKSPACE;
    // (a tile's offsets are 32 bits: 256 rows of codes, 32 rows of C)
    const NtPlan p = plan(M, N, K, ldca >= 1 << 23 || ldcb >= 1 << 23 || ldc >= 1 << 24);
    MxNT a{(const uint8_t*)ca, (const uint8_t*)sa, (const uint8_t*)cb, (const uint8_t*)sb, ldca, ldsa, ldcb, ldsb, M, N,
           mx_blocks(K), p.step, alpha, bias, C, ldc, (uintptr_t)C % 128 == 0 && ldc * (out_type == VT_TYPE_F32 ? 4 : 2) % 128 == 0, (float*)ws};
    return out_type == VT_TYPE_F32 ? launch<float>(a, p, (hipStream_t)stream) : launch<__bf16>(a, p, (hipStream_t)stream);
}
