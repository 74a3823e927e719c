// Row operators on compact rows: link, gradient, value, fused HVP, A v and A^T (u1 .* u2), with fp64 vectors and sums.
//     for every row n:  dot_n = x_n . v,  t_n = op(dot_n, per-row scalars) -> per-row outputs,  out += t_n x_n
// One pass: a team of threads holds the codes of R rows in registers from the dot to the column sums, 16 columns
// ("a piece": half a block, 16 bytes of E4M3 or 8 of E2M1) a thread and round, and their sums of the columns for the
// whole kernel.  Partial sums are combined in a fixed order (no atomics: the same bits every time).
// What bounds it: HBM for E4M3 (A v and A^T u 4.9 to 5.8 TB/s, HVP 4.0 to 4.5; a copy reaches 4.9).  For E2M1 a round's
// chain -- decode, dots, sums over the waves, barrier, link, columns -- which the one or two workgroups of a CU hardly
// overlap.  An element costs half a conversion to float and one to double, once if its double is kept and twice if not, and
// two fp64 FMAs: 3.5 to 5 instructions of 4 cycles for 64 elements, and about 130 more a wave and round for sums, link and
// addresses.  Of the cycles held the VALU issues in 45 % (gradient, E4M3, N = 10^6, D = 100), 42 % (gradient, E2M1, 20011 x
// 5003: three of eight waves have no piece there and decode the last one again, all eight evaluate the link) and 74 % (HVP,
// E4M3, 10^5 x 20 000, which decodes twice).  Medians, HVP in TB/s of stored bytes: E4M3 N = 4 10^6, D = 100 4.5; N = 10^5,
// D = 8192 4.5, D = 20 000 4.0 - 4.2 (494 - 515 us); E2M1 2.9, 2.7, 2.6 (411 - 419 us).
// (One wave a round for the gradient's coefficients, handed on through LDS and a second barrier: 5 to 12 % longer.)
#include "vt_mx.h"
#include <type_traits>
#include <utility>

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

// The row's scalars, fetched a round before they are used.
struct RowScal {
    double y, w, off;
};
template <int OP>
__device__ __forceinline__ RowScal row_scal(const MxRows& a, int64_t n) {
    RowScal s{0.0, 0.0, 0.0};
    if constexpr (OP == OP_GEMV) return s;
    s.y = a.y[n];
    if constexpr (OP == OP_GEMVT) s.w = a.w ? a.w[n] : 1.0;
    if constexpr (OP == OP_LINK || OP == OP_GRAD || OP == OP_VALUE) {
        s.w = a.w[n];
        if (a.offset) s.off = a.offset[n];
    }
    return s;
}

// The row's coefficient in the column sum (VALUE: its loss); the leading lane writes the row's outputs.
template <int OP>
__device__ __forceinline__ double mx_row_op(const MxRows& a, int64_t n, const RowScal& s, double dot, bool lead) {
    if constexpr (OP == OP_GEMVT) {
        return s.y * s.w;
    } else if constexpr (OP == OP_HVP) {
        return s.y * dot;
    } else if constexpr (OP == OP_GEMV) {
        if (lead) a.z[n] = dot;
        return 0.0;
    } else {
        const double z = dot + s.off;
        if constexpr (OP == OP_VALUE) {
            return s.w * vt_loss(a.family, z, s.y);
        } else {
            double l1, l2;
            vt_link(a.family, z, s.y, l1, l2);
            if (lead) {
                if (a.z) a.z[n] = z;
                if (a.r) a.r[n] = a.scale * l1;
                if (a.d) a.d[n] = a.scale * s.w * l2;
            }
            return s.w * (a.scale * l1);
        }
    }
}

// ---- one pass ---------------------------------------------------------------------------------------------------------
// Codes and scales come through buffer descriptors that begin at a workgroup's rows of the round and end with the
// matrix: the lane's offset is 32 bits, and rows behind the end read as 0 (their coefficient is 0 too).
typedef __amdgpu_buffer_rsrc_t MxRsrc;
__device__ __forceinline__ MxRsrc rows_rsrc(const uint8_t* base, int64_t n0, int64_t ld, int64_t N, int64_t width) {
    const int64_t bytes = n0 < N ? (N - 1 - n0) * ld + width : 0;
    return mx_rsrc(base + n0 * ld, bytes);
}

template <int FMT> struct Piece;
template <> struct Piece<VT_MX_FP8> {
    typedef u32x4 type;
    static __device__ __forceinline__ type load(MxRsrc r, unsigned off) {
        return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
    }
};
template <> struct Piece<VT_MX_FP4> {
    typedef u32x2 type;
    static __device__ __forceinline__ type load(MxRsrc r, unsigned off) {
        return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
    }
};

// Columns 2 p, 2 p + 1 of a piece.
template <int FMT, int P>
__device__ __forceinline__ f32x2 piece_pair(const typename Piece<FMT>::type& w, float scale) {
    if constexpr (FMT == VT_MX_FP8) return mx_pair<FMT, P & 1>(w[P >> 1], scale);
    else return mx_pair<FMT, P & 3>(w[P >> 2], scale);
}

typedef double f64x2 __attribute__((ext_vector_type(2)));

template <int... I, typename F>
__device__ __forceinline__ void each_impl(std::integer_sequence<int, I...>, F&& f) { (f(std::integral_constant<int, I>()), ...); }
template <int N, typename F>
__device__ __forceinline__ void each(F&& f) { each_impl(std::make_integer_sequence<int, N>(), f); }

// The value of the lane's partner, for sums over pairs: lane ^ M for M = 1, 2, 8; lane ^ 7 for M = 4 (as good: it too
// joins the lower and the upper half of eight).  DPP moves on the VALU, a tenth of the latency of a permutation through LDS.
template <int M>
__device__ __forceinline__ double partner(double v) {
    constexpr int ctrl = M == 1 ? 0xb1 : M == 2 ? 0x4e : M == 4 ? 0x141 : 0x128;     // quad_perm, row_half_mirror, row_ror:8
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), ctrl, 0xf, 0xf, true);
    const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), ctrl, 0xf, 0xf, true);
    return __hiloint2double(hi, lo);
}
// Lanes without bit M: the sum of a over the lane and lane ^ M; lanes with it: that of b (M = 16, 32).
template <int M>
__device__ __forceinline__ double swap_sum(double a, double b) {
    unsigned al = __double2loint(a), ah = __double2hiint(a), bl = __double2loint(b), bh = __double2hiint(b);
    if constexpr (M == 32) {
        const auto l = __builtin_amdgcn_permlane32_swap(al, bl, false, false), h = __builtin_amdgcn_permlane32_swap(ah, bh, false, false);
        return __hiloint2double(h[0], l[0]) + __hiloint2double(h[1], l[1]);
    } else {
        const auto l = __builtin_amdgcn_permlane16_swap(al, bl, false, false), h = __builtin_amdgcn_permlane16_swap(ah, bh, false, false);
        return __hiloint2double(h[0], l[0]) + __hiloint2double(h[1], l[1]);
    }
}

// d[r], r < R, summed over the T lanes of a team: the result is the sum of row lane / (T / R) of the team.  Halving: in
// every step a lane gives away the half of its rows that its partner keeps.
template <int T, int R>
__device__ __forceinline__ double team_sum(const double (&d)[R], int lane) {
    if constexpr (T == 1) {
        return d[0];
    } else if constexpr (T >= 32) {
        if constexpr (R == 1) {
            const double sum[1] = {swap_sum<T / 2>(d[0], d[0])};
            return team_sum<T / 2, 1>(sum, lane);
        } else {
            double half[R / 2];
#pragma unroll
            for (int i = 0; i < R / 2; ++i) half[i] = swap_sum<T / 2>(d[i], d[i + R / 2]);
            return team_sum<T / 2, R / 2>(half, lane);
        }
    } else if constexpr (R == 1) {
        const double sum[1] = {d[0] + partner<T / 2>(d[0])};
        return team_sum<T / 2, 1>(sum, lane);
    } else {
        double half[R / 2];
        const bool up = lane & (T / 2);
#pragma unroll
        for (int i = 0; i < R / 2; ++i) {
            const double keep = up ? d[i + R / 2] : d[i], give = up ? d[i] : d[i + R / 2];
            half[i] = keep + partner<T / 2>(give);
        }
        return team_sum<T / 2, R / 2>(half, lane);
    }
}

// Keeps the compiler from holding on to numbers that are cheaper to decode again.
template <typename W>
__device__ __forceinline__ void decode_again(W& w, float& s) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(W) / 4); ++i) {
        unsigned u = w[i];
        asm volatile("" : "+v"(u));
        w[i] = u;
    }
    asm volatile("" : "+v"(s));
}

__device__ __forceinline__ double read_lane(double v, int lane) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}

// Rows of at most 16 T columns: T lanes of a wave a row, R rows a round; the round's numbers (decoded once, as doubles)
// and the column sums in registers, v in LDS.  After the sums every lane has one row (T = R) or T / R lanes have the same, so the
// link costs a wave once, not once a row.
template <int OP, int FMT, int T, int R>
__global__ __launch_bounds__(256, 2) void k_mx_rows_wave(MxRows a) {
    static_assert(R <= T, "a lane ends with one row");
    using W = typename Piece<FMT>::type;
    constexpr int kTeams = 256 / T, kBytes = sizeof(W), kLead = T / R;
    __shared__ double sh[kCols<OP> ? 4096 : 4];
    __shared__ f64x2 vl[kDot<OP> ? 8 * T : 1];            // v's pairs, [pair][lane of the team]
    const int tid = threadIdx.x, lane = tid & 63, tt = tid & (T - 1), team = tid / T;
    const int nb = mx_blocks(a.D), pc = std::min(tt, 2 * nb - 1), own = tt / kLead;
    const int64_t stride = (int64_t)gridDim.x * kTeams * R;
    const unsigned vc = team * R * (unsigned)a.ldc + pc * kBytes, vs = team * R * (unsigned)a.lds + (pc >> 1);

    double acc[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.0;
    if constexpr (kDot<OP>) {
        for (int i = tid; i < 8 * T; i += 256) {
            const int c = 16 * (i % T) + 2 * (i / T);
            vl[i] = f64x2{c < a.D ? a.v[c] : 0.0, c + 1 < a.D ? a.v[c + 1] : 0.0};
        }
        __syncthreads();
    }
    double val = 0.0;
    W next[R];
    unsigned next_s[R];
    RowScal next_r;
    auto load = [&](int64_t n0) {
        const MxRsrc rc = rows_rsrc(a.codes, n0, a.ldc, a.N, nb * (FMT == VT_MX_FP8 ? 32 : 16)), rs = rows_rsrc(a.scales, n0, a.lds, a.N, nb);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            next[r] = Piece<FMT>::load(rc, vc + r * (unsigned)a.ldc);
            next_s[r] = __builtin_amdgcn_raw_buffer_load_b8(rs, vs + r * (unsigned)a.lds, 0, 0);
        }
        next_r = row_scal<OP>(a, std::min(n0 + team * R + own, a.N - 1));
    };
    int64_t n0 = (int64_t)blockIdx.x * kTeams * R;
    load(n0);
    const int64_t rounds = (a.N + stride - 1) / stride;
    for (int64_t it = 0; it < rounds; ++it, n0 += stride) {
        double x[R][16];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float s = mx_scale(next_s[r]);
            each<8>([&](auto p) {
                const f32x2 q = piece_pair<FMT, p>(next[r], s);
                x[r][2 * p] = (double)q[0], x[r][2 * p + 1] = (double)q[1];
            });
        }
        const RowScal scal = next_r;
        load(n0 + stride);
        double dot = 0.0;
        if constexpr (kDot<OP>) {
            double d[R];
#pragma unroll
            for (int r = 0; r < R; ++r) d[r] = 0.0;
            asm volatile("" ::: "memory");       // v is read again every round: kept, it would take 32 registers
            each<8>([&](auto p) {
                const f64x2 vv = vl[p * T + tt];
#pragma unroll
                for (int r = 0; r < R; ++r) d[r] = fma(x[r][2 * p + 1], vv[1], fma(x[r][2 * p], vv[0], d[r]));
            });
            dot = team_sum<T, R>(d, lane);
        }
        const int64_t n = n0 + team * R + own;
        double t = 0.0;
        if (n < a.N) t = mx_row_op<OP>(a, n, scal, dot, tt % kLead == 0);
        if constexpr (OP == OP_VALUE) val += tt % kLead == 0 ? t : 0.0;
        if constexpr (kCols<OP>) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                double tr;
                if constexpr (T == 64) tr = read_lane(t, r * kLead);
                else tr = __shfl(t, (lane & ~(T - 1)) + r * kLead, 64);
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[e] = fma(tr, x[r][e], acc[e]);
            }
        }
    }
    if constexpr (kCols<OP>) {
#pragma unroll
        for (int e = 0; e < 16; ++e) sh[team * 16 * T + 16 * tt + e] = acc[e];
        __syncthreads();
        for (int c = tid; c < a.D; c += 256) {
            double sum = 0.0;
#pragma unroll
            for (int g = 0; g < kTeams; ++g) sum += sh[g * 16 * T + c];
            a.part[(int64_t)blockIdx.x * a.D + c] = sum;
        }
    }
    if constexpr (OP == OP_VALUE) {
        const double w = vt_sum64(val);
        if (lane == 0) sh[tid >> 6] = w;
        __syncthreads();
        if (tid == 0) a.part[blockIdx.x] = sh[0] + sh[1] + sh[2] + sh[3];
    }
}

// Wider rows: a workgroup of T threads a row, CPT pieces a thread, R rows a round; v in LDS (read once a round for all R
// rows), the column sums in registers, one barrier a round for the dots.  v's pairs lie [piece / T][pair][piece % T] so
// that the lanes of a read are next to each other.  KEEP: the round's numbers stay in registers as doubles (16 CPT R of
// them) from the dot to the column sums; else the codes are decoded twice.
// TEAM = 0, for the operators without column sums: exactly the waves that a row needs, and more of them resident (A v
// N = 100 000, D = 5003, E2M1: 123 -> 78 us; with column sums that costs 10 to 30 %).
constexpr int few_waves(int op) { return op == OP_VALUE ? 3 : 4; }       // of a SIMD (a fourth of VALUE's would spill)
template <int OP, int FMT, int TEAM, int CPT, int R, bool KEEP>
__global__ __launch_bounds__(TEAM ? TEAM : 512, TEAM ? 2 : few_waves(OP)) void k_mx_rows_wide(MxRows a) {
    using W = typename Piece<FMT>::type;
    constexpr int kBytes = sizeof(W), kWaves = TEAM ? TEAM / 64 : 8, kLead = 64 / R;
    const int T = TEAM ? TEAM : blockDim.x;
    static_assert(kWaves <= kLead, "a row's wave sums fit its lanes");
    extern __shared__ __align__(16) double dyn[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nb = mx_blocks(a.D), pieces = 2 * nb, own = lane / kLead;
    f64x2* const vl = (f64x2*)dyn;
    double* const red = dyn + 16 * pieces;       // [2][R][kWaves]
    const int last = pieces - (CPT - 1) * T;                      // pieces of the last round of threads, >= 1
    unsigned vc[CPT], vs[CPT];
    double acc[kCols<OP> ? CPT : 1][16];
#pragma unroll
    for (int k = 0; k < CPT; ++k) {
        const int pc = std::min(tid + T * k, pieces - 1);
        vc[k] = pc * kBytes, vs[k] = pc >> 1;
        if constexpr (kCols<OP>) {
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[k][e] = 0.0;
        }
    }
    if constexpr (kDot<OP>) {
        for (int i = tid; i < 8 * pieces; i += T) {          // pair i: piece i / 8, its pair i % 8
            const int c = 2 * i, piece = i >> 3, k = piece / T, width = k < CPT - 1 ? T : last;
            vl[8 * T * k + (i & 7) * width + piece - T * k] = f64x2{c < a.D ? a.v[c] : 0.0, c + 1 < a.D ? a.v[c + 1] : 0.0};
        }
        __syncthreads();
    }
    double val = 0.0;
    int turn = 0;                // without column sums: the wave whose turn it is to finish the round's rows
    W next[R][CPT];
    unsigned next_s[R][CPT];
    RowScal next_r;
    auto load = [&](int64_t n0) {
        const MxRsrc rc = rows_rsrc(a.codes, n0, a.ldc, a.N, nb * (FMT == VT_MX_FP8 ? 32 : 16)), rs = rows_rsrc(a.scales, n0, a.lds, a.N, nb);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int k = 0; k < CPT; ++k) {
                next[r][k] = Piece<FMT>::load(rc, vc[k] + r * (unsigned)a.ldc);
                next_s[r][k] = __builtin_amdgcn_raw_buffer_load_b8(rs, vs[k] + r * (unsigned)a.lds, 0, 0);
            }
        next_r = row_scal<OP>(a, std::min(n0 + own, a.N - 1));
    };
    const int64_t stride = (int64_t)gridDim.x * R, rounds = (a.N + stride - 1) / stride;
    int64_t n0 = (int64_t)blockIdx.x * R;
    load(n0);
    for (int64_t it = 0; it < rounds; ++it, n0 += stride) {
        W w[R][CPT];
        float s[R][CPT];
        double x[KEEP ? R : 1][KEEP ? CPT : 1][16];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int k = 0; k < CPT; ++k) {
                w[r][k] = next[r][k], s[r][k] = mx_scale(next_s[r][k]);
                if constexpr (KEEP)
                    each<8>([&](auto p) {
                        const f32x2 q = piece_pair<FMT, p>(w[r][k], s[r][k]);
                        x[r][k][2 * p] = (double)q[0], x[r][k][2 * p + 1] = (double)q[1];
                    });
            }
        const RowScal scal = next_r;
        load(n0 + stride);
        double dot = 0.0;
        if constexpr (kDot<OP>) {
            double d[R];
#pragma unroll
            for (int r = 0; r < R; ++r) d[r] = 0.0;
#pragma unroll
            for (int k = 0; k < CPT; ++k) {
                const int width = k < CPT - 1 ? T : last;
                if (k < CPT - 1 || tid < width)
                    each<8>([&](auto p) {
                        const f64x2 vv = vl[8 * T * k + p * width + tid];
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            if constexpr (KEEP) {
                                d[r] = fma(x[r][k][2 * p], vv[0], d[r]);
                                d[r] = fma(x[r][k][2 * p + 1], vv[1], d[r]);
                            } else {
                                const f32x2 q = piece_pair<FMT, p>(w[r][k], s[r][k]);
                                d[r] = fma((double)q[0], vv[0], d[r]);
                                d[r] = fma((double)q[1], vv[1], d[r]);
                            }
                        }
                    });
            }
            // this wave's sum of row `own`, then the waves' sums: every lane of the row's group adds them all
            const double mine = team_sum<64, R>(d, lane);
            double* const slot = red + (it & 1) * kWaves * R + own * kWaves;
            if (lane % kLead == 0) slot[wave] = mine;
            vt_lds_barrier();
            if (kCols<OP> || wave == turn) {
                const double part[1] = {TEAM || (lane & (kWaves - 1)) < T / 64 ? slot[lane & (kWaves - 1)] : 0.0};
                dot = team_sum<kWaves, 1>(part, lane);
            }
        }
        const int64_t n = n0 + own;
        double t = 0.0;
        if (n < a.N && (kCols<OP> || wave == turn)) t = mx_row_op<OP>(a, n, scal, dot, (!kCols<OP> || wave == 0) && lane % kLead == 0);
        if constexpr (OP == OP_VALUE) val += lane % kLead == 0 ? t : 0.0;
        if constexpr (!kCols<OP>) turn = turn + 1 < T / 64 ? turn + 1 : 0;
        if constexpr (kCols<OP>) {
            double tr[R];
#pragma unroll
            for (int r = 0; r < R; ++r) tr[r] = read_lane(t, r * kLead);
            if constexpr (kDot<OP> && !KEEP) {
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int k = 0; k < CPT; ++k) decode_again(w[r][k], s[r][k]);
            }
#pragma unroll
            for (int k = 0; k < CPT; ++k)
                if (k < CPT - 1 || tid < last)
                    each<8>([&](auto p) {
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            double x0, x1;
                            if constexpr (KEEP) {
                                x0 = x[r][k][2 * p], x1 = x[r][k][2 * p + 1];
                            } else {
                                const f32x2 q = piece_pair<FMT, p>(w[r][k], s[r][k]);
                                x0 = (double)q[0], x1 = (double)q[1];
                            }
                            acc[k][2 * p] = fma(tr[r], x0, acc[k][2 * p]);
                            acc[k][2 * p + 1] = fma(tr[r], x1, acc[k][2 * p + 1]);
                        }
                    });
        }
    }
    if constexpr (kCols<OP>) {
        // through LDS, so that the slab is written in order (a lane's own 16 columns are 128 bytes apart); the pairs of a
        // piece are turned by its number: other banks for every lane
        __syncthreads();
#pragma unroll
        for (int k = 0; k < CPT; ++k) {
            const int piece = tid + T * k;
            if (piece < pieces)
#pragma unroll
                for (int p = 0; p < 8; ++p) vl[8 * piece + (p ^ (piece & 7))] = f64x2{acc[k][2 * p], acc[k][2 * p + 1]};
        }
        __syncthreads();
        double* out = a.part + (int64_t)blockIdx.x * a.D;
        for (int c = tid; c < a.D; c += T) {
            const int piece = c >> 4;
            out[c] = vl[8 * piece + ((c >> 1 & 7) ^ (piece & 7))][c & 1];
        }
    }
    if constexpr (OP == OP_VALUE) {
        val = vt_sum64(val);
        __syncthreads();
        if (lane == 0) red[wave] = val;
        __syncthreads();
        if (tid == 0) {
            for (int i = 1; i < T / 64; ++i) val += red[i];
            a.part[blockIdx.x] = val;
        }
    }
}

// ---- two passes: rows too wide for one workgroup's registers and LDS ----------------------------------------------------
// One wave per row takes the dots and leaves t_n in the workspace; then every thread owns eight columns and walks a slab.
// The dots are far from their bytes: eight bytes of codes a load, v from L2 for every row, a row a wave, nothing fetched
// ahead.  At 50 000 x 20 353 HVP 1.30 ms (E4M3; E2M1 1.23), gradient 2.03, link 1.71, A v 0.98, A^T u 0.32, where one pass
// takes 0.50, 0.54, 0.46, 0.37 and 0.36 for twice the numbers (10^5 x 20 000).

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
            const double t = mx_row_op<OP>(a, n, row_scal<OP>(a, n), dot, true);
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

// out[c] = sum_p part[p][c] + beta[c] bvec[c] from column c0 on, 32 columns a workgroup, 32 groups each summing every 32nd
// slab.
__global__ __launch_bounds__(1024) void k_mx_finalize(const double* part, int P, int D, int c0, const double* beta,
                                                      const double* bvec, double beta_scalar, double* out) {
    __shared__ double sh[32][33];
    const int cl = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int c = c0 + blockIdx.x * 32 + cl;
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

// Which kernel takes a width: 2 to 64 lanes of a wave (D <= 1024), a workgroup of 128, 256 or 512 threads with one
// piece each (D <= 8192: fewer threads with more pieces were slower, D = 4096: 112 us in 256 x 1, 143 in 128 x 2), 512 with
// two or three, else two passes.  v and the sums of a round share 160 KB of LDS: D <= 20352 in one pass.
constexpr int kOnePassPieces = (160 * 1024 - 1024) / 128;

struct RowsPlan {
    int lanes, threads, cpt;      // lanes > 0: wave kernel; else threads > 0: wide kernel
    int grid;                     // = slabs of partial sums
};

// Rows a round.  One piece a thread: 4, kept as doubles (128 registers).  Two pieces: 4, decoded twice (N = 50 000,
// D = 16 384: 206 us; 2 kept rows 222).  Three pieces: 4 fit for E2M1; for E4M3 2 (N = 100 000, D = 20 000: about 490 us; 4
// spill: 985).  Of one piece, two rows a round with more waves resident: 20 to 40 % longer, the sums, the barrier and the link
// are paid once a round.
constexpr int wave_rows(int lanes) { return lanes < 4 ? lanes : 4; }
constexpr int wide_rows(int cpt, int format) { return cpt == 3 && format == VT_MX_FP8 ? 2 : 4; }

int col_tiles(int D) { return (D + 2047) / 2048; }

// `op`: an operator with column sums unless said otherwise (those without may have more workgroups, and need no slabs)
RowsPlan rows_plan(int format, int64_t N, int D, int64_t ldc, int64_t lds, int op = OP_GRAD) {
    const int pieces = 2 * mx_blocks(D), cu = vt_num_cu();
    RowsPlan p{0, 0, 0, 0};
    int64_t rounds;               // of all workgroups together
    int most;                     // workgroups that are resident together
    // (offsets inside a round are 32 bits: 256 rows at most)
    const bool far = ldc >= 1 << 22 || lds >= 1 << 22;
    if (pieces <= 64 && !far) {
        for (p.lanes = 2; p.lanes < pieces;) p.lanes *= 2;
        const int rows = 256 / p.lanes * wave_rows(p.lanes);
        rounds = (N + rows - 1) / rows, most = 2 * cu;
    } else if (pieces <= kOnePassPieces && !far) {
        p.threads = pieces <= 128 ? 128 : pieces <= 256 ? 256 : 512;
        p.cpt = (pieces + p.threads - 1) / p.threads;
        const int rows = wide_rows(p.cpt, format);
        rounds = (N + rows - 1) / rows;
        int waves = 8;                // of a CU
        if (p.cpt == 1 && (op == OP_LINK || op == OP_VALUE || op == OP_GEMV)) p.threads = (pieces + 63) / 64 * 64, waves = 4 * few_waves(op);
        most = cu * std::max(1, std::min(64 * waves / p.threads, (160 * 1024) / (128 * pieces + 1024)));
    } else {
        p.grid = (int)std::max<int64_t>(1, std::min<int64_t>(N, std::max(1, 4 * cu / col_tiles(D))));
        return p;
    }
    // the same number of rounds for every workgroup
    const int64_t each = std::max<int64_t>(1, (rounds + most - 1) / most);
    p.grid = (int)std::max<int64_t>(1, (rounds + each - 1) / each);
    return p;
}

template <int OP, int FMT, int T>
void launch_wave(const MxRows& a, int grid, hipStream_t st) {
    hipLaunchKernelGGL((k_mx_rows_wave<OP, FMT, T, wave_rows(T)>), dim3(grid), dim3(256), 0, st, a);
}

template <int OP, int FMT, int T, int CPT>
int launch_wide(const MxRows& a, const RowsPlan& p, hipStream_t st) {
    constexpr bool keep = kCols<OP> && CPT == 1;
    constexpr int R = wide_rows(CPT, FMT);
    const size_t lds = 128 * (size_t)(2 * mx_blocks(a.D)) + 2 * (T ? T / 64 : 8) * R * sizeof(double);
    static VtLdsAttr attr;
    if (vt_allow_big_lds((const void*)k_mx_rows_wide<OP, FMT, T, CPT, R, keep>, attr, 160 * 1024) != VT_OK) return VT_ERR_HIP;
    hipLaunchKernelGGL((k_mx_rows_wide<OP, FMT, T, CPT, R, keep>), dim3(p.grid), dim3(p.threads), lds, st, a);
    return VT_OK;
}

template <int OP, int FMT>
int run(MxRows a, const RowsPlan& p, hipStream_t st) {
    if (p.lanes > 0) {
        switch (p.lanes) {
            case 2: launch_wave<OP, FMT, 2>(a, p.grid, st); break;
            case 4: launch_wave<OP, FMT, 4>(a, p.grid, st); break;
            case 8: launch_wave<OP, FMT, 8>(a, p.grid, st); break;
            case 16: launch_wave<OP, FMT, 16>(a, p.grid, st); break;
            case 32: launch_wave<OP, FMT, 32>(a, p.grid, st); break;
            default: launch_wave<OP, FMT, 64>(a, p.grid, st); break;
        }
        return vt_launch_status();
    }
    if (p.threads > 0) {
        int rc;
        if (p.cpt == 3) rc = launch_wide<OP, FMT, 512, 3>(a, p, st);
        else if (p.cpt == 2) rc = launch_wide<OP, FMT, 512, 2>(a, p, st);
        else if constexpr (!kCols<OP>) rc = launch_wide<OP, FMT, 0, 1>(a, p, st);
        else rc = p.threads == 128   ? launch_wide<OP, FMT, 128, 1>(a, p, st)
                  : p.threads == 256 ? launch_wide<OP, FMT, 256, 1>(a, p, st)
                                     : launch_wide<OP, FMT, 512, 1>(a, p, st);
        return rc != VT_OK ? rc : vt_launch_status();
    }
    const int grid = (int)std::min<int64_t>((a.N + 3) / 4, 8 * (int64_t)vt_num_cu());
    hipLaunchKernelGGL((k_mx_dots<OP, FMT>), dim3(grid), dim3(256), 0, st, a);
    if constexpr (kCols<OP>) hipLaunchKernelGGL((k_mx_columns<FMT>), dim3(col_tiles(a.D), p.grid), dim3(256), 0, st, a);
    return vt_launch_status();
}

template <int OP>
int run(int format, const MxRows& a, const RowsPlan& p, hipStream_t st) {
    return format == VT_MX_FP8 ? run<OP, VT_MX_FP8>(a, p, st) : run<OP, VT_MX_FP4>(a, p, st);
}

int finalize(const double* part, int P, int D, const double* beta, const double* bvec, double beta_scalar, double* out,
             hipStream_t st) {
    // (a launch holds fewer than 2^32 threads: 2^26 columns are 2^31 of them)
    constexpr int kPanel = 1 << 26;
    for (int c0 = 0; c0 < D; c0 += kPanel)
        hipLaunchKernelGGL(k_mx_finalize, dim3((std::min(D - c0, kPanel) + 31) / 32), dim3(1024), 0, st, part, P, D, c0, beta, bvec,
                           beta_scalar, out);
    return vt_launch_status();
}

// Workspace: slabs of partial column sums (VALUE: one number a workgroup, or a row), and t for the two passes.
// Enough for both formats and any strides.
size_t ws_doubles(int64_t N, int D) {
    const int g = std::max(rows_plan(VT_MX_FP8, N, D, 0, 0).grid, rows_plan(VT_MX_FP4, N, D, 0, 0).grid);
    return std::max((size_t)g * D, (size_t)rows_plan(VT_MX_FP8, N, D, 1 << 30, 0).grid * D + (size_t)N);
}

MxRows rows_of(const void* codes, int64_t ldc, const void* scales, int64_t lds, int64_t N, int D, void* ws, const RowsPlan& p) {
    MxRows a{};
    a.codes = (const uint8_t*)codes;
    a.scales = (const uint8_t*)scales;
    a.ldc = ldc, a.lds = lds, a.N = N, a.D = D;
    a.part = (double*)ws;
    a.t = a.part + (size_t)p.grid * D;
    return a;
}

}  // namespace

extern "C" size_t vt_mx_rows_workspace_bytes(int64_t N, int D) {
    if (N < 0 || D < 1) return 0;
    return ws_doubles(N, D) * sizeof(double);
}

#define VT_MX_ROWS_PROLOGUE(op)                                                              \
    if (!mx_rows_ok(format, codes, ldc, scales, lds, N, D)) return VT_ERR_BAD_ARG;           \
    if (!ws || ws_bytes < vt_mx_rows_workspace_bytes(N, D)) return VT_ERR_WORKSPACE;         \
    hipStream_t st = (hipStream_t)stream;                                                    \
    const RowsPlan p = rows_plan(format, N, D, ldc, lds, op);                                \
    MxRows a = rows_of(codes, ldc, scales, lds, N, D, ws, p);

extern "C" int vt_mx_glm_link(int family, int format, const void* codes, int64_t ldc, const void* scales, int64_t lds,
                              const double* theta, const double* y, const double* w, const double* offset, double scale,
                              int64_t N, int D, double* z, double* r, double* d, void* ws, size_t ws_bytes, void* stream) {
    VT_MX_ROWS_PROLOGUE(OP_LINK)
    if (family < 0 || family > 2) return VT_ERR_BAD_ARG;
    if (N == 0) return VT_OK;
    if (!theta || !y || !w) return VT_ERR_BAD_ARG;
    a.v = theta, a.y = y, a.w = w, a.offset = offset, a.scale = scale, a.family = family;
    a.z = z, a.r = r, a.d = d, a.t = nullptr;
    return run<OP_LINK>(format, a, p, st);
}

extern "C" int vt_mx_glm_grad(int family, int format, const void* codes, int64_t ldc, const void* scales, int64_t lds,
                              const double* theta, const double* y, const double* w, const double* offset, double scale,
                              const double* prior, int64_t N, int D, double* g, double* r, double* d, void* ws,
                              size_t ws_bytes, void* stream) {
    VT_MX_ROWS_PROLOGUE(OP_GRAD)
    if (family < 0 || family > 2 || !theta || !g || (N > 0 && (!y || !w))) return VT_ERR_BAD_ARG;
    a.v = theta, a.y = y, a.w = w, a.offset = offset, a.scale = scale, a.family = family, a.r = r, a.d = d;
    if (N > 0)
        if (int rc = run<OP_GRAD>(format, a, p, st)) return rc;
    return finalize(a.part, N > 0 ? p.grid : 0, D, prior, prior ? theta : nullptr, 0.0, g, st);
}

extern "C" int vt_mx_glm_value(int family, int format, const void* codes, int64_t ldc, const void* scales, int64_t lds,
                               const double* theta, const double* y, const double* w, const double* offset, double scale,
                               int64_t N, int D, double* value, void* ws, size_t ws_bytes, void* stream) {
    VT_MX_ROWS_PROLOGUE(OP_VALUE)
    if (family < 0 || family > 2 || !theta || !value || (N > 0 && (!y || !w))) return VT_ERR_BAD_ARG;
    a.v = theta, a.y = y, a.w = w, a.offset = offset, a.family = family;
    if (N > 0)
        if (int rc = run<OP_VALUE>(format, a, p, st)) return rc;
    const bool one_pass = p.lanes > 0 || p.threads > 0;
    hipLaunchKernelGGL(k_mx_sum, dim3(1), dim3(1024), 0, st, one_pass ? a.part : a.t, one_pass && N > 0 ? p.grid : N, scale, value);
    return vt_launch_status();
}

extern "C" int vt_mx_glm_hvp(int format, const void* codes, int64_t ldc, const void* scales, int64_t lds, const double* d,
                             const double* prior, double prior_scalar, const double* v, int64_t N, int D, double* out,
                             void* ws, size_t ws_bytes, void* stream) {
    VT_MX_ROWS_PROLOGUE(OP_HVP)
    if (!v || !out || (N > 0 && !d)) return VT_ERR_BAD_ARG;
    a.v = v, a.y = d;
    if (N > 0)
        if (int rc = run<OP_HVP>(format, a, p, st)) return rc;
    return finalize(a.part, N > 0 ? p.grid : 0, D, prior, prior || prior_scalar != 0.0 ? v : nullptr, prior_scalar, out, st);
}

extern "C" int vt_mx_gemv(int format, const void* codes, int64_t ldc, const void* scales, int64_t lds, const double* v,
                          int64_t N, int D, double* out, void* ws, size_t ws_bytes, void* stream) {
    VT_MX_ROWS_PROLOGUE(OP_GEMV)
    if (N == 0) return VT_OK;
    if (!v || !out) return VT_ERR_BAD_ARG;
    a.v = v, a.z = out, a.t = nullptr;
    return run<OP_GEMV>(format, a, p, st);
}

extern "C" int vt_mx_gemv_t(int format, const void* codes, int64_t ldc, const void* scales, int64_t lds, const double* u1,
                            const double* u2, int64_t N, int D, double* out, void* ws, size_t ws_bytes, void* stream) {
    VT_MX_ROWS_PROLOGUE(OP_GEMVT)
    if (!out || (N > 0 && !u1)) return VT_ERR_BAD_ARG;
    a.y = u1, a.w = u2;
    if (N > 0)
        if (int rc = run<OP_GEMVT>(format, a, p, st)) return rc;
    return finalize(a.part, N > 0 ? p.grid : 0, D, nullptr, nullptr, 0.0, out, st);
}
