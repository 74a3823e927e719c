// Compact rows: microscaled E4M3 / E2M1 blocks of 32 columns with one E8M0 scale byte (see include/vittles_hip.h).
// The gfx950 conversions take the scale with them: v_cvt_scalef32_pk_f32_fp8 / _fp4 return code * 2^(s - 127) for the
// scale 2^(s - 127) given as float bits s << 23, for every s: s = 0 is 2^-127 and s = 255 gives NaN, whatever the code
// (all 2 x 256 x 256 cases were compared with the definition).
#pragma once
#include "vt_common.h"

constexpr int kMxBlock = 32;
constexpr int kMxF32One = 0x3f800000;

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// 16 bytes at an element's own alignment (2, 4 or 8): the gfx950 ABI runs with unaligned wide accesses allowed.
template <int ALIGN> struct Unaligned16;
template <> struct Unaligned16<2> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Unaligned16<4> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Unaligned16<8> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(8))); };

__host__ __device__ __forceinline__ constexpr int mx_blocks(int D) { return D / kMxBlock + (D % kMxBlock != 0); }
__host__ __device__ __forceinline__ constexpr int mx_block_bytes(int format) { return format == VT_MX_FP8 ? 32 : 16; }
// codes in one 32-bit word
template <int FMT> constexpr int kMxPerWord = FMT == VT_MX_FP8 ? 4 : 8;

__device__ __forceinline__ float mx_scale(unsigned s) { return __builtin_bit_cast(float, s << 23); }

// Two values of a word: P-th pair of codes.
template <int FMT, int P>
__device__ __forceinline__ f32x2 mx_pair(unsigned word, float scale) {
    if constexpr (FMT == VT_MX_FP8) return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, scale, P != 0);
    else return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, P);
}
template <int FMT, int P>
__device__ __forceinline__ bf16x2 mx_pair_bf16(unsigned word, float scale) {
    if constexpr (FMT == VT_MX_FP8) return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, P != 0);
    else return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, P);
}

// All values of a word, in column order.
template <int FMT>
__device__ __forceinline__ void mx_word(unsigned word, float scale, float (&v)[kMxPerWord<FMT>]) {
    f32x2 p = mx_pair<FMT, 0>(word, scale);
    v[0] = p[0], v[1] = p[1];
    p = mx_pair<FMT, 1>(word, scale);
    v[2] = p[0], v[3] = p[1];
    if constexpr (FMT == VT_MX_FP4) {
        p = mx_pair<FMT, 2>(word, scale);
        v[4] = p[0], v[5] = p[1];
        p = mx_pair<FMT, 3>(word, scale);
        v[6] = p[0], v[7] = p[1];
    }
}

// A buffer descriptor of `bytes` from p on: loads past it give 0, stores past it are dropped.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_rsrc(const void* p, int64_t bytes) {
    const uint64_t b = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)b), hi = __builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
    const uint32_t n = bytes <= 0 ? 0 : (uint32_t)std::min<int64_t>(bytes, 0x7fffffff);
    return __builtin_amdgcn_make_buffer_rsrc((void*)(((uint64_t)hi << 32) | lo), 0, __builtin_amdgcn_readfirstlane(n), 0x00020000);
}
constexpr unsigned kNowhere = 0x80000000u;       // an offset past every descriptor

// Host-side check of a compact matrix, shared by every entry point.
inline bool mx_rows_ok(int format, const void* codes, int64_t ldc, const void* scales, int64_t lds, int64_t N, int D) {
    if ((format != VT_MX_FP4 && format != VT_MX_FP8) || N < 0 || D < 1 || D > (1 << 30)) return false;
    if (N == 0) return true;
    const int64_t nb = mx_blocks(D);
    return codes && scales && (uintptr_t)codes % 16 == 0 && ldc % 16 == 0 && ldc >= nb * mx_block_bytes(format) && lds >= nb;
}
