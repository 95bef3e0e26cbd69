// Pieces shared by the attention kernels that work on whole tiles of fp16 tokens (prompt attention, wide trees): the score
// modifiers, the LDS layout of a tile and the two matrix products on it.
//
// Everything is computed transposed: S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16_f16.  A lane then owns one
// query row (column lane & 31 of the accumulators) and half of a tile's tokens, so the softmax of a row is arithmetic
// inside a lane plus one exchange with lane ^ 32, and the probabilities leave the first product in the very lanes in which
// the second one wants them: accumulator register r of half h holds token 8 (r / 4) + 4 h + r % 4, and since a contraction
// index may be numbered at will, the second product takes its tokens in that order.
#pragma once

#include "akv_common.h"

namespace akv {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4v __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kNegInf = -__builtin_inff();

__device__ __forceinline__ f16x8 as_f16x8(u32x4 w) { return __builtin_bit_cast(f16x8, w); }
__device__ __forceinline__ u32 pack_f16(float a, float b) {   // round to nearest even
    const f32x2 f = {a, b};
    return __builtin_bit_cast(u32, __builtin_convertvector(f, f16x2v));
}

// Maximum / sum over a lane and the lane 32 away (the other half of the wave), the same in both.
__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// tanh in 32 bits.  Near zero a series keeps the relative error at rounding level, where 1 - 2 / (exp(2 y) + 1) would
// lose it to cancellation; a capped score is cap * tanh, so what is lost here is multiplied by the cap.
// |y| < 1/2: odd polynomial through y^13 (Taylor coefficients; the first one left out is below 2e-8 relative there).
__device__ __forceinline__ float tanh_f32(float y) {
    const float e = __builtin_amdgcn_exp2f(y * (2.f * kLog2e));
    const float far = 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
    const float z = y * y;
    float p = fmaf(z, 21844.f / 6081075.f, -1382.f / 155925.f);
    p = fmaf(z, p, 62.f / 2835.f);
    p = fmaf(z, p, -17.f / 315.f);
    p = fmaf(z, p, 2.f / 15.f);
    p = fmaf(z, p, -1.f / 3.f);
    const float near = fmaf(y * z, p, y);
    return fabsf(y) < 0.4f ? near : far;
}

// What a raw product q . k goes through, in units of log2 e (so that the softmax takes 2^x):
//   no cap: x = raw * c0;  cap: x = c1 * tanh(raw * c0);  then x -= slope * |distance|.
struct ScoreForm {
    float c0, c1;
};
__host__ __device__ __forceinline__ ScoreForm score_form(float scale, float cap) {
    ScoreForm f;
    f.c0 = cap > 0.f ? scale / cap : scale * kLog2e;
    f.c1 = cap * kLog2e;
    return f;
}
template <bool CAP>
__device__ __forceinline__ float modified(float raw, const ScoreForm &f) {
    if constexpr (CAP) return f.c1 * tanh_f32(raw * f.c0);
    return raw * f.c0;
}

// ---- a tile of BN tokens x D channels in LDS, fp16, token-major ------------------------------------------------------------
// 16-byte chunk c of row r lies at chunk c ^ swizzle(r): the lanes of one LDS access then spread over all banks, both for
// the K operand (8 consecutive rows, one chunk) and for the transposed V operand (4 consecutive rows, 64 bytes each).
template <int D>
__device__ __forceinline__ int tile_swizzle(int row) {
    if constexpr (D == 64) return ((row >> 1) & 1) << 2 | ((row >> 2) & 3);   // two rows per 256 bytes of banks
    return (row & 3) << 2 | ((row >> 2) & 3);
}
template <int D>
__device__ __forceinline__ int tile_byte(int row, int chunk) {
    return row * (D * 2) + ((chunk ^ tile_swizzle<D>(row)) << 4);
}

typedef __attribute__((address_space(3))) const uint8_t *lds_ptr;
typedef __attribute__((address_space(3))) s16x4 *lds_s16x4_ptr;

// S^T of one tile: acc[tb] += K rows 32 tb .. 32 tb + 31 times the wave's 32 query rows.  qf[ks]: channels 16 ks + 8 half ..
template <int D, int BN>
__device__ __forceinline__ void tile_scores(f32x16 (&acc)[BN / 32], const uint8_t *k_tile, const f16x8 (&qf)[D / 16]) {
    const int lane = threadIdx.x & 63, row = lane & 31, half = lane >> 5;
#pragma unroll
    for (int tb = 0; tb < BN / 32; ++tb)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[tb][r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        const int off = tile_byte<D>(row, 2 * ks + half);
#pragma unroll
        for (int tb = 0; tb < BN / 32; ++tb) {
            const f16x8 a = *reinterpret_cast<const f16x8 *>(k_tile + off + tb * 32 * D * 2);
            acc[tb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qf[ks], acc[tb], 0, 0, 0);
        }
    }
}

// The V^T operand for channels 32 cb .. + 31 and the 16 tokens whose probabilities are registers 8 s .. 8 s + 7 of block tb:
// two transposing reads of four tokens each (lane group of 16: row r from the lanes 4 r .. 4 r + 3, column = lane).
template <int D>
__device__ __forceinline__ f16x8 tile_v_operand(const uint8_t *v_tile, int cb, int tb, int s) {
    const int lane = threadIdx.x & 63;
    const int row = tb * 32 + s * 16 + 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int chunk = cb * 4 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), in_chunk = (lane & 1) * 8;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(v_tile + tile_byte<D>(row, chunk) + in_chunk));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(v_tile + tile_byte<D>(row + 8, chunk) + in_chunk));
    return __builtin_bit_cast(f16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Any value of the operand infinite or not a number?
__device__ __forceinline__ bool any_nonfinite(f16x8 v) {
    const u32x4 w = __builtin_bit_cast(u32x4, v);
    u32 bad = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const u32 e = w[i] & 0x7C007C00u;
        bad |= ((e & 0xFFFFu) == 0x7C00u || (e >> 16) == 0x7C00u) ? 1u : 0u;
    }
    return bad != 0;
}
__device__ __forceinline__ f16x8 zero_nonfinite(f16x8 v) {
    u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        u32 x = w[i];
        if ((x & 0x7C00u) == 0x7C00u) x &= 0xFFFF0000u;
        if ((x & 0x7C000000u) == 0x7C000000u) x &= 0x0000FFFFu;
        w[i] = x;
    }
    return __builtin_bit_cast(f16x8, w);
}

// O^T += V^T P^T for one tile.  p[tb][s]: the probabilities as packed above.
template <int D, int BN>
__device__ __forceinline__ void tile_output(f32x16 (&o)[D / 32], const uint8_t *v_tile, const f16x8 (&p)[BN / 32][2]) {
#pragma unroll
    for (int tb = 0; tb < BN / 32; ++tb)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int cb = 0; cb < D / 32; ++cb)
                o[cb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(tile_v_operand<D>(v_tile, cb, tb, s), p[tb][s], o[cb], 0, 0, 0);
}

// The same where some rows do not see some tokens of the tile.  A hidden token's probability is zero, but zero times an
// infinite or undefined value is undefined: such values are taken out of the product and added to the rows that do see
// their token (which makes them infinite or undefined, as the formula does).  visible(t): does this lane's row see token t
// of the tile?  Tiles without such values, the rule, pay one pass over the operands.
template <int D, int BN, typename Visible>
__device__ __forceinline__ void tile_output_masked(f32x16 (&o)[D / 32], const uint8_t *v_tile, const f16x8 (&p)[BN / 32][2],
                                                   Visible visible) {
    bool bad = false;
#pragma unroll
    for (int tb = 0; tb < BN / 32; ++tb)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int cb = 0; cb < D / 32; ++cb) {
                f16x8 a = tile_v_operand<D>(v_tile, cb, tb, s);
                if (any_nonfinite(a)) {
                    bad = true;
                    a = zero_nonfinite(a);
                }
                o[cb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, p[tb][s], o[cb], 0, 0, 0);
            }
    if (!__any(bad)) return;
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll 1
    for (int t = 0; t < BN; ++t) {
        if (!visible(t)) continue;
#pragma unroll
        for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int ch = cb * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
                const _Float16 v = *reinterpret_cast<const _Float16 *>(v_tile + tile_byte<D>(t, ch >> 3) + (ch & 7) * 2);
                const float f = (float)v;
                if (!(fabsf(f) < __builtin_inff())) o[cb][r] += f;
            }
    }
}

// Running softmax state of the wave's 32 rows (a row's two lanes hold the same m and their own part of l).
struct RowState {
    float m = kNegInf;   // maximum the sums are relative to (units of log2 e)
    float l = 0.f;       // this lane's share of the sum
};

// x[tb][r] (units of log2 e, -inf where hidden) -> packed probabilities 2^(x - m); rescales l and o when the maximum grew
// by more than 8 (a probability is then at most 2^8: far from fp16's limit, and sums keep their relative precision), which
// after the first tiles of a row is rare.
template <int D, int BN>
__device__ __forceinline__ void tile_softmax(f32x16 (&x)[BN / 32], RowState &st, f32x16 (&o)[D / 32], f16x8 (&p)[BN / 32][2]) {
    float mx = x[0][0];
#pragma unroll
    for (int tb = 0; tb < BN / 32; ++tb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, x[tb][r]);
    mx = halves_max(mx);
    if (__any(mx > st.m + 8.f)) {     // (m = -inf: any finite maximum)
        const float m_new = fmaxf(st.m, mx);
        const float alpha = st.m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(st.m - m_new);
        st.m = m_new;
        st.l *= alpha;
#pragma unroll
        for (int cb = 0; cb < D / 32; ++cb)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[cb][r] *= alpha;
    }
    const float m = st.m == kNegInf ? 0.f : st.m;
    float sum = 0.f;
#pragma unroll
    for (int tb = 0; tb < BN / 32; ++tb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[tb][r] = __builtin_amdgcn_exp2f(x[tb][r] - m);
            sum += x[tb][r];
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_f16(x[tb][8 * s + 2 * i], x[tb][8 * s + 2 * i + 1]);
            p[tb][s] = as_f16x8(w);
        }
    }
    st.l += sum;
}

int check_layer(const akv_cache_layer *c, const char *what);   // of a cache layer's descriptor: AKV_OK or the error

}  // namespace akv
