// Eviction from the split-plane cache by accumulated attention weight.
//
// Per sequence and KV head a weight for each cached token is kept in 32 bits: the attention probability it received, summed over
// the query heads of the group and over steps (accumulate_weights: the probabilities a decode step leaves; attention_weights: a
// prompt's rows).  evict keeps `keep` of the tokens that are in the planes -- the first ones (sinks), the newest (recent), then the
// largest weights, ties to the lowest index -- and moves them to the front in their order; the rest buffer follows unchanged.
#include "akv_attention.h"

namespace akv {

constexpr int kUnit = 64;       // tokens enter and leave the planes in units of the rest buffer's length

typedef float f32x4_dword __attribute__((ext_vector_type(4), aligned(4)));   // 16 bytes at any dword

// ---- accumulate_weights ------------------------------------------------------------------------------------------------------------------
// out[b, h, t] = decay * in[b, h, t] + sum over the group's heads of probs[b, g, t], t < length.  Bound by its bytes (2 per
// probability, 8 per weight): a thread takes 8 tokens, 16 bytes of each head's row.
__global__ __launch_bounds__(256) void accumulate_weights_kernel(const float *in, const uint8_t *__restrict__ probs, const int *__restrict__ lens, float *out,
                                                                 int G, int Hkv, int row_stride, int64_t in_b, int64_t in_h, int64_t out_b, int64_t out_h,
                                                                 int capacity, float decay) {
    const int b = blockIdx.z, h = blockIdx.y, t0 = (blockIdx.x * 256 + threadIdx.x) * 8;
    const int n = max(0, min(lens[b], capacity));
    if (t0 >= n) return;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const uint8_t *p = probs + (((int64_t)b * Hkv + h) * G * row_stride + t0) * 2;
    for (int g = 0; g < G; ++g) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(p + (int64_t)g * row_stride * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[2 * i] += lo_half_to_float(w[i]);
            s[2 * i + 1] += hi_half_to_float(w[i]);
        }
    }
    const float *ip = in + b * in_b + h * in_h + t0;
    float *op = out + b * out_b + h * out_h + t0;
    if (t0 + 8 <= n) {
        const f32x4_dword x = *reinterpret_cast<const f32x4_dword *>(ip), y = *reinterpret_cast<const f32x4_dword *>(ip + 4);
        f32x4_dword u, v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = fmaf(x[i], decay, s[i]);
            v[i] = fmaf(y[i], decay, s[4 + i]);
        }
        *reinterpret_cast<f32x4_dword *>(op) = u;
        *reinterpret_cast<f32x4_dword *>(op + 4) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (t0 + i < n) op[i] = fmaf(ip[i], decay, s[i]);
    }
}

// ---- evict: which tokens stay --------------------------------------------------------------------------------------------------------------
// Weights as integers in the same order; not-a-number below everything, both zeros alike.
__device__ __forceinline__ u32 weight_key(float f) {
    if (f != f) return 0u;
    const u32 u = __float_as_uint(f == 0.f ? 0.f : f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Choice {
    int n, flushed, have, lo, hi, need;     // cached, in the planes, kept of these; candidates [lo, hi), `need` of them are chosen
};
__device__ __forceinline__ Choice make_choice(int n, int keep, int sinks, int recent) {
    Choice c;
    c.n = n;
    c.flushed = n / kUnit * kUnit;
    c.have = min(keep, c.flushed);
    c.lo = min(sinks, c.flushed);
    c.hi = max(c.lo, min(c.flushed, max(0, n - recent)));
    c.need = c.have - (c.lo + c.flushed - c.hi);
    return c;
}

// One workgroup of 1024 per (sequence, KV head).  The `need`-th largest key is found by its digits, 11 + 11 + 10 bits, each from
// a histogram in LDS; then every wave writes the chosen tokens of its stretch of the row behind those of the waves before it.
__global__ __launch_bounds__(1024) void evict_select_kernel(const float *__restrict__ weights, int64_t w_b, int64_t w_h, const int *__restrict__ lens,
                                                            int *__restrict__ kept, int *__restrict__ old_lens, int Hkv, int capacity, int keep, int sinks,
                                                            int recent) {
    __shared__ u32 hist[2048];
    __shared__ int wave_tot[16], wave_eq[16];
    __shared__ u32 digit_s;
    __shared__ int above_s;
    const int h = blockIdx.x % Hkv, b = blockIdx.x / Hkv, tid = threadIdx.x, lane = tid & 63, wave = wave_index();
    const Choice c = make_choice(max(0, min(lens[b], capacity)), keep, sinks, recent);
    int *out = kept + (int64_t)blockIdx.x * keep;
    if (h == 0 && tid == 0) old_lens[b] = c.n;
    for (int i = c.have + tid; i < keep; i += 1024) out[i] = -1;
    if (c.flushed <= keep) {
        for (int i = tid; i < c.have; i += 1024) out[i] = i;
        return;
    }
    const float *w = weights + b * w_b + h * w_h;
    u32 prefix = 0;             // digits found so far
    int need = c.need;          // still to be taken among the keys that share them
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < 2048; i += 1024) hist[i] = 0;
        __syncthreads();
        for (int j = c.lo + tid; j < c.hi; j += 1024) {
            const u32 k = weight_key(w[j]);
            if (pass == 0 || (k >> (shift + bits)) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
        }
        __syncthreads();
        // thread i holds bins 2046 - 2 i and 2047 - 2 i: counts from the top
        const int top = 2047 - 2 * tid;
        const int c1 = (int)hist[top], c0 = (int)hist[top - 1];
        int inc = c0 + c1;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(inc, d);
            if (lane >= d) inc += o;
        }
        if (lane == 63) wave_tot[wave] = inc;
        __syncthreads();
        int before = inc - c0 - c1;
        for (int k = 0; k < wave; ++k) before += wave_tot[k];
        if (before < need && need <= before + c1) {
            digit_s = (u32)top;
            above_s = before;
        } else if (before + c1 < need && need <= before + c1 + c0) {
            digit_s = (u32)(top - 1);
            above_s = before + c1;
        }
        __syncthreads();
        if (need > 0) {
            prefix = (prefix << bits) | digit_s;
            need -= above_s;
        }
        __syncthreads();
    }
    // need > 0: `prefix` is the smallest chosen key and `need` of the tokens that have it are chosen, the first ones
    const bool any = c.need > 0;
    const int per = (c.flushed + 1023) / 1024 * 64, first = wave * per, end = min(first + per, c.flushed);
    int gt = 0, eq = 0;
    for (int j0 = first; j0 < end; j0 += 64) {
        const int j = j0 + lane;
        const bool in = j < end, must = in && (j < c.lo || j >= c.hi), cand = in && !must && any;
        const u32 k = cand ? weight_key(w[j]) : 0u;
        gt += __popcll(__ballot(must || (cand && k > prefix)));
        eq += __popcll(__ballot(cand && k == prefix));
    }
    if (lane == 0) {
        wave_tot[wave] = gt;
        wave_eq[wave] = eq;
    }
    __syncthreads();
    int at = 0, eq_before = 0;
    for (int k = 0; k < wave; ++k) {
        at += wave_tot[k] + max(0, min(wave_eq[k], need - eq_before));
        eq_before += wave_eq[k];
    }
    for (int j0 = first; j0 < end; j0 += 64) {
        const int j = j0 + lane;
        const bool in = j < end, must = in && (j < c.lo || j >= c.hi), cand = in && !must && any;
        const u32 k = cand ? weight_key(w[j]) : 0u;
        const unsigned long long below = (1ull << lane) - 1, same = __ballot(cand && k == prefix);
        const bool tie = cand && k == prefix && eq_before + __popcll(same & below) < need;
        const bool take = must || (cand && k > prefix) || tie;
        const unsigned long long all = __ballot(take);
        if (take) {
            const int slot = at + __popcll(all & below);
            if (slot < keep) out[slot] = j;
        }
        at += __popcll(all);
        eq_before += __popcll(same);
    }
}

// ---- evict: the move ------------------------------------------------------------------------------------------------------------------------
struct MoveArgs {
    akv_cache_layer from, to;
    const int *kept;            // [B, Hkv, keep]; null: token i moves to place i
    const int *old_lens;        // [B]
    const float *w_from;
    float *w_to;
    int64_t wf_b, wf_h, wt_b, wt_h;
    int keep, sinks, recent, w_cap, only_moved;   // only_moved: sequences that keep everything stay as they are
};

// grid (2 * keep / 64, B * Hkv), 256 threads: 64 kept tokens of one KV head, keys (even blockIdx.x) or values (odd).
__global__ __launch_bounds__(256) void evict_planes_kernel(MoveArgs a) {
    __shared__ int src[kUnit];
    const int H = a.from.n_kv_heads, D = a.from.head_dim, bh = blockIdx.y, b = bh / H, i0 = (blockIdx.x >> 1) * kUnit, tid = threadIdx.x;
    const Choice c = make_choice(a.old_lens[b], a.keep, a.sinks, a.recent);
    if (i0 >= c.have || (a.only_moved && c.flushed <= a.keep)) return;
    if (tid < kUnit) src[tid] = max(0, min(a.kept ? a.kept[(int64_t)bh * a.keep + i0 + tid] : i0 + tid, c.flushed - 1));
    __syncthreads();
    if (blockIdx.x & 1) {
        const int64_t from = (int64_t)bh * a.from.max_seq_len, to = (int64_t)bh * a.to.max_seq_len + i0;
        const int cpr = D / 16;       // 16-byte pieces of a row of high bytes
        for (int id = tid; id < kUnit * cpr; id += 256) {
            const int r = id / cpr, p = id - r * cpr;
            *reinterpret_cast<u32x4 *>(a.to.v_first_8 + (to + r) * D + p * 16) = *reinterpret_cast<const u32x4 *>(a.from.v_first_8 + (from + src[r]) * D + p * 16);
        }
        for (int id = tid; id < kUnit * cpr; id += 256) {
            const int r = id / cpr, p = id - r * cpr;
            *reinterpret_cast<u32x2 *>(a.to.v_mid_4 + (to + r) * (D / 2) + p * 8) = *reinterpret_cast<const u32x2 *>(a.from.v_mid_4 + (from + src[r]) * (D / 2) + p * 8);
            *reinterpret_cast<u32x2 *>(a.to.v_last_4 + (to + r) * (D / 2) + p * 8) = *reinterpret_cast<const u32x2 *>(a.from.v_last_4 + (from + src[r]) * (D / 2) + p * 8);
        }
        return;
    }
    // keys: a thread takes four kept tokens of a channel
    const int kb = a.from.k_block, r = (tid & 15) * 4;
    const int64_t to = ((int64_t)bh * a.to.n_max_blocks + i0 / kb) * D * kb + i0 % kb + r;
    int64_t from[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) from[t] = ((int64_t)bh * a.from.n_max_blocks + src[r + t] / kb) * D * kb + src[r + t] % kb;
    for (int d = tid >> 4; d < D; d += 16) {
        u32 hi = 0, mid = 0, last = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int64_t at = from[t] + (int64_t)d * kb;
            const u32 sh = at & 1 ? 0 : 4, place = (t >> 1) * 8 + (t & 1 ? 0 : 4);
            hi |= (u32)a.from.k_first_8[at] << (8 * t);
            mid |= ((a.from.k_mid_4[at >> 1] >> sh) & 15u) << place;
            last |= ((a.from.k_last_4[at >> 1] >> sh) & 15u) << place;
        }
        *reinterpret_cast<u32 *>(a.to.k_first_8 + to + (int64_t)d * kb) = hi;
        *reinterpret_cast<unsigned short *>(a.to.k_mid_4 + (to + (int64_t)d * kb) / 2) = (unsigned short)mid;
        *reinterpret_cast<unsigned short *>(a.to.k_last_4 + (to + (int64_t)d * kb) / 2) = (unsigned short)last;
    }
}

// grid B * Hkv, 256 threads: weights (kept ones, then the rest buffer's, zeros behind; in order, so that they may move within their
// row), rest buffers, column maxima and lengths.
__global__ __launch_bounds__(256) void evict_rest_kernel(MoveArgs a, int copy) {
    const int H = a.from.n_kv_heads, D = a.from.head_dim, bh = blockIdx.x, b = bh / H, h = bh - b * H, tid = threadIdx.x;
    const Choice c = make_choice(a.old_lens[b], a.keep, a.sinks, a.recent);
    const int left = c.n - c.flushed + c.have;
    if (copy) {
        const int pieces = D / 8;
        for (int id = tid; id < kUnit * pieces; id += 256) {
            const int64_t at = (((int64_t)b * kUnit + id / pieces) * H + h) * D * 2 + (id % pieces) * 16;
            *reinterpret_cast<u32x4 *>(a.to.restk + at) = *reinterpret_cast<const u32x4 *>(a.from.restk + at);
            *reinterpret_cast<u32x4 *>(a.to.restv + at) = *reinterpret_cast<const u32x4 *>(a.from.restv + at);
        }
        for (int d = tid; d < D; d += 256) {
            a.to.k_exp_column_max[(int64_t)bh * D + d] = a.from.k_exp_column_max[(int64_t)bh * D + d];
            a.to.v_exp_column_max[(int64_t)bh * D + d] = a.from.v_exp_column_max[(int64_t)bh * D + d];
        }
    }
    if (h == 0 && tid == 0) a.to.seq_lens[b] = left;
    if (a.w_to == nullptr || (!copy && c.flushed <= a.keep)) return;
    const float *w = a.w_from + b * a.wf_b + h * a.wf_h;
    float *o = a.w_to + b * a.wt_b + h * a.wt_h;
    for (int i0 = 0; i0 < left; i0 += 256) {
        const int i = i0 + tid;
        float x = 0.f;
        if (i < left) x = w[i < c.have ? max(0, min(a.kept[(int64_t)bh * a.keep + i], c.flushed - 1)) : c.flushed + i - c.have];
        __syncthreads();          // a weight never moves up its row: what later rounds read is not overwritten yet
        if (i < left) o[i] = x;
    }
    for (int i = left + tid; i < a.w_cap; i += 256) o[i] = 0.f;
}

}  // namespace akv

extern "C" int akv_accumulate_weights(const float *weights, int64_t weights_stride_b, int64_t weights_stride_h, const uint8_t *probs, int row_stride,
                                      const int *seq_lens, float *out, int64_t out_stride_b, int64_t out_stride_h, int bsz, int n_q_heads, int n_kv_heads,
                                      int capacity, float decay, akv_stream_t stream) {
    AKV_REQUIRE(weights && probs && seq_lens && out, "accumulate_weights: null pointer");
    AKV_REQUIRE(bsz >= 1 && bsz <= 65535 && n_kv_heads >= 1 && n_kv_heads <= 65535 && n_q_heads >= 1 && n_q_heads % n_kv_heads == 0,
                "accumulate_weights: bsz %d, heads %d / %d", bsz, n_q_heads, n_kv_heads);
    AKV_REQUIRE(row_stride % 8 == 0 && ((uintptr_t)probs & 15) == 0, "accumulate_weights: probabilities need 16-byte aligned rows");
    AKV_REQUIRE(capacity >= 1 && capacity <= row_stride, "accumulate_weights: capacity %d outside [1, row_stride %d]", capacity, row_stride);
    AKV_REQUIRE(decay == decay && decay <= 1e30f && decay >= -1e30f, "accumulate_weights: decay must be finite");
    const dim3 grid((capacity + 2047) / 2048, n_kv_heads, bsz);
    hipLaunchKernelGGL(akv::accumulate_weights_kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), weights, probs, seq_lens, out, n_q_heads / n_kv_heads,
                       n_kv_heads, row_stride, weights_stride_b, weights_stride_h, out_stride_b, out_stride_h, capacity, decay);
    return akv::check_launch("accumulate_weights");
}

namespace akv {
// Where the planes of an eviction in place wait between the two moves: the kept tokens, laid out as a small cache.
struct EvictPlan {
    size_t lens_bytes, k_first, v_first, total;
    int blocks;
};
static EvictPlan evict_plan(int bsz, int n_kv_heads, int head_dim, int k_block, int keep, bool in_place) {
    EvictPlan p;
    p.lens_bytes = ((size_t)bsz * sizeof(int) + 255) / 256 * 256;
    p.blocks = (keep + k_block - 1) / k_block;
    p.k_first = (size_t)bsz * n_kv_heads * p.blocks * k_block * head_dim;
    p.v_first = (size_t)bsz * n_kv_heads * keep * head_dim;
    p.total = p.lens_bytes + (in_place ? 2 * (p.k_first + p.v_first) : 0);
    return p;
}
}  // namespace akv

extern "C" size_t akv_evict_workspace_bytes(int bsz, int n_kv_heads, int head_dim, int k_block, int keep, int in_place) {
    if (bsz < 1 || n_kv_heads < 1 || head_dim < 1 || (k_block != 64 && k_block != 256) || keep < 64) return 0;
    return akv::evict_plan(bsz, n_kv_heads, head_dim, k_block, keep, in_place != 0).total;
}

extern "C" int akv_evict(const akv_cache_layer *from, const akv_cache_layer *to, const float *weights, int64_t weights_stride_b, int64_t weights_stride_h,
                         float *weights_to, int64_t to_stride_b, int64_t to_stride_h, int weights_to_capacity, int *kept, int keep, int sinks, int recent,
                         void *workspace, size_t workspace_bytes, akv_stream_t stream) {
    int rc = akv::check_layer(from, "evict");
    if (rc == AKV_OK) rc = akv::check_layer(to, "evict");
    if (rc != AKV_OK) return rc;
    AKV_REQUIRE(weights && kept, "evict: null pointer");
    AKV_REQUIRE(from->bsz == to->bsz && from->n_kv_heads == to->n_kv_heads && from->head_dim == to->head_dim && from->k_block == to->k_block,
                "evict: the caches differ in batch, heads, head_dim or k_block");
    AKV_REQUIRE(keep >= 64 && keep % 64 == 0, "evict: keep %d must be a positive multiple of 64", keep);
    AKV_REQUIRE(sinks >= 0 && recent >= 0 && (int64_t)sinks + recent <= keep, "evict: sinks %d and recent %d must fit into keep %d", sinks, recent, keep);
    const void *f[] = {from->k_first_8, from->k_mid_4, from->k_last_4, from->v_first_8, from->v_mid_4, from->v_last_4, from->k_exp_column_max,
                       from->v_exp_column_max, from->restk, from->restv, from->seq_lens};
    const void *t[] = {to->k_first_8, to->k_mid_4, to->k_last_4, to->v_first_8, to->v_mid_4, to->v_last_4, to->k_exp_column_max,
                       to->v_exp_column_max, to->restk, to->restv, to->seq_lens};
    int same = 0;
    for (int i = 0; i < 11; ++i) same += f[i] == t[i];
    AKV_REQUIRE(same == 0 || same == 11, "evict: the destination is the same cache or another one, not some of both");
    const bool in_place = same == 11;
    AKV_REQUIRE(in_place || to->max_seq_len >= keep + 63, "evict: a destination of %d tokens cannot hold %d and a rest buffer", to->max_seq_len, keep);
    AKV_REQUIRE(weights_to == nullptr || in_place == (weights_to == weights), "evict: the weights move with the cache: in place or not");
    AKV_REQUIRE(weights_to == nullptr || weights_to_capacity >= (in_place ? from->max_seq_len : keep + 63), "evict: room for %d weights", weights_to_capacity);
    const akv::EvictPlan p = akv::evict_plan(from->bsz, from->n_kv_heads, from->head_dim, from->k_block, keep, in_place);
    AKV_REQUIRE(workspace && workspace_bytes >= p.total && ((uintptr_t)workspace & 15) == 0, "evict: needs a 16-byte aligned workspace of %zu bytes, got %zu", p.total,
                workspace_bytes);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int streams = from->bsz * from->n_kv_heads;
    akv::MoveArgs a;
    a.from = *from;
    a.to = *to;
    a.kept = kept;
    a.old_lens = static_cast<int *>(workspace);
    a.w_from = weights; a.w_to = weights_to;
    a.wf_b = weights_stride_b; a.wf_h = weights_stride_h; a.wt_b = to_stride_b; a.wt_h = to_stride_h;
    a.keep = keep; a.sinks = sinks; a.recent = recent; a.w_cap = weights_to_capacity;
    a.only_moved = in_place;
    hipLaunchKernelGGL(akv::evict_select_kernel, dim3(streams), dim3(1024), 0, st, weights, weights_stride_b, weights_stride_h, from->seq_lens, kept,
                       static_cast<int *>(workspace), from->n_kv_heads, from->max_seq_len, keep, sinks, recent);
    const dim3 grid(2 * (keep / 64), streams);
    if (!in_place) {
        hipLaunchKernelGGL(akv::evict_planes_kernel, grid, dim3(256), 0, st, a);
    } else {
        uint8_t *w = static_cast<uint8_t *>(workspace) + p.lens_bytes;
        akv::MoveArgs m = a;
        m.to.k_first_8 = w;
        m.to.k_mid_4 = m.to.k_first_8 + p.k_first;
        m.to.k_last_4 = m.to.k_mid_4 + p.k_first / 2;
        m.to.v_first_8 = m.to.k_last_4 + p.k_first / 2;
        m.to.v_mid_4 = m.to.v_first_8 + p.v_first;
        m.to.v_last_4 = m.to.v_mid_4 + p.v_first / 2;
        m.to.n_max_blocks = p.blocks;
        m.to.max_seq_len = keep;
        hipLaunchKernelGGL(akv::evict_planes_kernel, grid, dim3(256), 0, st, m);
        m.from = m.to;
        m.to = a.to;
        m.kept = nullptr;
        hipLaunchKernelGGL(akv::evict_planes_kernel, grid, dim3(256), 0, st, m);
    }
    hipLaunchKernelGGL(akv::evict_rest_kernel, dim3(streams), dim3(256), 0, st, a, in_place ? 0 : 1);
    return akv::check_launch("evict");
}
