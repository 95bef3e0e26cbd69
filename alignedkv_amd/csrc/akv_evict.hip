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
// probability, 8 per weight): a thread takes 8 tokens, 16 bytes of each head's row.  8 x 4050 to 8100 tokens, 32 heads over 8: 3.8 us, of
// which 1.2 are its bytes; a launch that does nothing takes 2.
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

// One workgroup per (sequence, KV head), of 1024 threads, or of 256 where the rows are short (their barriers are cheaper: 1024 tokens
// 11.5 us against 14.8).  The `need`-th largest key is found by its digits, 11 + 11 + 10 bits, each from a
// histogram in LDS; then the chosen tokens are written in order.  Token THREADS i + thread is this thread's i-th: the keys of the first
// kHeld * THREADS tokens are read once and kept in registers (32000 tokens: 46 us with every pass reading them, latency, not
// bytes, 34 with the registers), those of a longer row again in every pass.  Weights crowd in few exponents: eight histograms side by side,
// a lane's by its number, keep lanes of one bin apart (32000 tokens 34.5 -> 31.6 us); with 256 threads clearing and adding them costs more than
// it saves (1000 tokens 11.4 -> 17.3 us), and one does.  Latency bounds it: 8 MB of weights at 8 x 8 rows of 32000.
constexpr int kHeld = 32;
template <int THREADS>
__global__ __launch_bounds__(THREADS) void evict_select_kernel(const float *__restrict__ weights, int64_t w_b, int64_t w_h, const int *__restrict__ lens,
                                                            int *__restrict__ kept, int *__restrict__ old_lens, int Hkv, int capacity, int keep, int sinks,
                                                            int recent) {
    constexpr int WAVES = THREADS / 64, BINS = 2048 / THREADS, COPIES = THREADS == 1024 ? 8 : 1;
    __shared__ __attribute__((aligned(16))) u32 hist[2048 * COPIES];
    __shared__ int wave_tot[WAVES];
    __shared__ u32 digit_s;
    __shared__ int above_s;
    const int h = blockIdx.x % Hkv, b = blockIdx.x / Hkv, tid = threadIdx.x, lane = tid & 63, wave = wave_index();
    const Choice c = make_choice(max(0, min(lens[b], capacity)), keep, sinks, recent);
    int *out = kept + (int64_t)blockIdx.x * keep;
    if (h == 0 && tid == 0) old_lens[b] = c.n;
    for (int i = c.have + tid; i < keep; i += THREADS) out[i] = -1;
    if (c.flushed <= keep) {
        for (int i = tid; i < c.have; i += THREADS) out[i] = i;
        return;
    }
    const float *w = weights + b * w_b + h * w_h;
    u32 held[kHeld];
    // (behind the row's end: out of the descriptor's range, nothing is fetched)
    const auto row = make_rsrc(w, (u32)min(c.flushed, kHeld * THREADS) * 4u);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = (u32)__builtin_amdgcn_raw_buffer_load_b32(row, (i * THREADS + tid) * 4, 0, 0);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = weight_key(__uint_as_float(held[i]));
    // f(token, key, i) for every token of this thread
    const auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (i * THREADS < c.flushed) f(i * THREADS + tid, held[i]);
#pragma unroll 4
        for (int j0 = kHeld * THREADS; j0 < c.flushed; j0 += THREADS) f(j0 + tid, weight_key(w[min(j0 + tid, c.flushed - 1)]));
    };
    const auto candidate = [&](int j) { return j >= c.lo && j < c.hi; };
    u32 prefix = 0;             // digits found so far
    int need = c.need;          // still to be taken among the keys that share them
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < 2048 * COPIES / 4; i += THREADS) reinterpret_cast<u32x4 *>(hist)[i] = u32x4{0u, 0u, 0u, 0u};
        __syncthreads();
        each([&](int j, u32 k) {
            if (candidate(j) && (pass == 0 || (k >> (shift + bits)) == prefix)) atomicAdd(&hist[((k >> shift) & ((1u << bits) - 1)) * COPIES + (lane & (COPIES - 1))], 1u);
        });
        __syncthreads();
        // thread i holds BINS bins below 2048 - BINS i: counts from the top
        const int top = 2047 - BINS * tid;
        int own[BINS], inc = 0;
#pragma unroll
        for (int k = 0; k < BINS; ++k) {
            own[k] = 0;
#pragma unroll
            for (int i = 0; i < COPIES; ++i) own[k] += (int)hist[(top - k) * COPIES + i];
            inc += own[k];
        }
        const int mine = inc;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(inc, d);
            if (lane >= d) inc += o;
        }
        if (lane == 63) wave_tot[wave] = inc;
        __syncthreads();
        int before = lane < wave ? wave_tot[lane] : 0;
        before = wave_sum_i32(before) + inc - mine;
#pragma unroll
        for (int k = 0; k < BINS; ++k) {
            if (before < need && need <= before + own[k]) {
                digit_s = (u32)(top - k);
                above_s = before;
            }
            before += own[k];
        }
        __syncthreads();
        if (need > 0) {
            prefix = (prefix << bits) | digit_s;
            need -= above_s;
        }
        __syncthreads();
    }
    // need > 0: `prefix` is the smallest chosen key and `need` of the tokens that have it are chosen, the first ones: a token's place is the
    // number of tokens before it that are chosen for sure plus the number of equal ones before it, at most `need`.
    // Token THREADS r + 64 wave + lane: in order of r, then the wave, then the lane.  Eight rounds at a time.
    const bool any = c.need > 0;
    const unsigned long long below = (1ull << lane) - 1;
    __shared__ u32 counts[8 * WAVES];          // [round][wave]: chosen for sure, equal << 16
    int sure_before = 0, eq_before = 0;
    const auto rounds8 = [&](int j0, const u32 (&key)[8]) {
        unsigned long long sure[8], same[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int j = j0 + r * THREADS + tid;
            const bool in = j < c.flushed, cand = in && candidate(j) && any;
            sure[r] = __ballot((in && !candidate(j)) || (cand && key[r] > prefix));
            same[r] = __ballot(cand && key[r] == prefix);
            if (lane == 0) counts[r * WAVES + wave] = (u32)__popcll(sure[r]) | (u32)__popcll(same[r]) << 16;
        }
        __syncthreads();
        // every wave sums the counts up: two entries a lane
        const bool real = lane < 4 * WAVES;
        const u32 v0 = real ? counts[2 * lane] : 0u, v1 = real ? counts[2 * lane + 1] : 0u;
        u32 inc = v0 + v1;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const u32 o = (u32)__shfl_up((int)inc, d);
            if (lane >= d) inc += o;
        }
        const u32 excl = inc - v0 - v1 + (wave & 1 ? v0 : 0u);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const u32 before = (u32)__builtin_amdgcn_readlane((int)excl, r * (WAVES / 2) + (wave >> 1));
            const int s0 = sure_before + (int)(before & 0xFFFFu), e0 = eq_before + (int)(before >> 16) + __popcll(same[r] & below);
            const bool tie = (same[r] >> lane) & 1;
            if (((sure[r] >> lane) & 1) || (tie && e0 < need)) {
                const int slot = s0 + __popcll(sure[r] & below) + min(e0, need);
                if (slot < keep) out[slot] = j0 + r * THREADS + tid;
            }
        }
        const u32 all = (u32)__builtin_amdgcn_readlane((int)inc, 63);
        sure_before += (int)(all & 0xFFFFu);
        eq_before += (int)(all >> 16);
        __syncthreads();
    };
#pragma unroll
    for (int q = 0; q < kHeld / 8; ++q) {
        if (q * (8 * THREADS) >= c.flushed) break;
        u32 key[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) key[r] = held[q * 8 + r];
        rounds8(q * (8 * THREADS), key);
    }
#pragma unroll 1
    for (int j0 = kHeld * THREADS; j0 < c.flushed; j0 += 8 * THREADS) {
        u32 key[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) key[r] = weight_key(w[min(j0 + r * THREADS + tid, c.flushed - 1)]);
        rounds8(j0, key);
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

// per_head = keep / 64 * (1 + D / 32) + rest chunks workgroups of 256 threads for each KV head.  The first keep / 64 workgroups of a KV head move the values of 64
// kept tokens each, the next keep / 64 * D / 32 the keys of 64 kept tokens and 32 channels, the last ones everything else.
constexpr int kRestChunk = 4096;       // weights a workgroup moves

// Values: rows of D + D / 2 + D / 2 bytes, gathered 16 and 8 bytes a lane.
__device__ __forceinline__ void move_values(const MoveArgs &a, int bh, int i0, const int *src) {
    const int D = a.from.head_dim, tid = threadIdx.x, cpr = D / 16;
    const int64_t from = (int64_t)bh * a.from.max_seq_len, to = (int64_t)bh * a.to.max_seq_len + i0;
#pragma unroll 4
    for (int id = tid; id < kUnit * cpr; id += 256) {
        const int r = id / cpr, p = id - r * cpr;
        const int64_t f = (from + src[r]) * D + p * 16, t = (to + r) * D + p * 16;
        *reinterpret_cast<u32x4 *>(a.to.v_first_8 + t) = *reinterpret_cast<const u32x4 *>(a.from.v_first_8 + f);
        *reinterpret_cast<u32x2 *>(a.to.v_mid_4 + t / 2) = *reinterpret_cast<const u32x2 *>(a.from.v_mid_4 + f / 2);
        *reinterpret_cast<u32x2 *>(a.to.v_last_4 + t / 2) = *reinterpret_cast<const u32x2 *>(a.from.v_last_4 + f / 2);
    }
}

// Keys: a channel's tokens lie side by side, so a kept token is a byte here and a nibble there in 3 D places, and nearly every line
// of a block that holds kept tokens is touched.  Blocks of 256 source tokens that hold any are brought into LDS whole (32 channels:
// 16 KB, asynchronous, the next one while this one is searched); a lane owns a kept token, a wave eight channels: reading a byte a
// lane out of one channel's row is free of bank conflicts, and the token's bytes stay in four registers until its block has come by.
// Gathering the bytes from memory kept the address units busy instead: 217 us at 8 x 32000 tokens x 8 heads x 128 to 4096, against 148 for the
// whole move.  Its bound: 515 MB of lines that hold kept tokens and 134 MB written, 4.4 TB/s.
__device__ __forceinline__ void move_keys(const MoveArgs &a, int bh, int i0, int ch0, const int *src, uint8_t *stage, uint8_t *done) {
    const int D = a.from.head_dim, kb = a.from.k_block, tid = threadIdx.x, lane = tid & 63, wave = wave_index();
    const int my = src[lane];
    const int per = 256 / kb;                       // plane blocks of a stretch of 256 tokens
    const int blocks = a.from.n_max_blocks;
    const u32 lds0 = lds_address(stage) + wave * 1024;
    // the next stretch that holds a kept token at or behind place i: uniform in the workgroup
    const auto stretch = [&](int i) { return i < kUnit ? src[i] >> 8 : -1; };
    const auto first_behind = [&](int s) { return (int)__popcll(__ballot((my >> 8) <= s)); };       // (kept tokens ascend)
    auto request = [&](int s, int buf) {
        // piece p (16 bytes of the high bytes) of the stretch: block p / (2 kb), channel, part; the nibble planes half as many
        const int64_t blk = (int64_t)bh * blocks + (int64_t)s * per;
        const int have = min(per, blocks - s * per);
        const auto rh = make_rsrc(a.from.k_first_8 + blk * D * kb, (u32)(have * D * kb));
        const auto rm = make_rsrc(a.from.k_mid_4 + blk * D * kb / 2, (u32)(have * D * kb / 2));
        const auto rl = make_rsrc(a.from.k_last_4 + blk * D * kb / 2, (u32)(have * D * kb / 2));
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int byte = (c * 256 + tid) * 16, z = byte / (32 * kb), in = byte - z * (32 * kb);
            load_to_lds(rh, lds0 + buf * 16384 + c * 4096, z < have ? z * D * kb + ch0 * kb + in : kSkip);
        }
        const int byte = tid * 16, z = byte / (16 * kb), in = byte - z * (16 * kb);
        load_to_lds(rm, lds0 + buf * 16384 + 8192, z < have ? z * D * kb / 2 + ch0 * kb / 2 + in : kSkip);
        load_to_lds(rl, lds0 + buf * 16384 + 12288, z < have ? z * D * kb / 2 + ch0 * kb / 2 + in : kSkip);
    };
    u32 hi[2] = {0u, 0u}, lo[2] = {0u, 0u};
    int s = stretch(0), buf = 0;
    request(s, 0);
    while (s >= 0) {
        const int next = stretch(first_behind(s));
        wait_tile();
        if (next >= 0) request(next, buf ^ 1);
        if ((my >> 8) == s) {
            const int z = (my & 255) / kb, slot = (my & 255) % kb;
            const uint8_t *h = stage + buf * 16384 + z * (32 * kb) + wave * 8 * kb + slot, *m = stage + buf * 16384 + 8192 + z * (16 * kb) + wave * 4 * kb + (slot >> 1);
            const int sh = slot & 1 ? 0 : 4;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                hi[k >> 2] |= (u32)h[k * kb] << (8 * (k & 3));
                lo[k >> 2] |= ((((u32)m[k * kb / 2] >> sh) & 15u) << 4 | (((u32)m[4096 + k * kb / 2] >> sh) & 15u)) << (8 * (k & 3));
            }
        }
        buf ^= 1;
        s = next;
    }
    // token-major registers -> channel-major rows of 64 tokens
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        done[(wave * 8 + k) * kUnit + lane] = (uint8_t)(hi[k >> 2] >> (8 * (k & 3)));
        done[2048 + (wave * 8 + k) * kUnit + lane] = (uint8_t)(lo[k >> 2] >> (8 * (k & 3)));
    }
    __syncthreads();
    const int d = tid >> 3, r = (tid & 7) * 8;          // eight tokens of a channel
    const u32x2 h8 = *reinterpret_cast<const u32x2 *>(done + d * kUnit + r), l8 = *reinterpret_cast<const u32x2 *>(done + 2048 + d * kUnit + r);
    u32 mid = 0, last = 0;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const u32 x = q ? l8.y : l8.x;                  // low bytes of tokens 4 q ..: even ones to the high nibbles
        const u32 m2 = (x & 0xF0u) | ((x >> 12) & 15u) | (((x >> 16) & 0xF0u) | (x >> 28)) << 8;
        const u32 l2 = (x & 15u) << 4 | ((x >> 8) & 15u) | (((x >> 16) & 15u) << 4 | ((x >> 24) & 15u)) << 8;
        mid |= m2 << (16 * q);
        last |= l2 << (16 * q);
    }
    const int64_t to = (((int64_t)bh * a.to.n_max_blocks + i0 / kb) * D + ch0 + d) * kb + i0 % kb + r;
    *reinterpret_cast<u32x2 *>(a.to.k_first_8 + to) = h8;
    *reinterpret_cast<u32 *>(a.to.k_mid_4 + to / 2) = mid;
    *reinterpret_cast<u32 *>(a.to.k_last_4 + to / 2) = last;
}

// Weights (kept ones, then the rest buffer's, zeros behind), rest buffers, column maxima and lengths.  Into another cache the chunks of a
// row are independent; within a row (copy == 0) one workgroup goes through it in order.
__device__ __forceinline__ void move_rest(const MoveArgs &a, const Choice &c, int bh, int chunk, int copy) {
    const int H = a.from.n_kv_heads, D = a.from.head_dim, b = bh / H, h = bh - b * H, tid = threadIdx.x;
    const int left = c.n - c.flushed + c.have;
    if (chunk == 0) {
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
    }
    if (a.w_to == nullptr || (!copy && c.flushed <= a.keep)) return;
    const float *w = a.w_from + b * a.wf_b + h * a.wf_h;
    float *o = a.w_to + b * a.wt_b + h * a.wt_h;
    const int first = copy ? chunk * kRestChunk : 0, end = copy ? min(first + kRestChunk, a.w_cap) : a.w_cap;
    const int moved = min(left, end);
    for (int i0 = first; i0 < moved; i0 += 2048) {
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = min(i0 + k * 256 + tid, moved - 1);
            x[k] = w[i < c.have ? max(0, min(a.kept[(int64_t)bh * a.keep + i], c.flushed - 1)) : c.flushed + i - c.have];
        }
        if (!copy) __syncthreads();          // a weight never moves up its row: what later rounds read is not overwritten yet
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (i0 + k * 256 + tid < moved) o[i0 + k * 256 + tid] = x[k];
    }
    for (int i = max(first, left) + tid; i < end; i += 256) o[i] = 0.f;
}

__global__ __launch_bounds__(256) void evict_rest_kernel(MoveArgs a) {
    move_rest(a, make_choice(a.old_lens[blockIdx.x / a.from.n_kv_heads], a.keep, a.sinks, a.recent), blockIdx.x, 0, 0);
}

__global__ __launch_bounds__(256) void evict_move_kernel(MoveArgs a, int per_head, int with_rest, int copy) {
    __shared__ __attribute__((aligned(1024))) uint8_t stage[2 * 16384];
    __shared__ __attribute__((aligned(16))) uint8_t done[4096];
    __shared__ int src[kUnit];
    // workgroups are dealt out to the 8 XCDs in turn: a KV head's go to one of them, where neighbouring tiles find the stretch they share in L2
    const int bh = (int)(blockIdx.x / 8 / per_head) * 8 + (int)(blockIdx.x % 8), x = blockIdx.x / 8 % per_head;
    if (bh >= a.from.bsz * a.from.n_kv_heads) return;
    const int b = bh / a.from.n_kv_heads, tid = threadIdx.x, tiles = a.keep / kUnit, groups = a.from.head_dim / 32;
    const Choice c = make_choice(a.old_lens[b], a.keep, a.sinks, a.recent);
    if (x >= tiles * (1 + groups)) {
        if (with_rest) move_rest(a, c, bh, x - tiles * (1 + groups), copy);
        return;
    }
    // (the channel groups of a tile share their lines' neighbours: next to each other)
    const int tile = x < tiles ? x : (x - tiles) / groups, i0 = tile * kUnit;
    if (i0 >= c.have || (a.only_moved && c.flushed <= a.keep)) return;
    if (tid < kUnit) src[tid] = max(0, min(a.kept ? a.kept[(int64_t)bh * a.keep + i0 + tid] : i0 + tid, c.flushed - 1));
    __syncthreads();
    if (x < tiles) move_values(a, bh, i0, src);
    else move_keys(a, bh, i0, (x - tiles) % groups * 32, src, stage, done);
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
    AKV_REQUIRE(akv::rows_apart(bsz, n_kv_heads, capacity, out_stride_b, out_stride_h), "accumulate_weights: rows of out share memory (strides %lld, %lld)",
                (long long)out_stride_b, (long long)out_stride_h);
    const int64_t span = akv::rows_span(bsz, n_kv_heads, capacity, out_stride_b, out_stride_h);
    const bool same = out == weights && (bsz == 1 || out_stride_b == weights_stride_b) && (n_kv_heads == 1 || out_stride_h == weights_stride_h);
    AKV_REQUIRE((same || !akv::share_memory(out, span, weights, akv::rows_span(bsz, n_kv_heads, capacity, weights_stride_b, weights_stride_h))) &&
                    !akv::share_memory(out, span, probs, (int64_t)bsz * n_q_heads * row_stride * 2),
                "accumulate_weights: out must be the weights themselves or not overlap them, nor the probabilities");
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
    AKV_REQUIRE(keep >= 64 && keep % 64 == 0 && keep <= (1 << 20), "evict: keep %d must be a positive multiple of 64, at most 2^20", keep);
    AKV_REQUIRE(((int64_t)from->bsz * from->n_kv_heads + 8) * (keep / 64 * 9 + 1 + weights_to_capacity / 4096) < (1ll << 31), "evict: too many tokens");
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
    AKV_REQUIRE(weights_to == nullptr || akv::rows_apart(from->bsz, from->n_kv_heads, weights_to_capacity, to_stride_b, to_stride_h),
                "evict: rows of weights share memory (strides %lld, %lld)", (long long)to_stride_b, (long long)to_stride_h);
    AKV_REQUIRE(weights_to == nullptr || in_place ||
                    !akv::share_memory(weights, akv::rows_span(from->bsz, from->n_kv_heads, from->max_seq_len, weights_stride_b, weights_stride_h), weights_to,
                                       akv::rows_span(from->bsz, from->n_kv_heads, weights_to_capacity, to_stride_b, to_stride_h)),
                "evict: the weights that move to another cache must not overlap those they come from");
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
#define AKV_SELECT(THREADS)                                                                                                             \
    hipLaunchKernelGGL(akv::evict_select_kernel<THREADS>, dim3(streams), dim3(THREADS), 0, st, weights, weights_stride_b, weights_stride_h, \
                       from->seq_lens, kept, static_cast<int *>(workspace), from->n_kv_heads, from->max_seq_len, keep, sinks, recent)
    if (from->max_seq_len <= 256 * akv::kHeld) AKV_SELECT(256);
    else AKV_SELECT(1024);
#undef AKV_SELECT
    const int moves = keep / 64 * (1 + from->head_dim / 32);
    const auto grid = [&](int per_head) { return dim3((u32)((int64_t)((streams + 7) / 8 * 8) * per_head)); };
    if (!in_place) {
        const int chunks = weights_to ? (weights_to_capacity + akv::kRestChunk - 1) / akv::kRestChunk : 1;
        hipLaunchKernelGGL(akv::evict_move_kernel, grid(moves + chunks), dim3(256), 0, st, a, moves + chunks, 1, 1);
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
        hipLaunchKernelGGL(akv::evict_move_kernel, grid(moves), dim3(256), 0, st, m, moves, 0, 0);
        // back to the front of the cache's own planes, token i of the copy to place i; and the weights, within their rows
        akv::MoveArgs back = m;
        back.from = m.to;
        back.to = a.to;
        back.kept = nullptr;
        hipLaunchKernelGGL(akv::evict_move_kernel, grid(moves), dim3(256), 0, st, back, moves, 0, 0);
        hipLaunchKernelGGL(akv::evict_rest_kernel, dim3(streams), dim3(256), 0, st, a);
    }
    return akv::check_launch("evict");
}
