// k_logprobs.hip -- log probabilities of given tokens, entropy and the top alternatives of rows
// of f32 logits.
//
// With m the row's maximum, e_j = exp(x_j - m) and Z = sum e_j:
//   log p_t = (x_t - m) - log Z         entropy = log Z - (sum (x_j - m) e_j) / Z
// Both of the entropy's terms are at least 0, so it never cancels. The elements equal to m are
// counted rather than summed: Z = C + S with S the sum of the others, and log Z =
// log1p((C - 1) + S) keeps its relative accuracy where one token is almost certain.
//
// logprobs_part_kernel: a workgroup per (row, segment of PER * 256 logits), every logit read
// once into registers and used for the maximum, the sums and the selection. Its segment's
// state: m, S, C, A = sum (x_j - m) e_j, the target's logit where the segment holds it, and
// the top_n largest keys in order. logprobs_join_kernel: a workgroup per row joins the
// segments' states. Memory bound: the logits are read once; 512 rows of 65536 (134 MB) with five
// alternatives take 28 us, 4.8 TB/s, and the join 5.5. One row of 65536 with 20 alternatives: two
// launches of 6 and 5 us. (The join by the row's last segment, behind a fence and a counter, took longer:
// 11.2 us instead of 10.2 for one row of 32768, 83 instead of 19 for 600 of 13578.)
//
// Selection by unique 64-bit keys (the logit in an order-preserving form above the complement of
// its index, so that equal logits fall to the lower index): a bound that top_n to 1.5 top_n of the
// threads' largest keys reach is one that top_n elements reach, and only those threads' elements
// can (at most 1.5 PER top_n; a few more than top_n as a rule). They are gathered in LDS and
// ordered by counting, for each, those above it. The join does the same with each segment's
// sorted keys in place of a thread's elements.
#include "ds5_common.hpp"

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxSegs = 256;  // segments per row: one per thread of the join
constexpr uint32_t kTop = DS5_LOGPROBS_MAX_TOP;

struct SegState {
    float m, s, c, a, t;  // t: the target's logit, or NaN where the segment does not hold it
};

struct LogprobsParams {
    const float* logits;
    const int32_t* targets;
    float* logprobs;
    float* entropy;
    int32_t* top_ids;
    float* top_logprobs;
    uint32_t vocab, row_stride, top_n, n_segs;
    SegState* states;  // [n_rows, n_segs]
    uint64_t* keys;    // [n_rows, n_segs, top_n], descending, 0 past a segment's elements
};

constexpr uint32_t kLowest = 0x007fffffu;  // the order-preserving form of -inf
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 orders as +0
    const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return ((uint64_t)o << 32) | (uint32_t)~id;
}

__device__ __forceinline__ uint64_t kmax(uint64_t a, uint64_t b) { return a > b ? a : b; }

// A bound that n to kAccept(n) of the 256 keys in LDS reach, or 1 where fewer than n are there (0: none).
// Every wavefront works it out for itself, bit by bit from the highest: by the keys' logits alone, and on
// into their indices only where more than kAccept(n) share the last logit.
__device__ __forceinline__ constexpr uint32_t kAccept(uint32_t n) { return n + n / 2; }
__device__ __forceinline__ uint64_t find_bound(const uint64_t* s_own, uint32_t n) {
    uint64_t k[4];
#pragma unroll
    for (int i = 0; i < 4; i++) k[i] = s_own[64 * i + (threadIdx.x & 63)];
    uint32_t count = 0, hi = 0;
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
        uint32_t reach = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) reach += __popcll(__ballot((uint32_t)(k[i] >> 32) >= (hi | bit)));
        if (reach < n) continue;
        hi |= bit;
        count = reach;
        if (count <= kAccept(n)) break;
    }
    uint64_t bound = (uint64_t)hi << 32;
    if (!count) return 1;
    for (uint64_t bit = 0x80000000u; bit && count > kAccept(n); bit >>= 1) {
        uint32_t reach = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) reach += __popcll(__ballot(k[i] >= (bound | bit)));
        if (reach < n) continue;
        bound |= bit;
        count = reach;
    }
    return bound;
}

// The n largest of the keys in s_list into out[0, n), in descending order (0 where there are fewer).
__device__ __forceinline__ void order_top(const uint64_t* s_list, uint32_t count, uint32_t n, uint64_t* out) {
    const uint32_t tid = threadIdx.x;
    for (uint32_t i = tid; i < count; i += kThreads) {
        const uint64_t k = s_list[i];
        uint32_t rank = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < count; j++) rank += s_list[j] > k;
        if (rank < n) out[rank] = k;
    }
    if (tid >= count && tid < n) out[tid] = 0;
    __syncthreads();
}

// s, c and a summed over the workgroup, on every thread
__device__ __forceinline__ void block_sums(float& s, float& c, float& a, float (*s_sums)[3]) {
    const uint32_t wave = threadIdx.x >> 6;
    s = wave_allreduce(s, OpAdd{});
    c = wave_allreduce(c, OpAdd{});
    a = wave_allreduce(a, OpAdd{});
    if ((threadIdx.x & 63) == 0) {
        s_sums[wave][0] = s;
        s_sums[wave][1] = c;
        s_sums[wave][2] = a;
    }
    __syncthreads();
    s = (s_sums[0][0] + s_sums[1][0]) + (s_sums[2][0] + s_sums[3][0]);
    c = (s_sums[0][1] + s_sums[1][1]) + (s_sums[2][1] + s_sums[3][1]);
    a = (s_sums[0][2] + s_sums[1][2]) + (s_sums[2][2] + s_sums[3][2]);
}

// What a row's outputs are, from its joined state and keys in LDS. Called by all threads.
__device__ __forceinline__ void write_row(const LogprobsParams& p, uint32_t row, float m, float s, float c, float a, float t,
                                          const uint64_t* s_keys) {
    const uint32_t tid = threadIdx.x;
    const bool none = !(fabsf(m) < INFINITY && s < INFINITY);  // NaN (in s), +inf, or nothing but -inf
    const float rest = (c - 1.0f) + s, log_z = log1pf(rest);
    if (tid == 0) {
        // (t is NaN where no segment held the target)
        if (p.logprobs) p.logprobs[row] = none ? NAN : (t - m) - log_z;
        if (p.entropy) p.entropy[row] = none ? NAN : log_z - a / (1.0f + rest);
    }
    if (tid < p.top_n) {
        const uint64_t k = s_keys[tid];
        const uint32_t o = (uint32_t)(k >> 32), u = o & 0x80000000u ? o & 0x7fffffffu : ~o;
        p.top_ids[(uint64_t)row * p.top_n + tid] = none ? -1 : (int32_t)~(uint32_t)k;
        p.top_logprobs[(uint64_t)row * p.top_n + tid] = none ? NAN : (__uint_as_float(u) - m) - log_z;
    }
}

template <int PER, bool VEC>
__global__ __launch_bounds__(kThreads) void logprobs_part_kernel(LogprobsParams p) {
    __shared__ uint64_t s_own[kThreads], s_list[PER * kAccept(kTop)], s_keys[kTop];
    __shared__ float s_max[4], s_sums[4][3];
    __shared__ uint32_t s_count;
    const uint32_t tid = threadIdx.x, row = blockIdx.x / p.n_segs, seg = blockIdx.x % p.n_segs;
    const uint32_t first = seg * (PER * kThreads);
    const float* x = p.logits + (uint64_t)row * p.row_stride;
    // element e of this thread: VEC: quads of 4, tid + 256 j; else single ones
    auto id_of = [&](int e) -> uint32_t {
        return first + (VEC ? 4 * (tid + kThreads * (e / 4)) + e % 4 : tid + kThreads * e);
    };
    float v[PER];
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < PER / 4; j++) {
            const uint32_t i = id_of(4 * j);
            float4 q = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (i + 3 < p.vocab) q = *(const float4*)(x + i);
            else {
                if (i < p.vocab) q.x = x[i];
                if (i + 1 < p.vocab) q.y = x[i + 1];
                if (i + 2 < p.vocab) q.z = x[i + 2];
            }
            v[4 * j] = q.x, v[4 * j + 1] = q.y, v[4 * j + 2] = q.z, v[4 * j + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < PER; e++) v[e] = id_of(e) < p.vocab ? x[id_of(e)] : -INFINITY;
    }
    const int32_t target = p.logprobs ? p.targets[row] : -1;
    const bool here = target >= 0 && (uint32_t)target < p.vocab && (uint32_t)target - first < PER * kThreads;
    const float t = here ? x[target] : NAN;
    float mx = -INFINITY;
    uint32_t at = id_of(0);  // of the thread's largest
#pragma unroll
    for (int e = 0; e < PER; e++)
        if (v[e] > mx) {
            mx = v[e];
            at = id_of(e);
        }
    s_own[tid] = at < p.vocab ? key_of(mx, at) : 0;
    const float wave_mx = wave_allreduce(mx, OpMax{});
    if ((tid & 63) == 0) s_max[tid >> 6] = wave_mx;
    if (tid == 0) s_count = 0;
    __syncthreads();
    const float m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    float s = 0.0f, c = 0.0f, a = 0.0f;
    if (m == -INFINITY) {  // (uniform) the largest of NaN and -inf is -inf
#pragma unroll
        for (int e = 0; e < PER; e++) s = v[e] == v[e] ? s : NAN;
    } else if (m < INFINITY) {
        uint32_t equal = 0;
#pragma unroll
        for (int e = 0; e < PER; e++) {
            const float d = v[e] - m, w = fast_exp2(d * kLog2e);
            a = __builtin_fmaf(fmaxf(d, -200.0f), w, a);  // exp(-200) is 0 here, and 0 * -200 is 0 where 0 * -inf is not
            s += d == 0.0f ? 0.0f : w;
            equal += d == 0.0f;
        }
        c = (float)equal;
    }
    if (p.top_n) {
        const uint64_t bound = find_bound(s_own, p.top_n);
        if (s_own[tid] >= bound) {
            // (below the form of -inf, where fewer than top_n threads hold a finite logit, a prefix is no float's)
            const uint32_t o = (uint32_t)(bound >> 32);
            const float least = o <= kLowest ? -INFINITY : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
#pragma unroll
            for (int e = 0; e < PER; e++)
                if (v[e] >= least && id_of(e) < p.vocab) {
                    const uint64_t k = key_of(v[e], id_of(e));
                    if (k >= bound) s_list[atomicAdd(&s_count, 1u)] = k;
                }
        }
    }
    block_sums(s, c, a, s_sums);
    if (p.top_n) order_top(s_list, s_count, p.top_n, s_keys);
    if (p.n_segs == 1) {
        write_row(p, row, m, s, c, a, t, s_keys);
        return;
    }
    if (tid == 0) p.states[(uint64_t)row * p.n_segs + seg] = SegState{m, s, c, a, t};
    if (tid < p.top_n) p.keys[((uint64_t)row * p.n_segs + seg) * p.top_n + tid] = s_keys[tid];
}

__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(LogprobsParams p) {
    __shared__ uint64_t s_own[kThreads], s_list[kTop * kAccept(kTop)], s_keys[kTop];
    __shared__ float s_state[4][2], s_sums[4][3];
    __shared__ uint32_t s_count;
    const uint32_t tid = threadIdx.x, row = blockIdx.x, n = p.top_n;
    const uint64_t* keys = p.keys + (uint64_t)row * p.n_segs * n;
    // The bound comes from every segment's first `depth` keys, 2 n of them at least; at most 256, as more
    // than one of each are taken from fewer than 2 n segments only.
    const uint32_t n_keys = p.n_segs * n, depth = n ? min(n, (2 * n + p.n_segs - 1) / p.n_segs) : 0;
    constexpr int kHeld = 8;  // keys a thread holds; it reads those past 256 * kHeld twice
    uint64_t held[kHeld];
    s_own[tid] = 0;
    SegState st{-INFINITY, 0.0f, 0.0f, 0.0f, NAN};
    if (tid < p.n_segs) st = p.states[(uint64_t)row * p.n_segs + tid];
#pragma unroll
    for (int i = 0; i < kHeld; i++) held[i] = tid + kThreads * i < n_keys ? keys[tid + kThreads * i] : 0;
    const float wave_m = wave_allreduce(st.m, OpMax{});
    const float wave_t = wave_allreduce(st.t == st.t ? st.t : -INFINITY, OpMax{});  // one segment holds it, or none
    const bool wave_has = __any(st.t == st.t);
    if (tid == 0) s_count = 0;
    __syncthreads();
    auto sample = [&](uint32_t i, uint64_t k) {
        const uint32_t seg = i / n, at = i - seg * n;
        if (at < depth) s_own[seg * depth + at] = k;
    };
#pragma unroll
    for (int i = 0; i < kHeld; i++)
        if (tid + kThreads * i < n_keys) sample(tid + kThreads * i, held[i]);
    for (uint32_t i = tid + kThreads * kHeld; i < n_keys; i += kThreads) sample(i, keys[i]);
    if ((tid & 63) == 0) {
        s_state[tid >> 6][0] = wave_m;
        s_state[tid >> 6][1] = wave_has ? wave_t : NAN;
    }
    __syncthreads();
    const float m = fmaxf(fmaxf(s_state[0][0], s_state[1][0]), fmaxf(s_state[2][0], s_state[3][0]));
    const float t = fmaxf(fmaxf(s_state[0][1], s_state[1][1]), fmaxf(s_state[2][1], s_state[3][1]));  // of those not NaN
    float s = st.s, c = 0.0f, a = 0.0f;
    if (st.m == m) {
        c = st.c;
        a = st.a;
    } else if (st.m > -INFINITY) {
        const float d = fmaxf(st.m - m, -200.0f), w = fast_exp2(d * kLog2e), z = st.s + st.c;
        s = z * w;
        a = w * __builtin_fmaf(d, z, st.a);
    }
    if (n) {
        const uint64_t bound = find_bound(s_own, n);
        auto take = [&](uint64_t k) {
            if (k >= bound) s_list[atomicAdd(&s_count, 1u)] = k;
        };
#pragma unroll
        for (int i = 0; i < kHeld; i++) take(held[i]);
        for (uint32_t i = tid + kThreads * kHeld; i < n_keys; i += kThreads) take(keys[i]);
    }
    block_sums(s, c, a, s_sums);
    if (n) order_top(s_list, s_count, n, s_keys);
    write_row(p, row, m, s, c, a, t, s_keys);
}

}  // namespace

int launch_token_logprobs(ds5_hip_ctx* ctx, const LogprobsLaunch& a) {
    // Segments of 8192 logits, or of 2048 where the longer ones would leave compute units idle, or be mostly empty:
    // one row of 32768 logits with 20 alternatives takes 10.2 us so, 2032 rows of 820 11.4 (17.2 in the longer).
    // A row that fits one segment needs no join: of 8192 logits 7.8 us, in four segments 10.4.
    uint32_t per = 32;
    uint64_t segs = (a.vocab + kLogprobsSegment - 1) / kLogprobsSegment;
    if (((segs > 1 && segs * a.n_rows < 256) || a.vocab <= 2048) && (a.vocab + 2047) / 2048 <= kMaxSegs) {
        per = 8;
        segs = (a.vocab + 2047) / 2048;
    }
    static_assert(32 * kThreads == kLogprobsSegment && DS5_LOGPROBS_MAX_VOCAB / kLogprobsSegment <= kMaxSegs, "a join thread per segment");
    LogprobsParams p{a.logits, a.targets, a.logprobs, a.entropy, a.top_ids, a.top_logprobs, a.vocab, a.row_stride, a.top_n,
                     (uint32_t)segs, nullptr, nullptr};
    if (segs > 1) {
        const size_t key_bytes = (size_t)a.n_rows * segs * a.top_n * sizeof(uint64_t);
        void* ws = nullptr;
        if (int rc = ds5_workspace(ctx, key_bytes + (size_t)a.n_rows * segs * sizeof(SegState), &ws)) return rc;
        p.keys = (uint64_t*)ws;
        p.states = (SegState*)((char*)ws + key_bytes);
    }
    const bool vec = ((uintptr_t)a.logits & 15u) == 0 && a.row_stride % 4 == 0;
    const dim3 grid((uint32_t)(segs * a.n_rows)), block(kThreads);
    const char* name = "logprobs_part_kernel";
    if (per == 32) {
        if (vec) DS5_TIMED_LAUNCH(ctx, name, (logprobs_part_kernel<32, true>), grid, block, 0, ctx->stream, p);
        else DS5_TIMED_LAUNCH(ctx, name, (logprobs_part_kernel<32, false>), grid, block, 0, ctx->stream, p);
    } else {
        if (vec) DS5_TIMED_LAUNCH(ctx, name, (logprobs_part_kernel<8, true>), grid, block, 0, ctx->stream, p);
        else DS5_TIMED_LAUNCH(ctx, name, (logprobs_part_kernel<8, false>), grid, block, 0, ctx->stream, p);
    }
    if (int rc = ds5_after_launch(ctx, name)) return rc;
    if (segs > 1) {
        DS5_TIMED_LAUNCH(ctx, "logprobs_join_kernel", logprobs_join_kernel, dim3(a.n_rows), block, 0, ctx->stream, p);
        return ds5_after_launch(ctx, "logprobs_join_kernel");
    }
    return DS5_OK;
}
