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
// segments' states. Memory bound: the logits are read once.
//
// Selection by unique 64-bit keys (the logit in an order-preserving form above the complement of
// its index, so that equal logits fall to the lower index): every thread's largest key; the
// top_n-th largest of those is a bound that at least top_n elements reach, and only the elements
// of the top_n threads whose largest reaches it can (at most PER * top_n; a few more than top_n
// as a rule). They are gathered in LDS and ordered by counting, for each, those above it. The
// join does the same with each segment's sorted keys in place of a thread's elements.
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

__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 orders as +0
    const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return ((uint64_t)o << 32) | (uint32_t)~id;
}

__device__ __forceinline__ uint64_t kmax(uint64_t a, uint64_t b) { return a > b ? a : b; }

// The n largest of the keys that the threads' lists hold, in descending order into out[0, n) (0
// where there are fewer). own: the thread's largest key (0: none); each(f) calls f for the keys
// of its list that may reach `bound`. All threads call it.
template <class Each>
__device__ __forceinline__ void select_top(uint64_t own, uint32_t n, uint64_t* s_own, uint64_t* s_list, uint32_t* s_count,
                                           uint64_t* out, Each each) {
    const uint32_t tid = threadIdx.x;
    uint64_t* s_bound = s_own + kThreads;
    s_own[tid] = own;
    if (tid == 0) {
        *s_bound = 1;  // any key
        *s_count = 0;
    }
    if (tid < n) out[tid] = 0;
    __syncthreads();
    uint32_t above = 0;
    for (int i = 0; i < kThreads; i++) above += s_own[i] > own;
    if (own && above == n - 1) *s_bound = own;  // keys are unique: one thread at most
    __syncthreads();
    const uint64_t bound = *s_bound;
    if (own >= bound)
        each(bound, [&](uint64_t k) {
            if (k >= bound) s_list[atomicAdd(s_count, 1u)] = k;
        });
    __syncthreads();
    const uint32_t count = *s_count;
    for (uint32_t i = tid; i < count; i += kThreads) {
        const uint64_t k = s_list[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < count; j++) rank += s_list[j] > k;
        if (rank < n) out[rank] = k;
    }
    __syncthreads();
}

// op over the workgroup, on every thread; s_red: 4 floats, free again after a barrier
template <class F>
__device__ __forceinline__ float block_reduce(float v, F op, float* s_red) {
    v = wave_allreduce(v, op);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
    __syncthreads();
    return op(op(s_red[0], s_red[1]), op(s_red[2], s_red[3]));
}

// What a row's outputs are, from its joined state and keys in LDS. Called by all threads.
__device__ __forceinline__ void write_row(const LogprobsParams& p, uint32_t row, float m, float s, float c, float a, float t,
                                          const uint64_t* s_keys) {
    const uint32_t tid = threadIdx.x;
    const bool none = !(fabsf(m) < INFINITY);  // NaN, +inf, or nothing but -inf
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
    __shared__ uint64_t s_own[kThreads + 1], s_list[PER * kTop], s_keys[kTop];
    __shared__ float s_red[4];
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
    float mx = -INFINITY;
    bool odd = false;
#pragma unroll
    for (int e = 0; e < PER; e++) {
        mx = fmaxf(mx, v[e]);
        odd = odd || !(v[e] < INFINITY);
    }
    if (odd) mx = INFINITY;  // NaN or +inf
    const float m = block_reduce(mx, OpMax{}, s_red);
    float s = 0.0f, c = 0.0f, a = 0.0f;
    if (fabsf(m) < INFINITY) {  // uniform
#pragma unroll
        for (int e = 0; e < PER; e++) {
            const float d = fmaxf(v[e] - m, -200.0f);  // exp(-200) is 0 here, and 0 * -200 is 0 where 0 * -inf is not
            const float w = fast_exp2(d * kLog2e);
            a = __builtin_fmaf(d, w, a);
            s += v[e] == m ? 0.0f : w;
            c += v[e] == m ? 1.0f : 0.0f;
        }
        s = block_reduce(s, OpAdd{}, s_red);
        c = block_reduce(c, OpAdd{}, s_red);
        a = block_reduce(a, OpAdd{}, s_red);
    }
    if (p.top_n) {
        uint64_t own = 0;
#pragma unroll
        for (int e = 0; e < PER; e++)
            if (id_of(e) < p.vocab) own = kmax(own, key_of(v[e], id_of(e)));
        select_top(own, p.top_n, s_own, s_list, &s_count, s_keys, [&](uint64_t, auto take) {
#pragma unroll
            for (int e = 0; e < PER; e++)
                if (id_of(e) < p.vocab) take(key_of(v[e], id_of(e)));
        });
    }
    const int32_t target = p.logprobs ? p.targets[row] : -1;
    const bool here = target >= 0 && (uint32_t)target < p.vocab && (uint32_t)target - first < PER * kThreads;
    const float t = here ? x[target] : NAN;
    if (p.n_segs == 1) {
        write_row(p, row, m, s, c, a, t, s_keys);
        return;
    }
    if (tid == 0) p.states[(uint64_t)row * p.n_segs + seg] = SegState{m, s, c, a, t};
    if (tid < p.top_n) p.keys[((uint64_t)row * p.n_segs + seg) * p.top_n + tid] = s_keys[tid];
}

__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(LogprobsParams p) {
    __shared__ uint64_t s_own[kThreads + 1], s_list[kTop * kTop], s_keys[kTop];
    __shared__ float s_red[4];
    __shared__ uint32_t s_count;
    const uint32_t tid = threadIdx.x, row = blockIdx.x;
    SegState st{-INFINITY, 0.0f, 0.0f, 0.0f, NAN};
    const uint64_t* keys = nullptr;
    if (tid < p.n_segs) {
        st = p.states[(uint64_t)row * p.n_segs + tid];
        keys = p.keys + ((uint64_t)row * p.n_segs + tid) * p.top_n;
    }
    const float m = block_reduce(st.m, OpMax{}, s_red);
    float s = 0.0f, c = 0.0f, a = 0.0f;
    if (st.m == m) {
        s = st.s;
        c = st.c;
        a = st.a;
    } else if (st.m > -INFINITY) {
        const float d = fmaxf(st.m - m, -200.0f), w = fast_exp2(d * kLog2e), z = st.s + st.c;
        s = z * w;
        a = w * __builtin_fmaf(d, z, st.a);
    }
    s = block_reduce(s, OpAdd{}, s_red);
    c = block_reduce(c, OpAdd{}, s_red);
    a = block_reduce(a, OpAdd{}, s_red);
    const float t = block_reduce(st.t == st.t ? st.t : -INFINITY, OpMax{}, s_red);  // one segment holds it, or none
    const float held = block_reduce(st.t == st.t ? 1.0f : 0.0f, OpMax{}, s_red);
    if (p.top_n)
        select_top(keys ? keys[0] : 0, p.top_n, s_own, s_list, &s_count, s_keys, [&](uint64_t bound, auto take) {
            for (uint32_t i = 0; i < p.top_n && keys[i] >= bound; i++) take(keys[i]);
        });
    write_row(p, row, m, s, c, a, held > 0.0f ? t : NAN, s_keys);
}

}  // namespace

int launch_token_logprobs(ds5_hip_ctx* ctx, const LogprobsLaunch& a) {
    // Segments of 8192 logits, or of 2048 where the longer ones would leave compute units idle.
    uint32_t per = 32;
    uint64_t segs = (a.vocab + 8191) / 8192;
    if (segs * a.n_rows < 256 && (a.vocab + 2047) / 2048 <= kMaxSegs) {
        per = 8;
        segs = (a.vocab + 2047) / 2048;
    }
    static_assert((DS5_LOGPROBS_MAX_VOCAB + 8191) / 8192 <= kMaxSegs, "a join thread per segment");
    LogprobsParams p{a.logits, a.targets, a.logprobs, a.entropy, a.top_ids, a.top_logprobs, a.vocab, a.row_stride, a.top_n,
                     (uint32_t)segs, nullptr, nullptr};
    if (segs * a.n_rows > INT32_MAX) return ds5_fail(ctx, DS5_SHAPE_MISMATCH, "token_logprobs: too many rows");
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
