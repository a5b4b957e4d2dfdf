// k_paged.hip -- a ragged batch over the paged pool: its rows appended with norm and rotation
// (paged_append_kernel), and their causal attention (paged_attention_kernel).
//
// The pool is that of k_decode.hip's paged decode: f16 [n_kv_heads, n_pages * page_size, D],
// position p of sequence b in slot page_table[b][p / page_size] * page_size + p % page_size.
// Sequence b holds the batch's rows starts[b] .. starts[b + 1] - 1, its newest tokens.
#include "ds5_common.hpp"

namespace {

// ---------------------------------------------------------------------------
// Rows and sequences
// ---------------------------------------------------------------------------
struct RowInfo {
    bool held;     // a sequence holds the row
    bool ok;       // and its rows and length are in range
    uint32_t b;    // the sequence
    uint32_t pos;  // the row's position
};

// The sequence that holds row t, found by a whole wavefront: the number of entries of
// starts[1 ..] that are at most t, by 64 parts at a time (one round trip for up to 64
// sequences, two for 4096). starts that decrease can name a sequence that does not hold the
// row, which the last check sees.
__device__ __forceinline__ RowInfo find_row(const PagedBatch& p, uint32_t t, uint32_t lane) {
    uint32_t lo = 0, hi = p.n_seqs;  // starts[1 ..][lo, hi) are yet to be told apart
    while (lo < hi) {  // uniform; at most step - 1 entries stay
        const uint32_t step = (hi - lo + 63) / 64, first = lo + lane * step;
        const bool le = first < hi && p.starts[min(first + step, hi)] <= (int32_t)t;
        const uint32_t next = lo + (uint32_t)__popcll(__ballot(le)) * step;
        if (next < hi) hi = min(next + step, hi) - 1;  // the next part's last entry is above t
        lo = min(next, hi);
    }
    RowInfo r{};
    if (lo >= p.n_seqs) return r;
    const int64_t s0 = p.starts[lo], s1 = p.starts[lo + 1], len = p.seq_lens[lo];
    r.b = lo;
    r.held = s0 <= (int64_t)t && (int64_t)t < s1;
    r.ok = r.held && s0 >= 0 && s1 <= (int64_t)p.n_tokens && len >= s1 - s0 && len <= (int64_t)p.max_seq_len;
    if (r.ok) r.pos = (uint32_t)(len - s1 + (int64_t)t);
    return r;
}

// ---------------------------------------------------------------------------
// Append. A workgroup per row (token): D / 8 lanes take one head of q, k or v, lane m the
// rotation pairs 4 m .. 4 m + 3 (elements i and i + D / 2): the norm's sum is three or four
// DPP adds, the rotation needs no other lane. The angles are the token's, worked out once
// (turns in 64 bits, of which only the fraction matters, then sine and cosine of at most half
// a turn in 32 bits: 2e-7 off at any position) and shared through LDS while the heads' loads
// are in flight. Memory bound: every element is read once and written once.
// ---------------------------------------------------------------------------
constexpr int kAppendThreads = 256;

template <int N>
__device__ __forceinline__ float lanes_sum(float v) {  // over N = 8 or 16 aligned lanes, on each of them
    v += dpp_mov<0xB1>(v);
    v += dpp_mov<0x4E>(v);
    v += dpp_mov<0x141>(v);
    if constexpr (N == 16) v += dpp_mov<0x140>(v);
    return v;
}

template <int D, bool Q16>
__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(PagedAppendLaunch a, RopeTurns turns) {
    constexpr int LPR = D / 8, GROUPS = kAppendThreads / LPR, UN = 2;
    __shared__ float s_cos[D / 2], s_sin[D / 2];
    const PagedBatch& p = a.batch;
    const uint32_t tid = threadIdx.x, lane = tid & 63, t = blockIdx.x;
    const uint32_t m = tid % LPR, grp = tid / LPR;
    const uint32_t hq = a.q ? p.n_q_heads : 0, hkv = p.n_kv_heads, heads = hq + 2 * hkv;

    const RowInfo r = find_row(p, t, lane);
    if (!r.held) return;  // uniform
    bool ok = r.ok;
    uint64_t slot = 0;
    if (ok) {
        const int32_t pg = p.page_table[(uint64_t)r.b * p.max_pages + r.pos / p.page_size];
        ok = pg >= 0 && (uint32_t)pg < p.n_pages;
        slot = (uint64_t)(uint32_t)pg * p.page_size + r.pos % p.page_size;
    }
    if (tid < D / 2) {
        double turn = (double)r.pos * turns.inv[tid];
        turn -= rint(turn);
        const float f = 2.0f * (float)turn;
        s_cos[tid] = cospif(f);
        s_sin[tid] = sinpif(f);
    }
    __syncthreads();
    const uint64_t slots = (uint64_t)p.n_pages * p.page_size;
    const float4 c4 = *(const float4*)(s_cos + 4 * m), s4 = *(const float4*)(s_sin + 4 * m);
    for (uint32_t h0 = grp; h0 < heads; h0 += UN * GROUPS) {
        float4 x0[UN], x1[UN], w0[UN], w1[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const uint32_t h = min(h0 + u * GROUPS, heads - 1);
            const float* src = h < hq         ? a.q + ((uint64_t)t * hq + h) * D
                               : h < hq + hkv ? a.k + ((uint64_t)t * hkv + (h - hq)) * D
                                              : a.v + ((uint64_t)t * hkv + (h - hq - hkv)) * D;
            const float* w = h < hq ? a.q_norm : a.k_norm;
            x0[u] = *(const float4*)(src + 4 * m);
            x1[u] = *(const float4*)(src + D / 2 + 4 * m);
            if (w && h < hq + hkv) {
                w0[u] = *(const float4*)(w + 4 * m);
                w1[u] = *(const float4*)(w + D / 2 + 4 * m);
            }
        }
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const uint32_t h = h0 + u * GROUPS;
            if (h >= heads) break;
            float4 y0 = x0[u], y1 = x1[u];
            if (h < hq + hkv) {
                if (h < hq ? a.q_norm != nullptr : a.k_norm != nullptr) {
                    const float ss = (y0.x * y0.x + y0.y * y0.y) + (y0.z * y0.z + y0.w * y0.w) +
                                     ((y1.x * y1.x + y1.y * y1.y) + (y1.z * y1.z + y1.w * y1.w));
                    const float inv = 1.0f / sqrtf(lanes_sum<LPR>(ss) / (float)D + a.eps);
                    y0 = float4{y0.x * inv * w0[u].x, y0.y * inv * w0[u].y, y0.z * inv * w0[u].z, y0.w * inv * w0[u].w};
                    y1 = float4{y1.x * inv * w1[u].x, y1.y * inv * w1[u].y, y1.z * inv * w1[u].z, y1.w * inv * w1[u].w};
                }
                const float4 z0 = y0, z1 = y1;
                y0 = float4{z0.x * c4.x - z1.x * s4.x, z0.y * c4.y - z1.y * s4.y, z0.z * c4.z - z1.z * s4.z,
                            z0.w * c4.w - z1.w * s4.w};
                y1 = float4{z0.x * s4.x + z1.x * c4.x, z0.y * s4.y + z1.y * c4.y, z0.z * s4.z + z1.z * c4.z,
                            z0.w * s4.w + z1.w * c4.w};
            }
            if (h < hq) {
                if (!ok) y0 = y1 = float4{NAN, NAN, NAN, NAN};
                if constexpr (Q16) {
                    f16* dst = (f16*)a.q_out + ((uint64_t)t * hq + h) * D;
                    *(f16x4*)(dst + 4 * m) = f16x4{(f16)y0.x, (f16)y0.y, (f16)y0.z, (f16)y0.w};
                    *(f16x4*)(dst + D / 2 + 4 * m) = f16x4{(f16)y1.x, (f16)y1.y, (f16)y1.z, (f16)y1.w};
                } else {
                    float* dst = (float*)a.q_out + ((uint64_t)t * hq + h) * D;
                    *(float4*)(dst + 4 * m) = y0;
                    *(float4*)(dst + D / 2 + 4 * m) = y1;
                }
            } else if (ok) {
                const bool k = h < hq + hkv;
                f16* dst = (k ? a.k_pool : a.v_pool) + ((uint64_t)(h - hq - (k ? 0 : hkv)) * slots + slot) * D;
                *(f16x4*)(dst + 4 * m) = f16x4{(f16)y0.x, (f16)y0.y, (f16)y0.z, (f16)y0.w};
                *(f16x4*)(dst + D / 2 + 4 * m) = f16x4{(f16)y1.x, (f16)y1.y, (f16)y1.z, (f16)y1.w};
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Attention: a wavefront per (row, q head), 64 positions at a time: each lane one position's
// score, then the weights' sum over the positions with two or one elements of v per lane.
// ---------------------------------------------------------------------------
template <int D, bool Q16>
__global__ __launch_bounds__(256) void paged_attention_kernel(PagedAttentionLaunch a) {
    __shared__ float s_q[4][D];
    const PagedBatch& p = a.batch;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t item = (uint64_t)blockIdx.x * 4 + wave;
    const uint32_t t = (uint32_t)(item / p.n_q_heads), h = (uint32_t)(item % p.n_q_heads);
    if (t >= p.n_tokens) return;
    const uint32_t kvh = h / (p.n_q_heads / p.n_kv_heads);
    const uint64_t slots = (uint64_t)p.n_pages * p.page_size;
    const uint64_t row = ((uint64_t)t * p.n_q_heads + h) * D;
    const RowInfo r = find_row(p, t, lane);
    if (!r.held) return;
    for (uint32_t i = lane; i < D; i += 64) s_q[wave][i] = Q16 ? (float)((const f16*)a.q)[row + i] : ((const float*)a.q)[row + i];
    __builtin_amdgcn_wave_barrier();
    const uint32_t L = r.ok ? r.pos + 1 : 0;
    float mx = -INFINITY, l = 0.0f, o[D / 64] = {};
    bool bad = !r.ok;
    for (uint32_t j0 = 0; j0 < L; j0 += 64) {
        const uint32_t j = min(j0 + lane, L - 1);
        const int32_t pg = p.page_table[(uint64_t)r.b * p.max_pages + j / p.page_size];
        const bool in = pg >= 0 && (uint32_t)pg < p.n_pages;
        bad = bad || !in;
        const uint64_t at = (uint64_t)kvh * slots + (uint64_t)(in ? pg : 0) * p.page_size + j % p.page_size;
        float s = 0.0f;
        for (int i = 0; i < D; i++) s += s_q[wave][i] * (float)a.k_pool[at * D + i];
        s = j0 + lane < L ? s * a.scale : -INFINITY;
        const float m_new = fmaxf(mx, wave_allreduce(s, OpMax{}));
        const float alpha = expf(mx - m_new), w = expf(s - m_new);
        l = l * alpha + wave_allreduce(w, OpAdd{});
        for (int e = 0; e < D / 64; e++) o[e] *= alpha;
        mx = m_new;
        const uint32_t n = min(64u, L - j0);
        for (uint32_t k = 0; k < n; k++) {
            const float wk = __shfl(w, (int)k, 64);
            const uint64_t ak = __shfl(at, (int)k, 64);
            for (int e = 0; e < D / 64; e++) o[e] += wk * (float)a.v_pool[ak * D + lane + 64 * e];
        }
    }
    bad = __ballot(bad) != 0;
    for (int e = 0; e < D / 64; e++) a.out[row + lane + 64 * e] = bad ? NAN : o[e] / l;
}

}  // namespace

int launch_paged_append(ds5_hip_ctx* ctx, const PagedAppendLaunch& a) {
    const dim3 grid(a.batch.n_tokens), block(kAppendThreads);
    const char* name = "paged_append_kernel";
    if (a.batch.head_dim == 128) {
        if (a.q_f16) DS5_TIMED_LAUNCH(ctx, name, (paged_append_kernel<128, true>), grid, block, 0, ctx->stream, a, *a.turns);
        else DS5_TIMED_LAUNCH(ctx, name, (paged_append_kernel<128, false>), grid, block, 0, ctx->stream, a, *a.turns);
    } else {
        if (a.q_f16) DS5_TIMED_LAUNCH(ctx, name, (paged_append_kernel<64, true>), grid, block, 0, ctx->stream, a, *a.turns);
        else DS5_TIMED_LAUNCH(ctx, name, (paged_append_kernel<64, false>), grid, block, 0, ctx->stream, a, *a.turns);
    }
    return ds5_after_launch(ctx, name);
}

int launch_paged_attention(ds5_hip_ctx* ctx, const PagedAttentionLaunch& a) {
    const uint64_t items = (uint64_t)a.batch.n_tokens * a.batch.n_q_heads;
    const dim3 grid((uint32_t)((items + 3) / 4)), block(256);
    const char* name = "paged_attention_kernel";
    if (a.batch.head_dim == 128) {
        if (a.q_f16) DS5_TIMED_LAUNCH(ctx, name, (paged_attention_kernel<128, true>), grid, block, 0, ctx->stream, a);
        else DS5_TIMED_LAUNCH(ctx, name, (paged_attention_kernel<128, false>), grid, block, 0, ctx->stream, a);
    } else {
        if (a.q_f16) DS5_TIMED_LAUNCH(ctx, name, (paged_attention_kernel<64, true>), grid, block, 0, ctx->stream, a);
        else DS5_TIMED_LAUNCH(ctx, name, (paged_attention_kernel<64, false>), grid, block, 0, ctx->stream, a);
    }
    return ds5_after_launch(ctx, name);
}
