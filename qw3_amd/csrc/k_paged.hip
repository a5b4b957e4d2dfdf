// k_paged.hip -- a ragged batch over the paged pool: its rows appended with norm and rotation
// (paged_append_kernel), and their causal attention (paged_attention_kernel).
//
// The pool is that of k_decode.hip's paged decode: f16 [n_kv_heads, n_pages * page_size, D],
// position p of sequence b in slot page_table[b][p / page_size] * page_size + p % page_size.
// Sequence b holds the batch's rows starts[b] .. starts[b + 1] - 1, its newest tokens.
#include <type_traits>

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
// are in flight. Memory bound: every element is read once and written once. 3498 tokens of ragged
// prompts (32 + 2 x 4 heads of 128 from f32 to f16, 107 MB) take 22.3 us, 4.8 TB/s, a large copy's
// rate; one token 4.3 us, a launch and four dependent loads.
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
// Attention. Row (t, head) of a sequence's new tokens:
//   out = sum_p w_p v_p / sum_p w_p, w_p = exp2(scale log2(e) q . k_p - reference), p up to its own position.
// One pass over the positions with the running reference and sums of a softmax. A kv head's query rows
// (token * group + head) make tiles of 128, so that every K and V row is read once for 128 of them, on
// v_mfma_f32_32x32x16_f16 with f32 accumulators. f32 accuracy from f16 operands: q (where it is f32) and
// the weights are hi + lo pairs, two products each, 22 bits (of the weights: see kHead); K and V are f16 as they are.
//
// How a batch is divided is known on the device only (starts, seq_lens): every workgroup works out its own
// part of one line of all tiles' work, and parts of a tile are merged by a second kernel (ds5_index.hpp has
// the line; the plan takes 2 us). Two forms of a tile: up to 32 rows (decode) the eight wavefronts take
// blocks of 32 positions in turn, each with K and V of its own in LDS; above, four wavefronts of 32 rows
// each share a 64-position step of a four-stage LDS ring with four others of the same rows, whose sums
// are folded through LDS at the end. K and V come by direct-to-LDS loads, a block or three steps ahead.
//
// What bounds it. Long decode: memory; 32 sequences of 0.5 .. 16 K positions (4 kv heads of 128, 584 MB)
// 110 us, 5.3 TB/s. Prompts: the matrix cores at the power that they may draw; 64 positions of 128 rows
// take 1.3 us with f16 q (48 products of 32 cycles a wavefront pair) and 1.5 with f32 q (64): 1.2 and 1.4
// PFLOP/s issued, above a large library product's 1.14; leaving out the exponentials, the V reads or the
// barriers changed neither. A prompt of 2048 65 us, 203 f32 tokens at 6000 86 + 8 merging. Small calls:
// the chain of launch, plan, page table, q, K and V through LDS, and output, 9 .. 13 us and 4 for the merge.
// ---------------------------------------------------------------------------
constexpr int kThreads = 512, kWaves = 8;
constexpr int kRows = ds5idx::kPbRows, kNarrow = ds5idx::kPbNarrow;
constexpr uint32_t kMaxSeqs = DS5_PAGED_MAX_SEQS;
constexpr uint32_t kMaxGrid = 256;
constexpr uint32_t kWindow = 1024;  // groups of 16 positions whose place in the pool is in LDS at a time
// Weights are exp2(score - reference): the reference starts 2^8 below the row's maximum and moves
// when a weight would pass 2^15. In f16 hi + lo a weight keeps its 22 bits down to 2^-3, 2^-11 of the
// largest (lo is subnormal below), and is within 2^-25, 2^-33 of the largest, from there on: n positions
// of such weights move a row by n 2^-33 of the values' size at most, 4e-6 for 2^15. (A reference nearer
// to 2^15 would keep 22 bits further down and move with nearly every new maximum.)
constexpr float kHead = 8.0f, kMove = 15.0f;

struct MergeDesc {
    uint32_t row0, kvh, token0;
};

struct AttnParams {
    PagedAttentionLaunch a;
    uint32_t group;
    double inv_group, inv_page, inv_heads;  // 1 / group, 1 / page_size, 1 / n_kv_heads
    bool whole;        // no tile is cut
    float* part_o;     // [2 * workgroups, kRows, D]: slot 2 w the part that workgroup w continues, 2 w + 1 the one it begins
    float2* part_ml;   // [2 * workgroups, kRows]: reference and sum
    // [workgroups]: of the tile that the workgroup begins and does not end (0: none) its rows, and above them the
    // last workgroup with a part of it: the parts are this one's head part, then those of w + 1 .. last. (In a word
    // of its own, as every workgroup of the merge reads them all: 20 bytes each made it 17 us instead of 4.)
    uint32_t* heads;
    MergeDesc* descs;
};

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

// The same value, worked out anew where it is used: the compiler otherwise keeps what follows from it in
// registers across the loops, and spills.
__device__ __forceinline__ uint32_t here(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}

__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
    return ((uint64_t)uniform((uint32_t)(v >> 32)) << 32) | uniform((uint32_t)v);
}

// Sums over the wavefront's lanes up to and with this one, in six DPP adds (rows of 16 lanes by shifts of 1, 2, 4
// and 8, then lane 15 of a row to the next row and lane 31 to the upper half; a lane without a source adds 0).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_or_0(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or_0(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)dpp_or_0<CTRL, ROWS>((uint32_t)(u >> 32)) << 32 | dpp_or_0<CTRL, ROWS>((uint32_t)u));
}
template <class T>
__device__ __forceinline__ T sums_upto(T v) {
    v += dpp_or_0<0x111, 0xF>(v);
    v += dpp_or_0<0x112, 0xF>(v);
    v += dpp_or_0<0x114, 0xF>(v);
    v += dpp_or_0<0x118, 0xF>(v);
    v += dpp_or_0<0x142, 0xA>(v);
    v += dpp_or_0<0x143, 0xC>(v);
    return v;
}

template <int N>
__device__ __forceinline__ void wait_loads() {  // at most N vector-memory operations of the wavefront in flight
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Hi and lo f16 of two values: 22 bits of each.
__device__ __forceinline__ void split2(float x0, float x1, f16x2& hi, f16x2& lo) {
    hi = f16x2{(f16)x0, (f16)x1};
    lo = f16x2{(f16)(x0 - (float)hi[0]), (f16)(x1 - (float)hi[1])};
}
// The same of two weights in three instructions: a packed conversion that rounds towards 0, and each
// residual x - hi as a mixed-precision fma that rounds its result to f16.
__device__ __forceinline__ void split2_weights(float x0, float x1, f16x2& hi, f16x2& lo) {
    hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x0, x1));
    const uint32_t h = __builtin_bit_cast(uint32_t, hi);
    uint32_t l;
    asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixhi_f16 %0, %1, -1.0, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=&v"(l)
        : "v"(h), "v"(x0), "v"(x1));
    lo = __builtin_bit_cast(f16x2, l);
}

// The largest of a block's 16 scores on both lanes of a row. max3 as asm takes the products as they are
// (compiled from fmaxf each operand is canonicalised first); the first maximum is compiled, so that it
// waits for the products' result, and the others depend on it.
__device__ __forceinline__ float row_max(const f32x16& S) {
    float a = fmaxf(S[0], S[15]);
    asm("v_max3_f32 %0, %0, %1, %2\n\tv_max3_f32 %0, %0, %3, %4\n\tv_max3_f32 %0, %0, %5, %6\n\t"
        "v_max3_f32 %0, %0, %7, %8\n\tv_max3_f32 %0, %0, %9, %10\n\tv_max3_f32 %0, %0, %11, %12\n\t"
        "v_max3_f32 %0, %0, %13, %14"
        : "+v"(a)
        : "v"(S[1]), "v"(S[2]), "v"(S[3]), "v"(S[4]), "v"(S[5]), "v"(S[6]), "v"(S[7]), "v"(S[8]), "v"(S[9]), "v"(S[10]), "v"(S[11]),
          "v"(S[12]), "v"(S[13]), "v"(S[14]));
    return swap32_op(a, OpMax{});
}

template <int D, bool Q16>
struct Attn {
    static constexpr int KS = D / 16, DT = D / 32, RB = 2 * D;
    static constexpr int NB = 16 * RB / 1024;      // direct-to-LDS loads of a group of 16 rows
    static constexpr int HALF = 32 * RB;           // bytes of 32 rows
    static_assert(kRows * D * 4 <= kWaves * HALF, "a tile's query rows fit half of the area");
    static constexpr int AREA = kWaves * 2 * HALF; // K and V of a block for each wavefront, or four stages of two blocks
    static constexpr int CH = D / 4;               // float4 of an O row

    f32x16 O[DT];
    f16x8 qh[KS], ql[Q16 ? 1 : KS];
    float fac;       // score = product * fac, log2 units
    float m, l;      // reference, this lane's part of the sum
    uint32_t lim;    // the row's last position
    uint32_t koff, voff;  // lane's offsets of a row group's first load

    // Loads the 8 rows from `row` (half a group) into 8 * RB bytes of LDS.
    template <bool V>
    __device__ __forceinline__ static void load_half(uint32_t lds, const f16* row, uint32_t off) {
        const uint64_t base = uniform64((uint64_t)row);
        const uint32_t o1 = V ? off : off ^ 64;
        if constexpr (NB == 4)
            asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2\n\t"
                         "global_load_lds_dwordx4 %1, %2 offset:1024" ::"v"(off), "v"(o1), "s"(base), "s"(uniform(lds))
                         : "m0", "memory");
        else
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(uniform(lds))
                         : "m0", "memory");
    }

    // The lane's 8 elements of each k-step of its query row, at element `from` of q: fetched, and made
    // the products' operands once they are here.
    struct Query {
        f16x8 h[Q16 ? KS : 1];
        float4 x0[Q16 ? 1 : KS], x1[Q16 ? 1 : KS];
    };
    __device__ __forceinline__ static void fetch_q(Query& q, const AttnParams& p, uint64_t from) {
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            if constexpr (Q16) {
                q.h[ks] = *(const f16x8*)((const f16*)p.a.q + from + 16 * ks);
            } else {
                const float* src = (const float*)p.a.q + from + 16 * ks;
                q.x0[ks] = *(const float4*)src;
                q.x1[ks] = *(const float4*)(src + 4);
            }
        }
    }
    // The rows of a wide tile through LDS, where their loads run along rows (in the operands' layout each load
    // instruction touches 64 cache lines: 3.7 us of a tile's 128 rows of f32): wavefront w loads rows 16 w ..
    // 16 w + 15, 16-byte chunk c of row r into the row's slot c ^ qswz(r).
    static constexpr int QB = D * (Q16 ? 2 : 4), QC = QB / 16;
    __device__ __forceinline__ static uint32_t qswz(uint32_t r) { return QC == 8 ? (r >> 1) & 7 : r & (QC - 1); }
    template <class RowOf>
    __device__ __forceinline__ static void stage_q(uint32_t lds, const void* q, uint32_t wave, uint32_t lane, RowOf row_of) {
#pragma unroll
        for (int j = 0; j < 16 * QB / 1024; j++) {
            const uint32_t at = 1024 * j + 16 * lane, r = 16 * wave + at / QB, slot = at % QB / 16;
            const char* src = (const char*)q + row_of(r) * QB + (slot ^ qswz(r)) * 16;
            asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src),
                         "s"(uniform(lds + 16 * wave * QB + 1024 * j))
                         : "m0", "memory");
        }
    }
    __device__ __forceinline__ static void staged_q(Query& q, const char* sq, uint32_t r, uint32_t h) {
        const char* row = sq + r * QB;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            if constexpr (Q16) {
                q.h[ks] = *(const f16x8*)(row + ((2 * ks + h) ^ qswz(r)) * 16);
            } else {
                q.x0[ks] = *(const float4*)(row + ((4 * ks + 2 * h) ^ qswz(r)) * 16);
                q.x1[ks] = *(const float4*)(row + ((4 * ks + 2 * h + 1) ^ qswz(r)) * 16);
            }
        }
    }
    __device__ __forceinline__ void form_q(const Query& q, float scale) {
        // fac stays above 0 (a negative scale goes into the row's sign), so that the largest product is
        // the largest score and -inf stays -inf; a scale of NaN stays NaN
        const bool minus = scale < 0.0f;
        auto positive = [](float x) { return x < 1e-37f ? 1e-37f : x; };
        if constexpr (Q16) {
            fac = positive(fabsf(scale) * kLog2e);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) qh[ks] = minus ? -q.h[ks] : q.h[ks];
        } else {
            // the row times a power of two that brings its largest element to 2^13 .. 2^14: whatever its
            // size the operands hold 22 bits of elements down to 2^-2, 2^-16 of the largest, and smaller
            // ones (lo is subnormal) to within 2^-25, 2^-38 of it
            float big = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
                big = fmaxf(big, fmaxf(fmaxf(fmaxf(fabsf(q.x0[ks].x), fabsf(q.x0[ks].y)), fmaxf(fabsf(q.x0[ks].z), fabsf(q.x0[ks].w))),
                                       fmaxf(fmaxf(fabsf(q.x1[ks].x), fabsf(q.x1[ks].y)), fmaxf(fabsf(q.x1[ks].z), fabsf(q.x1[ks].w)))));
            big = swap32_op(big, OpMax{});
            const int e = big > 0.0f && big < INFINITY ? __builtin_amdgcn_frexp_expf(big) - 14 : 0;
            fac = positive(ldexpf(fabsf(scale), e) * kLog2e);
            const float unit = minus ? -1.0f : 1.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const float x[8] = {q.x0[ks].x, q.x0[ks].y, q.x0[ks].z, q.x0[ks].w, q.x1[ks].x, q.x1[ks].y, q.x1[ks].z, q.x1[ks].w};
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    f16x2 hi, lo;
                    split2(ldexpf(x[i] * unit, -e), ldexpf(x[i + 1] * unit, -e), hi, lo);
                    qh[ks][i] = hi[0], qh[ks][i + 1] = hi[1];
                    ql[ks][i] = lo[0], ql[ks][i + 1] = lo[1];
                }
            }
        }
    }

    // Loads the 16 rows from `row` of the pool (rows of RB bytes) into 16 * RB bytes of LDS: a load's
    // immediate offset counts for both addresses, and load b's lanes read `off` with bit 6 (b's own
    // part of the K rows' swizzle) turned.
    template <bool V>
    __device__ __forceinline__ static void load_group(uint32_t lds, const f16* row, uint32_t off) {
        const uint64_t base = uniform64((uint64_t)row);
        const uint32_t o1 = V ? off : off ^ 64, o2 = V ? off : off ^ 128, o3 = V ? off : off ^ 192;
        if constexpr (NB == 4)
            asm volatile("s_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %4\n\t"
                         "global_load_lds_dwordx4 %1, %4 offset:1024\n\tglobal_load_lds_dwordx4 %2, %4 offset:2048\n\t"
                         "global_load_lds_dwordx4 %3, %4 offset:%6" ::"v"(off), "v"(o1), "v"(o2), "v"(o3), "s"(base),
                         "s"(uniform(lds)), "n"(3 * 1024)
                         : "m0", "memory");
        else
            asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2\n\t"
                         "global_load_lds_dwordx4 %1, %2 offset:1024" ::"v"(off), "v"(o1), "s"(base), "s"(uniform(lds))
                         : "m0", "memory");
    }

    // A block is 32 positions; its products' operands come from LDS:
    //   S^T [32 positions x 32 rows] = K . Q^T     O^T [D x 32 rows] += V^T . P^T    v_mfma_f32_32x32x16_f16
    // With S transposed a lane (r32, h) holds 16 scores of query row r32, score e that of position
    // 8 (e / 4) + 4 h + e % 4, and the P^T operand is the lane's own weights.
    struct Lane {
        uint32_t k, v;  // byte offsets of the lane's operands: the block's K row r32, V rows of the transpose read
        __device__ __forceinline__ explicit Lane(uint32_t lane) {
            const uint32_t r32 = lane & 31, h = lane >> 5, i16 = lane & 15, g16 = lane >> 4;
            k = r32 * RB + (ds5idx::pb_swz(D, false, r32) ^ h) * 16;
            v = (4 * h + (i16 >> 2)) * RB +
                ((2 * (g16 & 1) + ((i16 & 3) >> 1)) ^ ds5idx::pb_swz(D, true, i16 >> 2)) * 16 + 8 * (i16 & 1);
        }
    };
    // Addresses: a block's base plus the lane's offset, then the swizzled chunk by xor (a block begins on a
    // multiple of the row's RB bytes, so that xor in the low bits stays in the row).
    __device__ __forceinline__ static f16x8 kread(uint32_t k, int ks) {
        return *(const __attribute__((address_space(3))) f16x8*)(uintptr_t)(k ^ (32 * ks));
    }
    // positions 16 s + [0, 16): the transpose read gives lane i of 16 column i of 4 rows; element jj of the
    // operand is position 16 s + 8 (jj / 4) + 4 h + jj % 4, as the weights lie
    __device__ __forceinline__ static f16x8 vread(uint32_t v, int s, int dt) {
        typedef __attribute__((__vector_size__(4 * sizeof(__fp16)))) __fp16 v4h;
        typedef __attribute__((address_space(3))) v4h lds_v4h;
        const uint32_t at = (v ^ (64 * dt)) + 16 * s * RB;
        const f16x4 a = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_v4h*)(uintptr_t)at));
        const f16x4 b = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_v4h*)(uintptr_t)(at + 8 * RB)));
        return f16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
    __device__ __forceinline__ void product(f32x16& S, const f16x8& k, int ks) const {
        S = mfma_32x32x16(k, qh[ks], S);
        if constexpr (!Q16) S = mfma_32x32x16(k, ql[ks], S);
    }
    __device__ __forceinline__ void scores(f32x16& S, uint32_t k) const {
        S = f32x16{};
#pragma unroll
        for (int ks = 0; ks < KS; ks++) product(S, kread(k, ks), ks);
    }
    __device__ __forceinline__ void mask_scores(f32x16& S, uint32_t key0, uint32_t end, uint32_t h) const {
        const int seen = (int)min(lim, end - 1) - (int)key0 - 4 * (int)h;
#pragma unroll
        for (int e = 0; e < 16; e++)
            if (8 * (e / 4) + e % 4 > seen) S[e] = -INFINITY;
    }
    // Moves the reference where a score (the row's largest: mx, before fac) asks for it.
    __device__ __forceinline__ void rescale(float mx) {
        mx *= fac;
        if (__builtin_expect(__ballot(mx > m + kMove) != 0, 0)) {  // (m is -inf before the row's first score)
            const float m_new = mx > m + kMove ? mx - kHead : m;
            const float alpha = m_new == m ? 1.0f : fast_exp2(m - m_new);
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) O[dt] *= alpha;
            m = m_new;
        }
    }
    // The reference to subtract: 0 for a row that has seen nothing (its weights are exp2(-inf)).
    __device__ __forceinline__ float reference() const { return m == -INFINITY ? 0.0f : m; }

    // One block by itself. scored(): called when the scores stand (K is read), landed(): before V is read.
    template <class Scored, class Landed>
    __device__ __forceinline__ void block(uint32_t k, uint32_t v, uint32_t key0, uint32_t end, bool mask, uint32_t h,
                                          Scored scored, Landed landed) {
        f32x16 S;
        k = here(k), v = here(v);
        scores(S, k);
        scored();
        if (mask) mask_scores(S, key0, end, h);  // uniform
        rescale(row_max(S));
        const float ref = reference();
        float sum = 0.0f;
        f16x8 ph[2], pl[2];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const float p0 = fast_exp2(__builtin_fmaf(S[e], fac, -ref)), p1 = fast_exp2(__builtin_fmaf(S[e + 1], fac, -ref));
            sum += p0 + p1;
            f16x2 hi, lo;
            split2_weights(p0, p1, hi, lo);
            ph[e / 8][e % 8] = hi[0], ph[e / 8][e % 8 + 1] = hi[1];
            pl[e / 8][e % 8] = lo[0], pl[e / 8][e % 8 + 1] = lo[1];
        }
        l += sum;
        landed();
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const f16x8 a = vread(v, s, dt);
                O[dt] = mfma_32x32x16(a, ph[s], O[dt]);
                O[dt] = mfma_32x32x16(a, pl[s], O[dt]);
            }
    }

    // One block of a run of them: its scores S (largest mx) stand already. The products of the next block's,
    // Sn (K at k; after the last block whatever lies there, its scores dropped), go beside the weights of S,
    // the products with V beside the other half of the weights and the next scores' maximum. load_k(),
    // load_v(): later rows' loads, issued between products, where the wait for the load path to take them
    // costs nothing. LDS reads run kAhead operands ahead of their products. The scheduling fences keep this
    // order: a product occupies the matrix core for 32 cycles, in which the wavefront issues the VALU work
    // beside it.
    template <class LoadK, class LoadV>
    __device__ __forceinline__ void step(f32x16& S, f32x16& Sn, float& mx, uint32_t k, uint32_t v, LoadK load_k, LoadV load_v) {
        constexpr int kAhead = 3, NV = 2 * DT, E0 = 8 / KS, E1 = 8 / DT;
        rescale(mx);
        const float ref = reference();
        f16x8 ph[2], pl[2], kop[KS], vop[NV];
        float w[2], sum = 0.0f;
        auto weight = [&](int e) {
            w[e % 2] = fast_exp2(__builtin_fmaf(S[e], fac, -ref));
            sum += w[e % 2];
            if (e % 2) {
                f16x2 hi, lo;
                split2_weights(w[0], w[1], hi, lo);
                ph[e / 8][e % 8 - 1] = hi[0], ph[e / 8][e % 8] = hi[1];
                pl[e / 8][e % 8 - 1] = lo[0], pl[e / 8][e % 8] = lo[1];
                if (e % 8 == 7) asm volatile("" : "+v"(ph[e / 8]), "+v"(pl[e / 8]));  // here, not where they are used
            }
        };
        k = here(k), v = here(v);
        Sn = f32x16{};
#pragma unroll
        for (int n = 0; n < kAhead; n++) kop[n] = kread(k, n);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < KS; n++) {
            if (n + kAhead < KS) kop[n + kAhead] = kread(k, n + kAhead);
            else vop[n + kAhead - KS] = vread(v, (n + kAhead - KS) / DT, (n + kAhead - KS) % DT);
#pragma unroll
            for (int e = 0; e < E0; e++) weight(E0 * n + e);
            product(Sn, kop[n], n);
            if (n == 1) load_k();
            if (n == KS - 1) load_v();
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = 0; n < NV; n++) {
            if (n + kAhead < NV) vop[n + kAhead] = vread(v, (n + kAhead) / DT, (n + kAhead) % DT);
            O[n % DT] = mfma_32x32x16(vop[n], ph[n / DT], O[n % DT]);
            O[n % DT] = mfma_32x32x16(vop[n], pl[n / DT], O[n % DT]);
            if (n < DT) {
#pragma unroll
                for (int e = 0; e < E1; e++) weight(8 + E1 * n + e);
            }
            if (n == NV - 2) mx = row_max(Sn);
            __builtin_amdgcn_sched_barrier(0);
        }
        l += sum;
    }

    // V rows of a block from position `end` on to zero (their weights are 0, what they hold may be
    // anything), and with CLEAN every infinity and NaN: true if there was one. The wavefronts that
    // share the rows write the same values.
    __device__ __forceinline__ static void zero_tail(char* sv, uint32_t key0, uint32_t end, uint32_t lane) {
#pragma unroll 1
        for (uint32_t c = here(lane); c < 32 * RB / 16; c += 64)
            if (key0 + c / (RB / 16) >= end) *(u32x4*)(sv + 16 * c) = u32x4{0u, 0u, 0u, 0u};
        __builtin_amdgcn_wave_barrier();
    }
    __device__ __forceinline__ static bool clean(char* sv, uint32_t lane) {
        constexpr int N = 4;  // chunks at a time: the wait for LDS counts once for each batch
        bool found = false;
        static_assert(32 * RB / 16 % (64 * N) == 0, "whole batches");
#pragma unroll 1
        for (uint32_t c0 = here(lane); c0 < 32 * RB / 16; c0 += 64 * N) {
            u32x4 v[N];
            uint32_t odd = 0;
#pragma unroll
            for (int j = 0; j < N; j++) v[j] = *(const u32x4*)(sv + 16 * (c0 + 64 * j));
#pragma unroll
            for (int j = 0; j < N; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) {  // an exponent of all ones carries into bit 15 or 31 when one is added to it
                    const uint32_t x = ((v[j][i] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
                    odd |= x;
                }
            if (__ballot(odd != 0) != 0) {  // rare
                found = true;
#pragma unroll
                for (int j = 0; j < N; j++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if ((v[j][i] & 0x7c00u) == 0x7c00u) v[j][i] &= 0xffff0000u;
                        if ((v[j][i] & 0x7c000000u) == 0x7c000000u) v[j][i] &= 0xffffu;
                    }
                    *(u32x4*)(sv + 16 * (c0 + 64 * j)) = v[j];
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
        return found;
    }
};

// Infinities and NaN of V that were set aside, added to a row's 4 elements from 4 c: those of
// positions begin .. end of sequence b. (Only where there are any.)
__device__ __noinline__ f32x4 add_odd_values(const f16* vpool, const int32_t* table, uint32_t page_size, uint32_t n_pages, uint32_t D,
                                             uint32_t begin, uint32_t end, uint32_t c, f32x4 o) {
    for (uint32_t key = begin; key < end; key++) {
        const int32_t pg = table[key / page_size];
        if ((uint32_t)pg >= n_pages) continue;
        const f16x4 v = *(const f16x4*)(vpool + ((uint64_t)(uint32_t)pg * page_size + key % page_size) * D + 4 * c);
        for (int e = 0; e < 4; e++)
            if (!(fabsf((float)v[e]) < INFINITY)) o[e] += (float)v[e];
    }
    return o;
}

// The workgroup's way along the batch's line of work: its part's cuts; where the tile at hand begins on
// the line; and what the end of the piece at hand needs of it, read back from LDS so that the loops over
// positions hold nothing of it in registers.
struct Walk {
    ds5idx::PbCut at, stop;
    double line, total;  // (the line's length)
    uint32_t wg, n_wg;
    ds5idx::PbCut now;
    ds5idx::PbTile tile;
    uint32_t start, before, poison, end;  // the sequence's first row, tokens before its rows; the piece's end
};

template <int D, bool Q16>
__global__ __launch_bounds__(kThreads) void paged_attention_kernel(AttnParams p) {
    using A = Attn<D, Q16>;
    constexpr int DT = A::DT, RB = A::RB, NB = A::NB, HALF = A::HALF;
    __shared__ __attribute__((aligned(1024))) char s_kv[A::AREA];
    __shared__ uint32_t s_start[kMaxSeqs], s_n[kMaxSeqs], s_before[kMaxSeqs];
    __shared__ float s_m[kWaves][32], s_l[kWaves][32];
    __shared__ double s_scan[kWaves];
    __shared__ Walk s_walk;
    // the first position with a page out of range, infinities or NaN set aside, and met: of the pieces in turn
    __shared__ uint32_t s_bad[2], s_odd[2], s_broken[2];
    __shared__ uint64_t s_row[kRows];  // of the tile's rows: the row of q and of the output (or of the parts)
    __shared__ uint32_t s_groups[kWindow];  // of a window of the piece: each 16 positions' group of rows in the pool

    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = uniform(tid >> 6);
    const uint32_t n_seqs = p.a.batch.n_seqs;
    constexpr uint32_t kPoison = 0x80000000u;  // in s_before: the sequence's rows are NaN
    auto seq = [&](uint32_t b) { return ds5idx::PbSeq{s_n[b], s_before[b] & ~kPoison}; };

    // ---- the batch's sequences and their work; this workgroup's part of it
    {
        const PagedBatch& bt = p.a.batch;
        const uint32_t G = p.group;
        // The workgroup's two halves do the same for the part's two cuts: a thread's sequences are consecutive ones.
        constexpr uint32_t kHalf = kThreads / 2;
        const uint32_t cut = uniform(tid / kHalf), i = tid % kHalf, N = (n_seqs + kHalf - 1) / kHalf, b0 = i * N;
        double mine = 0.0;
#pragma unroll 1
        for (uint32_t b = b0; b < min(b0 + N, n_seqs); b++) {
            const int64_t s0 = bt.starts[b], s1 = bt.starts[b + 1], len = bt.seq_lens[b];
            const int64_t c0 = max(s0, (int64_t)0), c1 = min(s1, (int64_t)bt.n_tokens);
            const uint32_t n = c1 > c0 ? (uint32_t)(c1 - c0) : 0;
            const bool ok = c0 == s0 && c1 == s1 && len >= s1 - s0 && len <= (int64_t)bt.max_seq_len;
            s_start[b] = (uint32_t)c0;
            s_n[b] = n;
            s_before[b] = ok ? (uint32_t)(len - n) : kPoison;
            mine += ds5idx::pb_seq_work(seq(b), G);
        }
        const double upto = sums_upto(mine);
        if (lane == 63) s_scan[wave] = upto;
        if (tid == 0) {  // where decreasing starts make more work than the sums hold exactly: no part
            s_walk.at = s_walk.stop = ds5idx::PbCut{bt.n_kv_heads, 0, 0, 0};
            s_walk.line = 0.0;
            s_bad[0] = 0xffffffffu, s_odd[0] = s_broken[0] = 0;
        }
        __syncthreads();
        double from = upto - mine, per_head = 0.0;
#pragma unroll
        for (uint32_t w = 0; w < (uint32_t)kWaves / 2; w++) {
            const double x = s_scan[cut * (kWaves / 2) + w];
            from += w < wave % (kWaves / 2) ? x : 0.0;
            per_head += x;
        }
        const double total = per_head * bt.n_kv_heads;
        const uint32_t grid = gridDim.x;
        const uint32_t n_wg = uniform(total == 0.0 ? 0 : p.whole ? grid : ds5idx::pb_workgroups(total, p.inv_group, bt.n_kv_heads, p.inv_heads, grid));
        // A full grid's consecutive parts go to one XCD (workgroup i runs on XCD i % 8), so that a
        // sequence's K and V come into few L2s.
        const uint32_t wg = n_wg + bt.n_kv_heads > grid && grid % 8 == 0 ? blockIdx.x % 8 * (grid / 8) + blockIdx.x / 8 : blockIdx.x;
        if (tid == 0 && p.heads) p.heads[wg] = 0;  // until it begins a tile that it does not end
        if (wg >= n_wg) return;
        const double share = ds5idx::pb_inverse(n_wg);
        const double snap = ds5idx::pb_snap(total, share, G);
        if (tid == 0) {
            s_walk.total = total;
            s_walk.wg = wg, s_walk.n_wg = n_wg;
        }
        double y;
        const uint32_t h = ds5idx::pb_divide(ds5idx::pb_cut_at(total, wg + cut, n_wg, share), per_head, y);
        if (y >= from && y - from < mine && wg + cut < n_wg)
            for (uint32_t b = b0; b < min(b0 + N, n_seqs); b++) {
                const double work = ds5idx::pb_seq_work(seq(b), G);
                if (y - from >= work) {
                    from += work;
                    continue;
                }
                const ds5idx::PbPlace at =
                    ds5idx::pb_locate(seq(b), G, p.inv_group, y - from, snap, ds5idx::pb_lead(total, share, G), p.whole);
                (cut ? s_walk.stop : s_walk.at) = ds5idx::PbCut{h, b, at.j, at.k};
                if (cut == 0) s_walk.line = h * per_head + from + at.at;
                break;
            }
    }
    __syncthreads();

    auto scalar = [](const ds5idx::PbCut& c) { return ds5idx::PbCut{uniform(c.kvh), uniform(c.b), uniform(c.j), uniform(c.k)}; };
    ds5idx::PbCut at = scalar(s_walk.at);
    uint32_t turn = 0;
    for (bool last_piece = false; !last_piece; at.j++, at.k = 0, turn ^= 1) {
        // every wavefront walks by itself; what the piece's end needs of it lies in LDS until then
        const ds5idx::PbCut stop = scalar(s_walk.stop);
        if (!ds5idx::pb_next(at, stop, n_seqs, p.a.batch.n_kv_heads, p.group,
                             [&](uint32_t b) { return ds5idx::PbSeq{uniform(s_n[b]), 0}; }, last_piece))
            return;
        const Walk& wk = *(const Walk*)((const char*)&s_walk + here(0));
        const uint32_t mark = uniform(s_before[at.b]), start = uniform(s_start[at.b]);
        const ds5idx::PbSeq sq{uniform(s_n[at.b]), mark & ~kPoison};
        ds5idx::PbTile tile = ds5idx::pb_tile(sq, p.group, p.inv_group, ds5idx::pb_tile_at(at.j, ds5idx::pb_tiles(sq, p.group)));
        tile.kv = uniform(tile.kv);
        const uint32_t end = last_piece ? stop.k : tile.kv;
        if (tid == 0) {
            Walk& w = s_walk;
            w.now = at;
            w.tile = tile;
            w.start = start, w.before = sq.before, w.poison = mark & kPoison, w.end = end;
        }
        // The piece, in a form of its own for tiles of at most kNarrow rows (in one form of both the compiler
        // spills: the accumulators then meet where the forms part and join).
        auto piece = [&](auto form) {
        constexpr bool narrow = decltype(form)::value;
        const uint32_t tid = here(threadIdx.x), lane = tid & 63;
        const uint32_t r32 = lane & 31, h = lane >> 5;
        A t;
        t.koff = ds5idx::pb_load_off(D, false, 0, lane);
        t.voff = ds5idx::pb_load_off(D, true, 0, lane);
        {
            const typename A::Lane ln(lane);
            const uint32_t kb = at.k, rows = tile.rows, row0 = tile.row0, before = sq.before, kvh = at.kvh, b = at.b, G = p.group;
            const bool poison = (mark & kPoison) != 0;
            const uint32_t rg = narrow ? 0 : wave & 3;
            const PagedBatch& bt = p.a.batch;
            // ---- this wavefront's 32 query rows
            const uint32_t row = row0 + min(32 * rg + r32, rows - 1);
            const uint32_t token = ds5idx::pb_over(row, p.inv_group);
            t.lim = before + token;
            const uint32_t lim_lo = uniform(before + ds5idx::pb_over(row0 + min(32 * rg, rows - 1), p.inv_group));
            const uint32_t lim_hi = uniform(before + ds5idx::pb_over(row0 + min(32 * rg + 31, rows - 1), p.inv_group));
            typename A::Query query;
            if constexpr (narrow)
                A::fetch_q(query, p, ((uint64_t)(start + token) * bt.n_q_heads + kvh * G + (row - token * G)) * D + 8 * h);
            if (tid < (uint32_t)kRows) {
                const uint32_t packed = row0 + min(tid, rows - 1), token = ds5idx::pb_over(packed, p.inv_group);
                s_row[tid] = (uint64_t)(start + token) * bt.n_q_heads + kvh * G + (packed - token * G);
            }

            const uint64_t head = (uint64_t)kvh * bt.n_pages * bt.page_size * D;
            const f16* const kpool = p.a.k_pool + head;
            const f16* const vpool = p.a.v_pool + head;
            const int32_t* const table = bt.page_table + (uint64_t)b * bt.max_pages;
            const uint32_t page_size = bt.page_size;
            // The piece in windows of kWindow groups of 16 positions (most pieces are one): positions
            // from .. to, `last` the last group; what is read past it is it again.
            uint32_t from, to, last;
            auto window = [&](uint32_t begin) {
                from = begin;
                to = end - from > 16 * kWindow ? from + 16 * kWindow : end;
                last = (to - from - 1) / 16;
#pragma unroll 1
                for (uint32_t i = tid; i <= last; i += kThreads) {
                    const uint32_t pos = from + 16 * i, page = ds5idx::pb_over(pos, p.inv_page);
                    const uint32_t pg = (uint32_t)table[page];  // (a page out of range: page 0, and the rows that attend it are NaN)
                    s_groups[i] = (pg < bt.n_pages ? pg : 0) * (page_size / 16) + (pos - page * page_size) / 16;
                    if (pg >= bt.n_pages) atomicMin(&s_bad[turn], pos);
                }
                __syncthreads();
            };
            // narrow: blocks of 32 positions, one wavefront each, in an area of its own; the next block's K is
            // loaded once this one's scores stand, its V once this one's products do
            char* const sk = s_kv + wave * 2 * HALF;
            char* const sv = sk + HALF;
            uint64_t r0, r1;
            auto rows_at = [&](uint32_t key0) {
                const uint32_t g = (key0 - from) / 16;
                r0 = (uint64_t)uniform(s_groups[min(g, last)]) * (16 * D);
                r1 = (uint64_t)uniform(s_groups[min(g + 1, last)]) * (16 * D);
            };
            auto block_k = [&]() {
                A::template load_group<false>(lds_addr(sk), kpool + r0, t.koff);
                A::template load_group<false>(lds_addr(sk) + HALF / 2, kpool + r1, t.koff);
            };
            auto block_v = [&]() {
                A::template load_group<true>(lds_addr(sv), vpool + r0, t.voff);
                A::template load_group<true>(lds_addr(sv) + HALF / 2, vpool + r1, t.voff);
            };
            // wide: steps of 64 positions through a ring of four stages of K and V: wavefront w loads rows
            // 8 w .. 8 w + 7, three steps ahead, into the stage that everyone left before the last barrier;
            // wavefronts 0 .. 3 take the first block of a step, 4 .. 7 the second. A step's K and V have landed
            // one step before their block (its scores are formed a block ahead).
            constexpr uint32_t STAGE = 2 * 64 * RB;
            const uint32_t mine = 32 * (wave >> 2);
            const uint32_t koff = t.koff ^ (wave & 1) * (RB / 2);  // the K rows' swizzle of rows 8 .. 15 of 16
            const f16* const kw = kpool + (wave & 1) * 8 * D;
            const f16* const vw = vpool + (wave & 1) * 8 * D;
            const uint32_t lds0 = lds_addr(s_kv) + 8 * wave * RB;
            auto group_at = [&](uint32_t i) { return s_groups[min(4 * i + (wave >> 1), last)]; };
            auto step_k = [&](uint32_t i, uint32_t g) {
                A::template load_half<false>(lds0 + (i & 3) * STAGE, kw + (uint64_t)g * (16 * D), koff);
            };
            auto step_v = [&](uint32_t i, uint32_t g) {
                A::template load_half<true>(lds0 + (i & 3) * STAGE + STAGE / 2, vw + (uint64_t)g * (16 * D), t.voff);
            };
            // a window's first loads
            auto prime = [&]() {
                if constexpr (narrow) {
                    if (from + 32 * wave < to) {
                        rows_at(from + 32 * wave);
                        block_k();
                        block_v();
                    }
                } else {
                    uint32_t g[3];
#pragma unroll
                    for (uint32_t i = 0; i < 3; i++) g[i] = group_at(i);
#pragma unroll
                    for (uint32_t i = 0; i < 3; i++) {  // (steps past the last re-read its rows)
                        step_k(i, uniform(g[i]));
                        step_v(i, uniform(g[i]));
                    }
                }
            };
            const bool work = !poison && kb < end;
            if (work) window(kb);
            if constexpr (narrow) {
                if (work) prime();
            } else {
                if (work) {
                    A::stage_q(lds_addr(s_kv) + A::AREA / 2, p.a.q, wave, lane, [&](uint32_t r) { return s_row[r]; });
                    for (uint32_t i = 0; i < 2; i++) {
                        const uint32_t g = uniform(group_at(i));
                        step_k(i, g);
                        step_v(i, g);
                    }
                }
                wait_loads<0>();
                __syncthreads();
                A::staged_q(query, s_kv + A::AREA / 2, 32 * rg + r32, h);
                __syncthreads();  // the query rows' area is the ring's other half
                if (work) {
                    const uint32_t g = uniform(group_at(2));
                    step_k(2, g);
                    step_v(2, g);
                }
            }
            t.form_q(query, p.a.scale);  // while the first rows are on their way
            bool careful = false;
            for (;;) {  // a second time, with infinities and NaN of V set aside, if the first left any in O
                t.m = -INFINITY;
                t.l = 0.0f;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) t.O[dt] = f32x16{};
                bool odd = false;
                auto clean = [&](char* sv, uint32_t key0) {  // what V holds past the end, and infinities and NaN
                    if (key0 + 32 > end) A::zero_tail(sv, key0, end, lane);
                    if (careful) odd |= A::clean(sv, lane);
                };
                for (bool more = work; more;) {
                    if constexpr (narrow) {
#pragma unroll 1
                        for (uint32_t key0 = from + 32 * wave; key0 < to; key0 += 32 * kWaves) {
                            const uint32_t next = key0 + 32 * kWaves;
                            const bool mask = key0 + 31 > lim_lo || key0 + 32 > end;
                            rows_at(next);
                            wait_loads<2 * NB>();  // K is here; V may not be
                            t.block(lds_addr(sk) + ln.k, lds_addr(sv) + ln.v, key0, end, mask, h,
                                    [&]() {
                                        if (next < to) block_k();
                                    },
                                    [&]() {
                                        if (next < to) wait_loads<2 * NB>();
                                        else wait_loads<0>();
                                        if (mask || careful) clean(sv, key0);
                                    });
                            if (next < to) {
                                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                                block_v();
                            }
                        }
                    } else {
                        const uint32_t steps = (to - from + 63) / 64;
                        const uint32_t k0 = lds_addr(s_kv) + mine * RB + ln.k, v0 = lds_addr(s_kv) + mine * RB + STAGE / 2 + ln.v;
                        // this wavefront's blocks: the first of the steps whose block holds a position its rows attend;
                        // those before `plain` need no mask
                        const uint32_t upto = min(to, lim_hi + 1), first = from + mine;
                        const uint32_t blocks = 32 * rg < rows && upto > first ? (upto - first + 63) / 64 : 0;
                        const uint32_t whole = min(lim_lo + 1, end);  // positions below it all rows attend
                        const uint32_t plain = careful || whole < first + 32 ? 0 : (whole - first - 32) / 64 + 1;
                        wait_loads<NB>();
                        __syncthreads();
                        f32x16 Sa, Sb;
                        float mx = -INFINITY;
                        if (blocks) {
                            t.scores(Sa, k0);
                            mx = row_max(Sa);
                        }
                        uint32_t ahead = group_at(3);
                        auto run = [&](uint32_t i, f32x16& S, f32x16& Sn) {
                            const uint32_t g = uniform(ahead);
                            ahead = group_at(i + 4);
                            if (i < blocks) {
                                if (__builtin_expect(i >= plain, 0)) {
                                    const uint32_t key0 = first + 64 * i;
                                    if (key0 + 31 > lim_lo || key0 + 32 > end) {
                                        t.mask_scores(S, key0, end, h);
                                        mx = row_max(S);
                                    }
                                    clean(s_kv + (i & 3) * STAGE + STAGE / 2 + mine * RB, key0);
                                }
                                t.step(S, Sn, mx, k0 + ((i + 1) & 3) * STAGE, v0 + (i & 3) * STAGE, [&]() { step_k(i + 3, g); },
                                       [&]() { step_v(i + 3, g); });
                            } else {
                                step_k(i + 3, g);
                                step_v(i + 3, g);
                            }
                            wait_loads<NB>();
                            __syncthreads();
                        };
#pragma unroll 1
                        for (uint32_t i = 0; i < steps; i += 2) {  // (an odd count's last one works on nothing)
                            run(i, Sa, Sb);
                            run(i + 1, Sb, Sa);
                        }
                        // The last steps' loads ahead are still in flight past their barrier, into rows that O or
                        // another window goes to: every wavefront waits for its own, then for the others.
                        wait_loads<0>();
                        __syncthreads();
                    }
                    more = to < end;
                    if (more) {
                        if constexpr (narrow) __syncthreads();  // everyone is done with the window
                        window(to);
                        prime();
                    }
                }
                if (odd && lane == 0) s_odd[turn] = 1;
                float zero[4] = {};  // (NaN where O holds an infinity or NaN)
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int e = 0; e < 16; e++) zero[e % 4] = __builtin_fmaf(t.O[dt][e], 0.0f, zero[e % 4]);
                if (__ballot(!((zero[0] + zero[1]) + (zero[2] + zero[3]) == 0.0f)) != 0 && lane == 0) s_broken[turn] = 1;
                {  // rows of O through LDS
                    const float l = swap32_op(t.l, OpAdd{});
                    const uint32_t lane = here(tid) & 63, r32 = lane & 31, h = lane >> 5;
                    char* area = s_kv + wave * 2 * HALF;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint32_t c = 8 * dt + 2 * i + h;
                            *(float4*)(area + r32 * 4 * D + (c ^ (r32 & (A::CH - 1))) * 16) =
                                float4{t.O[dt][4 * i], t.O[dt][4 * i + 1], t.O[dt][4 * i + 2], t.O[dt][4 * i + 3]};
                        }
                    if (h == 0) {
                        s_m[wave][r32] = t.m;
                        s_l[wave][r32] = l;
                    }
                }
                __syncthreads();
                if (careful || uniform(s_broken[turn]) == 0) break;
                careful = true;
                if (work) {
                    window(kb);
                    prime();
                }
            }
        }

        // ---- the wavefronts' parts of the tile together
        const uint32_t kb = uniform(wk.now.k), end = uniform(wk.end), wg = uniform(wk.wg), G = p.group;
        const uint32_t row0 = uniform(wk.tile.row0), rows = uniform(wk.tile.rows), before = uniform(wk.before);
        const uint32_t start = uniform(wk.start), kvh = uniform(wk.now.kvh);
        const bool done = kb == 0 && end == uniform(wk.tile.kv), poison = uniform(wk.poison) != 0;
        const bool begins = kb == 0 && !done;
        const uint32_t slot = 2 * wg + (begins ? 1 : 0);
        const bool any_odd = uniform(s_odd[turn]) != 0;
        const uint32_t bad_pos = uniform(s_bad[turn]);
        if (tid == 0) s_bad[turn ^ 1] = 0xffffffffu, s_odd[turn ^ 1] = s_broken[turn ^ 1] = 0;  // the next piece's
        constexpr uint32_t N = narrow ? kWaves : 2, STEP = kWaves / N;  // wavefronts that hold a part of a row
        const bool output = done || poison;  // else a part
        // a row's factors; what a part keeps of it
        auto factors = [&](uint32_t rr, float (&f)[N], bool keep) {
            const uint32_t w0 = narrow ? 0 : rr >> 5, r = rr & 31;
            float M = s_m[w0][r], L = 0.0f;
#pragma unroll
            for (uint32_t i = 1; i < N; i++) M = fmaxf(M, s_m[w0 + STEP * i][r]);
#pragma unroll
            for (uint32_t i = 0; i < N; i++) {
                const float m = s_m[w0 + STEP * i][r];
                f[i] = m == -INFINITY ? 0.0f : fast_exp2(m - M);  // (a wavefront that saw none of the row's positions: O is 0)
                L = __builtin_fmaf(s_l[w0 + STEP * i][r], f[i], L);
            }
            if (poison || before + ds5idx::pb_over(row0 + rr, p.inv_group) >= bad_pos) M = 0.0f, L = NAN;
            if (!output && keep) p.part_ml[(uint64_t)slot * kRows + rr] = float2{M, L};
            const float unit = output ? 1.0f / L : 1.0f;
#pragma unroll
            for (uint32_t i = 0; i < N; i++) f[i] *= unit;
        };
        if constexpr (!narrow) {  // worked out once a row, and kept in place of its references
            if (tid < rows) {
                float f[N];
                factors(tid, f, true);
                if (!output) s_row[tid] = (uint64_t)slot * kRows + tid;
#pragma unroll
                for (uint32_t i = 0; i < N; i++) s_m[(tid >> 5) + STEP * i][tid & 31] = f[i];
            }
            __syncthreads();
        }
        {
            // a row's D / 4 columns to as many threads, kThreads / CH rows at a time
            constexpr uint32_t CH = A::CH, PER = kThreads / CH, U = narrow ? 1 : 4;
            const uint32_t c = here(tid) % CH, stride = narrow ? 2 * HALF : 8 * HALF;
            float* const to = output ? p.a.out : p.part_o;
            auto finish = [&](uint32_t rr) {
                const uint32_t w0 = narrow ? 0 : rr >> 5, r = rr & 31;
                float f[N];
                if constexpr (narrow) factors(rr, f, c == 0);
                else
                    for (uint32_t i = 0; i < N; i++) f[i] = s_m[w0 + STEP * i][r];
                f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (uint32_t i = 0; i < N; i++)
                    o += *(const f32x4*)(s_kv + w0 * 2 * HALF + i * stride + r * 4 * D + (c ^ (r & (CH - 1))) * 16) * f[i];
                if (any_odd) {
                    const PagedBatch& bt = p.a.batch;
                    o = add_odd_values(p.a.v_pool + (uint64_t)kvh * bt.n_pages * bt.page_size * D,
                                       bt.page_table + (uint64_t)wk.now.b * bt.max_pages, bt.page_size, bt.n_pages, D, kb,
                                       min(end, before + ds5idx::pb_over(row0 + rr, p.inv_group) + 1), c, o);
                }
                *(f32x4*)(to + (narrow && !output ? (uint64_t)slot * kRows + rr : s_row[rr]) * D + 4 * c) = o;
            };
#pragma unroll 1
            for (uint32_t r = here(tid) / CH; r < rows; r += U * PER)
#pragma unroll
                for (uint32_t u = 0; u < U; u++)
                    if (U == 1 || r + u * PER < rows) finish(r + u * PER);
        }
        __syncthreads();  // LDS is free again
        if (tid == 0) {
            Walk& w = s_walk;
            const ds5idx::PbSeq sq = seq(w.now.b);
            const double tile_end =
                w.line + ds5idx::pb_tile_work(sq, G, ds5idx::pb_tile_at(w.now.j, ds5idx::pb_tiles(sq, G)));
            // the last workgroup with a part of the tile: the last cut that is not within `snap` of its end
            if (begins && !poison) {
                const double share = ds5idx::pb_inverse(w.n_wg);
                const uint32_t last = ds5idx::pb_last_cut(w.total, w.n_wg, share, tile_end - ds5idx::pb_snap(w.total, share, G));
                static_assert(kRows < 256 && kMaxGrid <= 1u << 24, "rows and workgroup in a word");
                p.heads[wg] = rows | last << 8;
                p.descs[wg] = MergeDesc{row0, kvh, start};
            }
            w.line = tile_end;
        }
        };
        if (tile.rows <= (uint32_t)kNarrow) piece(std::true_type{});
        else piece(std::false_type{});
    }
}

// The parts of the tiles that several workgroups share: the head part of workgroup w, then the parts of
// w + 1 .. last, folded in that order. 256 threads are D / 4 columns and 1024 / D slots: with few parts a
// slot folds a row of its own, with many the slots share a row's parts and join through LDS. The
// workgroups go along all tiles' rows (or groups of rows) evenly. 4 us where there is little (its launch),
// 7.5 for the 17 MB of 256 parts of 128 rows of 128.
template <int D>
__global__ __launch_bounds__(kMaxGrid) void paged_merge_kernel(AttnParams p, uint32_t n_descs) {
    constexpr uint32_t CH = D / 4, SL = kMaxGrid / CH;
    __shared__ uint32_t s_wave[kMaxGrid / 64];
    __shared__ uint32_t s_item[3];  // the item at hand: its head part's workgroup, its place among the tile's items, the tile's word
    __shared__ f32x4 s_o[SL][CH];
    __shared__ float2 s_ml[SL];
    const uint32_t tid = threadIdx.x, lane = tid & 63, G = p.group;
    auto together = [&](uint32_t parts) { return parts <= SL; };  // SL rows at once
    const uint32_t mine = tid < n_descs ? p.heads[tid] : 0, mine_rows = mine & 255;
    const uint32_t items = mine == 0 ? 0 : together((mine >> 8) - tid + 1) ? (mine_rows + SL - 1) / SL : mine_rows;
    uint32_t upto = sums_upto(items);
    if (lane == 63) s_wave[tid >> 6] = upto;
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kMaxGrid / 64; w++) {
        if (w < tid >> 6) upto += s_wave[w];
        total += s_wave[w];
    }
    const uint32_t c = tid % CH, sl = tid / CH;
    for (uint32_t item = blockIdx.x; item < total; item += gridDim.x) {
        if (item < upto && item >= upto - items) {  // one thread's
            s_item[0] = tid;
            s_item[1] = item - (upto - items);
            s_item[2] = mine;
        }
        __syncthreads();
        const uint32_t w = uniform(s_item[0]), at = uniform(s_item[1]), head = uniform(s_item[2]);
        const MergeDesc d = p.descs[w];
        const uint32_t n = (head >> 8) - w + 1;
        // parts first, first + step, ... of a row
        auto fold = [&](uint32_t row, uint32_t first, uint32_t step, float& M, float& L, f32x4& o) {
            constexpr int U = 8;
            M = -INFINITY, L = 0.0f, o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            for (uint32_t i0 = first; i0 < n; i0 += U * step) {
                float2 ml[U];
                f32x4 v[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const uint32_t i = min(i0 + u * step, n - 1);
                    const uint64_t s = (uint64_t)(i == 0 ? 2 * w + 1 : 2 * (w + i)) * kRows + row;
                    ml[u] = p.part_ml[s];
                    v[u] = *(const f32x4*)(p.part_o + s * D + 4 * c);
                }
                float m = M;
#pragma unroll
                for (int u = 0; u < U; u++) m = i0 + u * step < n ? fmaxf(m, ml[u].x) : m;
                const float f0 = M == -INFINITY ? 0.0f : fast_exp2(M - m);
                L *= f0, o *= f0;
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (i0 + u * step < n && ml[u].y != 0.0f) {  // (nothing: none of the row's positions; scores of NaN alone: -inf and NaN)
                        const float f = fast_exp2(ml[u].x - m);
                        L = __builtin_fmaf(ml[u].y, f, L);
                        o += v[u] * f;
                    }
                M = m;
            }
        };
        auto write = [&](uint32_t row, f32x4 o, float L) {
            const uint32_t packed = d.row0 + row, token = ds5idx::pb_over(packed, p.inv_group);
            *(f32x4*)(p.a.out + ((uint64_t)(d.token0 + token) * p.a.batch.n_q_heads + d.kvh * G + (packed - token * G)) * D + 4 * c) =
                o * (1.0f / L);
        };
        float M, L;
        f32x4 o;
        if (together(n)) {
            const uint32_t row = at * SL + sl;
            if (row < (head & 255)) {
                fold(row, 0, 1, M, L, o);
                write(row, o, L);
            }
        } else {
            fold(at, sl, SL, M, L, o);
            s_o[sl][c] = o;
            if (c == 0) s_ml[sl] = float2{M, L};
            __syncthreads();
            if (sl == 0) {
                float mm = -INFINITY, ll = 0.0f;
                for (uint32_t i = 0; i < SL; i++) mm = fmaxf(mm, s_ml[i].x);
                f32x4 oo = {0.0f, 0.0f, 0.0f, 0.0f};
                for (uint32_t i = 0; i < SL; i++) {
                    if (s_ml[i].y == 0.0f) continue;
                    const float f = fast_exp2(s_ml[i].x - mm);
                    ll += s_ml[i].y * f;
                    oo += s_o[i][c] * f;
                }
                write(at, oo, ll);
            }
        }
        __syncthreads();  // s_item, s_o and s_ml are free again
    }
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

// Whether uncut tiles are the faster form, in the plan's units (4.7 ns), every sequence taken to have the
// mean rows and the longest length (the host knows no more, so that one long sequence among short ones whose
// tiles come near a multiple of the CUs runs whole: 63 of 500 positions and one of 16384 151 us; 50 of 500 and
// the long one, cut, 33): rounds of whole tiles, or even shares, in which a workgroup pays for a
// second tile as a rule, and the merge with the parts' way through memory. Measured with the caches in
// memory (not in the chip's), us, cut and whole (32 query and 4 kv heads of 128): one token 15.8 and 14.8 at
// 500 positions, 16.2 and 18.9 at 1000; 48 sequences' 37.7 and 29.3, 53.5 and 48.3, at 4000 145 and 137; six
// tokens 18.2 and 22.0, 19.9 and 30.7; 48 sequences of six 42.2 and 33.4, 59.5 and 53.4; eight of 40 32.6
// and 25.5, 43.7 and 35.0, at 2000 50.4 and 54.5.
static bool whole_tiles_do(const PagedBatch& b, uint32_t group, uint32_t cus) {
    const double live = std::min(b.n_seqs, b.n_tokens), rows = std::ceil(b.n_tokens / live) * group;
    const bool wide = rows > kNarrow;
    const double tile = ds5idx::kPbTileCost + (wide ? 5.0 : 2.0) * b.max_seq_len, tiles = b.n_kv_heads * live * std::ceil(rows / kRows);
    const double n = std::min<double>(cus, std::max(1.0, tiles * tile / ds5idx::kPbPiece));
    return std::ceil(tiles / cus) * tile <= tiles / n * tile + ds5idx::kPbTileCost + 1350.0 + (wide ? 1300.0 : 300.0) * n / cus;
}

int launch_paged_attention(ds5_hip_ctx* ctx, const PagedAttentionLaunch& a) {
    const PagedBatch& b = a.batch;
    AttnParams p{};
    p.a = a;
    p.group = b.n_q_heads / b.n_kv_heads;
    p.inv_group = 1.0 / p.group;
    p.inv_page = 1.0 / b.page_size;
    p.inv_heads = 1.0 / b.n_kv_heads;
    const uint64_t rows = (uint64_t)b.n_tokens * p.group, tiles = rows / kRows + std::min<uint64_t>(b.n_seqs, b.n_tokens);
    // the work that the plan counts, at most: below 2^53
    if ((double)b.n_kv_heads * tiles * ((double)p.group * (5.0 * b.max_seq_len + ds5idx::kPbTileCost) + 5.0 * (rows + kRows)) >= 9007199254740992.0)
        return ds5_fail(ctx, DS5_SHAPE_MISMATCH, "paged_attention: batch too large");
    const uint32_t cus = std::min(kMaxGrid, ctx->cu_count > 0 ? (uint32_t)ctx->cu_count : kMaxGrid);
    p.whole = !ctx->split_buf || whole_tiles_do(b, p.group, cus);
    const uint64_t most =
        b.n_kv_heads * tiles * (p.whole ? 1 : (5ull * b.max_seq_len + ds5idx::kPbTileCost) / ds5idx::kPbPiece + 1);
    const dim3 grid((uint32_t)std::min<uint64_t>(most, cus)), block(kThreads);
    if (!p.whole) {
        static_assert(2ull * kMaxGrid * kRows * 128 * sizeof(float) <= kSplitBytesMax, "parts fit the context's buffer");
        static_assert(2ull * kMaxGrid * kRows * sizeof(float2) + kMaxGrid * (sizeof(MergeDesc) + 4) <= kSplitStateBytes, "and their state");
        p.part_o = (float*)ctx->split_buf;
        p.part_ml = (float2*)((char*)ctx->split_buf + kSplitBytesMax);
        p.heads = (uint32_t*)(p.part_ml + 2ull * kMaxGrid * kRows);
        p.descs = (MergeDesc*)(p.heads + kMaxGrid);
    }
    const char* name = "paged_attention_kernel";
    if (b.head_dim == 128) {
        if (a.q_f16) DS5_TIMED_LAUNCH(ctx, name, (paged_attention_kernel<128, true>), grid, block, 0, ctx->stream, p);
        else DS5_TIMED_LAUNCH(ctx, name, (paged_attention_kernel<128, false>), grid, block, 0, ctx->stream, p);
    } else {
        if (a.q_f16) DS5_TIMED_LAUNCH(ctx, name, (paged_attention_kernel<64, true>), grid, block, 0, ctx->stream, p);
        else DS5_TIMED_LAUNCH(ctx, name, (paged_attention_kernel<64, false>), grid, block, 0, ctx->stream, p);
    }
    if (int rc = ds5_after_launch(ctx, name)) return rc;
    if (p.whole || grid.x == 1) return DS5_OK;  // one workgroup cuts nothing
    // an item is a row at least, and there are n_q_heads of a token
    const dim3 merge((uint32_t)std::min<uint64_t>((uint64_t)b.n_tokens * b.n_q_heads, 4 * kMaxGrid));
    name = "paged_merge_kernel";
    if (b.head_dim == 128) DS5_TIMED_LAUNCH(ctx, name, paged_merge_kernel<128>, merge, dim3(kMaxGrid), 0, ctx->stream, p, grid.x);
    else DS5_TIMED_LAUNCH(ctx, name, paged_merge_kernel<64>, merge, dim3(kMaxGrid), 0, ctx->stream, p, grid.x);
    return ds5_after_launch(ctx, name);
}
