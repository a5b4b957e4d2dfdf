// ds5_index.hpp -- the per-lane address arithmetic of the hot kernels, as
// __host__ __device__ functions: the kernels call them, and the library
// exports host wrappers (ds5_index_*, ds5_index.hip) through which the CPU
// tests enumerate every access of a launch. A change here changes both.
//
//   decode_split_kernel (k_decode.hip): the rows and columns of a tile's K and V
//     loads (issue_tile), the page-table slot of a paged position (page_base), and
//     the arithmetic of the paged plan (paged_plan);
//   matmul_q8_mfma_kernel (k_matmul.hip): the lane offsets of the direct-to-LDS
//     x-plane and raw Q8_0 row loads;
//   prefill_attention_kernel (k_prefill.hip): the lane offsets of a K/V tile's
//     direct-to-LDS loads and their clamp, and the staged q and output rows;
//   attn_f32_kernel (k_attn_f32.hip): a wavefront's query rows, the clamped positions of
//     its loads, and which split writes a row where;
//   paged_attention_kernel (k_paged.hip): the tiles of a ragged batch, how the batch's work is
//     cut over the workgroups, and the lane offsets of a row group's direct-to-LDS loads.
#pragma once

#include <math.h>
#include <stdint.h>

#if defined(__HIPCC__)
#include <hip/hip_runtime.h>
#endif

#if defined(__HIPCC__)
#define DS5_HD __host__ __device__ __forceinline__
#define DS5_HDC __host__ __device__ constexpr
#else
#define DS5_HD inline
#define DS5_HDC constexpr
#endif

namespace ds5idx {

DS5_HD uint32_t umin(uint32_t a, uint32_t b) { return a < b ? a : b; }
DS5_HD uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// decode_split_kernel's shape: 32-position tiles, four wavefronts (one per SIMD),
// up to 16 q heads of one kv head per workgroup, at most 64 splits per sequence.
constexpr int kDecTile = 32, kDecWaves = 4, kDecHeads = 16;
constexpr uint32_t kDecMaxSplits = 64;
// prefill_attention_kernel's shape: 4 q heads per workgroup, 32-row q tiles,
// 64-key K/V tiles; LDS row strides of K and V (bytes), padded for conflict-free reads.
constexpr int kPfHeads = 4, kPfQRows = 32, kPfKTile = 64;
DS5_HDC int pf_rsk(int D) { return 2 * D + 16; }
DS5_HDC int pf_rsv(int D) { return 2 * D + 64; }

// attn_f32_kernel's shape: 16 query rows and 16 positions a tile, four wavefronts.
constexpr int kAfRows = 16, kAfPos = 16, kAfWaves = 4;

// Split-K geometry of a contiguous decode launch: positions per split (a multiple
// of 128, at least max_len / 64; about four workgroups per CU unless decode_chunk
// fixes it) and the split count.
DS5_HD void dec_geometry(uint32_t cu_count, uint32_t decode_chunk, uint32_t n_seqs, uint32_t n_kv_heads,
                         uint32_t n_sub, uint32_t max_len, uint32_t& chunk, uint32_t& n_splits) {
    const uint32_t step = kDecWaves * kDecTile;
    chunk = decode_chunk;
    if (chunk == 0) {
        const uint64_t units = (uint64_t)n_seqs * n_kv_heads * n_sub;
        const uint64_t target = 4ull * (cu_count > 0 ? cu_count : 256);
        const uint64_t c = (max_len * units + target - 1) / target;
        chunk = (uint32_t)(c < max_len ? c : max_len);
    }
    chunk = umax((chunk + step - 1) / step * step, step);
    chunk = umax(chunk, (max_len + kDecMaxSplits - 1) / kDecMaxSplits);
    chunk = (chunk + step - 1) / step * step;
    n_splits = (max_len + chunk - 1) / chunk;
}

// ---------------------------------------------------------------------------
// decode_split_kernel: a 32-position tile [p0, p0 + 32) of a split ending at `end`.
// K: lane (g = lane / 16, c16 = lane % 16), half st, k-step kk reads 8 halves
//    (16 bytes) of row dec_k_row at column dec_k_col.
// V: 16-byte chunk c = lane + 64 r (r < VC) reads row dec_v_row (tile row
//    tr = c / RC, RC = head_dim / 8 chunks per row) at column dec_v_col.
// Contiguous cache: rows past `end` are clamped to end - 1. Paged: each
// 16-position half sits inside one page (page_size % 16 == 0, p0 % 32 == 0);
// rowA / rowB are the pool slots of the halves' first positions.
// ---------------------------------------------------------------------------
DS5_HD uint32_t dec_half_pos(uint32_t p0, uint32_t end, int st) { return st ? umin(p0 + 16, end - 1) : p0; }
DS5_HD uint64_t dec_k_row(uint32_t p0, uint32_t end, int st, int c16) {
    return umin(p0 + 16 * (uint32_t)st + (uint32_t)c16, end - 1);
}
DS5_HD uint64_t dec_v_row(uint32_t p0, uint32_t end, int tr) { return umin(p0 + (uint32_t)tr, end - 1); }
DS5_HD uint64_t dec_k_row_paged(uint64_t rowA, uint64_t rowB, int st, int c16) { return (st ? rowB : rowA) + c16; }
DS5_HD uint64_t dec_v_row_paged(uint64_t rowA, uint64_t rowB, int r, int VC, int tr) {
    return (r < VC / 2 ? rowA : rowB) + (tr & 15);
}
DS5_HD uint32_t dec_k_col(int kk, int g) { return (uint32_t)(kk * 32 + 8 * g); }
DS5_HD uint32_t dec_v_col(int c, int RC) { return (uint32_t)((c % RC) * 8); }
// Page-table entry of sequence b for position pos, and the first pool slot of
// the page it names (a position's slot adds pos % page_size). An entry outside
// [0, n_pages) reads page 0 and raises `bad`.
DS5_HD uint64_t dec_page_index(uint32_t b, uint32_t max_pages, uint32_t pos, uint32_t page_size) {
    return (uint64_t)b * max_pages + pos / page_size;
}
DS5_HD uint64_t dec_page_first(int32_t entry, uint32_t n_pages, uint32_t page_size, bool& bad) {
    const bool ok = (uint32_t)entry < n_pages;
    bad |= !ok;
    return (uint64_t)(ok ? entry : 0) * page_size;
}

// Paged plan: a length outside [1, max_len] is poisoned (0, one item); the chunk
// is the smallest multiple of `step` in [plan_cmin, plan_cmax] whose item count
// sum_b plan_items(L_b, c) fits the cap. Items: every sequence's whole chunks
// first, then the partial last chunks (and the poisoned sequences).
DS5_HD uint32_t plan_len(int32_t len, uint32_t max_len) {
    return (len < 1 || (uint32_t)len > max_len) ? 0u : (uint32_t)len;
}
DS5_HD uint32_t plan_items(uint32_t len, uint32_t c) { return len == 0 ? 1u : (len + c - 1) / c; }
DS5_HD uint32_t plan_cmax(uint32_t max_len, uint32_t step) { return (max_len + step - 1) / step * step; }
DS5_HD uint32_t plan_cmin(uint32_t max_len, uint32_t step, uint32_t max_splits) {
    return umax(step, (max_len + max_splits - 1) / max_splits + step - 1) / step * step;
}
DS5_HD uint32_t plan_whole(uint32_t len, uint32_t chunk) { return len / chunk; }
DS5_HD uint32_t plan_partial(uint32_t len, uint32_t chunk) { return (len == 0 || len % chunk != 0) ? 1u : 0u; }

// ---------------------------------------------------------------------------
// matmul_q8_mfma_kernel: block b's direct-to-LDS loads.
// x: load i of wavefront `wave` fills stage bytes o = 1024 (wave + W i) + 16 lane;
//    its plane byte offset (block 0) is row min(m0 + r, m - 1), swizzled chunk c.
// raw q: row r of the wavefront's 32 takes 48 bytes, three 16-byte lanes with dwords 0..3,
//    4..7 and 5..8 of the nine from the dword boundary at or below its block: unit u = 3 r +
//    part, 96 of them in two loads (the second's other lanes repeat the last). The offsets are
//    from the block's scalar base (w + 34 b, or w + 34 b - 2 for odd b).
// ---------------------------------------------------------------------------
DS5_HD uint32_t gemm_x_tile_row(uint32_t o, uint32_t BM) { return (o % (BM * 64)) / 64; }
// the offset of tile row r's swizzled chunk in plane row `row`
DS5_HD uint32_t gemm_x_off_row(uint32_t r, uint32_t lane, uint32_t row, uint32_t k) {
    return row * k * 2 + 16 * ((lane & 3) ^ ((r >> 2) & 3));
}
DS5_HD uint32_t gemm_x_off(uint32_t o, uint32_t lane, uint32_t BM, uint32_t m0, uint32_t m, uint32_t k) {
    const uint32_t r = gemm_x_tile_row(o, BM);
    return gemm_x_off_row(r, lane, umin(m0 + r, m - 1), k);
}
DS5_HD uint32_t gemm_q_unit(uint32_t i, uint32_t lane) { return umin(64u * i + lane, 95u); }
// the tile row and the first of the four dwords of unit u of wavefront `wave`
DS5_HD uint32_t gemm_q_row(uint32_t u, uint32_t wave) { return 32 * wave + u / 3; }
DS5_HD uint32_t gemm_q_dword(uint32_t u) { return u % 3 == 0 ? 0u : u % 3 + 3u; }
DS5_HD void gemm_q_off(uint32_t d, uint32_t row, uint32_t n0, uint32_t n, uint32_t row_bytes, uint32_t& even,
                       uint32_t& odd) {
    const uint32_t rb = umin(n0 + row, n - 1) * row_bytes;
    even = (rb & ~3u) + 4 * d;
    odd = ((rb + 2) & ~3u) + 4 * d;
}
// The blocks [first, first + count) of group `group` of ks (every group runs the same number
// of iterations; one past its blocks, or without any, repeats block `last`).
DS5_HD void gemm_group_blocks(uint32_t nb, uint32_t group, uint32_t ks, uint32_t& iters, uint32_t& first,
                              uint32_t& count, uint32_t& last) {
    iters = (nb + ks - 1) / ks;
    first = umin(group * iters, nb - 1);
    count = umin(iters, nb - umin(group * iters, nb));
    last = first + umax(count, 1u) - 1;
}

// ---------------------------------------------------------------------------
// prefill_attention_kernel: a K (or V) tile's direct-to-LDS loads fill one stage
// of 64 rows at row stride RS bytes; load b's lane covers stage bytes
// 1024 b + 16 lane: row r, chunk slot c (a padding slot re-reads the row's first
// chunk). pf_tile_off is that lane's byte offset from the tile's first key row
// (row bytes 2 D); on a tile that reaches past kv_end, rows at or past it are
// clamped to kv_end - 1 (pf_clamped_off).
// ---------------------------------------------------------------------------
DS5_HD uint32_t pf_tile_off(int b, int lane, int D, int RS) {
    const int pos = 1024 * b + 16 * lane;
    const int r = pos / RS, c = (pos % RS) / 16;
    return (uint32_t)(r * 2 * D + (c < D / 8 ? 16 * c : 0));
}
DS5_HD uint32_t pf_clamped_off(uint32_t off, uint32_t key0, uint32_t kv_end, int D) {
    const uint32_t last_row = kv_end - key0 - 1;
    return umin(off / (2 * D), last_row) * (2 * D) + off % (2 * D);
}
// Key tiles that q tile qt needs, and the first of them of part s of n_splits.
DS5_HD uint32_t pf_key_tiles(uint32_t pos, uint32_t qt, uint32_t n_tokens) {
    return (pos + umin(n_tokens, qt * kPfQRows + kPfQRows) + kPfKTile - 1) / kPfKTile;
}
DS5_HD uint32_t pf_split_first(uint32_t n, uint32_t s, uint32_t n_splits) { return n * s / n_splits; }
// A q tile's row `row` (< 32) reads token min(q0 + row, n_tokens - 1).
DS5_HD uint32_t pf_q_token(uint32_t q0, uint32_t row, uint32_t n_tokens) { return umin(q0 + row, n_tokens - 1); }

// ---------------------------------------------------------------------------
// attn_f32_kernel. Query rows R = t * group + head in the group; a wavefront (wave_rows) or
// a workgroup takes the kAfRows rows from af_row0. Positions at or past a split's end re-read
// the one before it.
// ---------------------------------------------------------------------------
DS5_HD uint32_t af_row0(uint32_t bx, uint32_t wave, bool wave_rows) {
    return (wave_rows ? bx * kAfWaves + wave : bx) * kAfRows;
}
DS5_HD uint32_t af_load_pos(uint32_t p, uint32_t end) { return umin(p, end - 1); }
// What the split of positions from `start` leaves of a row whose last position is lim: nothing
// where the row ends before the split (tiles hold rows of several tokens, and the other rows
// may go on), the output itself where the row has no other split, or a partial result.
enum AfStore : int { kAfNone = 0, kAfOut = 1, kAfPart = 2 };
DS5_HD int af_store(uint32_t lim, uint32_t start, uint32_t chunk) {
    return lim < start ? kAfNone : lim < chunk ? kAfOut : kAfPart;
}
// The splits that hold a partial result of the row (1: its only split wrote the output).
DS5_HD uint32_t af_row_splits(uint32_t lim, uint32_t chunk) { return lim / chunk + 1; }

// ---------------------------------------------------------------------------
// paged_attention_kernel. A sequence's query rows of one kv head are its new tokens' q heads
// of that group, row = token * group + head, in tiles of kPbRows; tile i attends the positions
// below its last token's. The batch's work is one line: for each kv head, each sequence, each
// tile in the order last, first, last but one, second, ... (a pair of them costs the same for
// every pair), its positions. Workgroup w of n takes the part from w / n to (w + 1) / n of it.
// Work is counted in half positions * group for the tiles of sequences of at most kPbNarrow rows
// and in fifths for the others (64 positions of heads of 128 measured 0.5 .. 0.7 us and 1.3 .. 1.5: 4.7 ns
// a unit), a tile's being its positions (taken as if every tile were full) and before them kPbTileCost
// for beginning and ending it (9 .. 12 us). From caches in memory, two prompts among 22 single tokens
// take 83 us so, 89 with sixths and 3200; six and six 120 and 124. A workgroup whose part begins inside
// a tile, or ends there, pays that as every other does; what counts is the tiles that it begins after
// another, so the cost lies at the tile's start, and cuts there fall on the start. A cut further on
// falls on a multiple of kPbUnit positions, or on the tile's start or end where that is no further
// than `snap`.
// ---------------------------------------------------------------------------
constexpr uint32_t kPbRows = 128, kPbNarrow = 32, kPbUnit = 64, kPbTileCost = 2304, kPbPiece = 384;

struct PbSeq {
    uint32_t n, before;  // new tokens, and the tokens before them
};
struct PbTile {
    uint32_t row0, rows, kv;  // first query row, rows, positions that the last of them attends
};
struct PbCut {
    uint32_t kvh, b, j, k;  // kv head, sequence, the j-th tile of its order, position
};

DS5_HD uint32_t pb_tiles(PbSeq s, uint32_t group) { return (s.n * group + kPbRows - 1) / kPbRows; }
// Work as a double that holds an integer below 2^53 (the device multiplies 64-bit integers several times slower).
DS5_HD double pb_weight(PbSeq s, uint32_t group) { return s.n * group > kPbNarrow ? 5.0 : 2.0; }
DS5_HD double pb_tile_work(PbSeq s, uint32_t group, uint32_t tile) {
    return (double)group * kPbTileCost + pb_weight(s, group) * ((double)group * s.before + (double)kPbRows * (tile + 1));
}
DS5_HD double pb_seq_work(PbSeq s, uint32_t group) {
    const double nt = pb_tiles(s, group);
    return nt * ((double)group * kPbTileCost + pb_weight(s, group) * ((double)group * s.before + kPbRows / 2 * (nt + 1.0)));
}
DS5_HD uint32_t pb_tile_at(uint32_t j, uint32_t nt) { return j % 2 ? j / 2 : nt - 1 - j / 2; }
// x / d with inv = 1.0 / d: the floor of (x + 1/2) / d, which is half of 1 / d or more away from every integer.
DS5_HD uint32_t pb_over(uint32_t x, double inv) { return (uint32_t)(((double)x + 0.5) * inv); }
DS5_HD PbTile pb_tile(PbSeq s, uint32_t group, double inv_group, uint32_t tile) {
    const uint32_t all = s.n * group, row0 = tile * kPbRows, end = umin(all, row0 + kPbRows);
    return PbTile{row0, end - row0, s.before + pb_over(end - 1, inv_group) + 1};
}
// 1 / d for d from 1 on, to 2^-44 or better: the device's estimate (to 2^-22) and one step of Newton's method.
// (A division of doubles takes several times as long there, one of 64-bit integers longer still.) The host's, which
// the tests walk the plan with, takes the step from an estimate as far off as they ask, another way for each d.
inline double pb_estimate_error = 0.0;
DS5_HD double pb_inverse(double d) {
#if defined(__HIP_DEVICE_COMPILE__)
    const double r = __builtin_amdgcn_rcp(d);
#else
    const double r = (1.0 / d) * (1.0 + pb_estimate_error * sin(d));
#endif
    return __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
}
// x = q * d + r in integers, q below 2^32: the rounded quotient is at most one off.
DS5_HD uint32_t pb_divide(double x, double d, double& r) {
    double q = floor(x * pb_inverse(d));
    r = fma(-q, d, x);
    if (r < 0.0) {
        q -= 1.0;
        r += d;
    } else if (r >= d) {
        q += 1.0;
        r -= d;
    }
    return (uint32_t)q;
}
// The cut at y of a sequence's work: tile j of its order (j may be one past the last) that begins
// `at` into that work, position k.
struct PbPlace {
    uint32_t j, k;
    double at;
};
DS5_HD PbPlace pb_locate(PbSeq s, uint32_t group, double inv_group, double y, double snap, double lead, bool whole) {
    const uint32_t nt = pb_tiles(s, group);
    double off = y;
    uint32_t j = 0;
    if (nt > 1) {
        const double pair = pb_tile_work(s, group, nt - 1) + pb_tile_work(s, group, 0);
        j = pb_divide(y, pair, off) * 2;
        const double heavy = pb_tile_work(s, group, pb_tile_at(j, nt));
        if (j + 1 < nt && off >= heavy) {
            j++;
            off -= heavy;
        }
    }
    const uint32_t tile = pb_tile_at(j, nt);
    const double w = pb_tile_work(s, group, tile), at = y - off;
    if (whole) return off * 2.0 >= w ? PbPlace{j + 1, 0, at + w} : PbPlace{j, 0, at};  // cuts between tiles only
    if (off < snap || off <= lead) return PbPlace{j, 0, at};
    if (w - off < snap) return PbPlace{j + 1, 0, at + w};
    const uint32_t kv = pb_tile(s, group, inv_group, tile).kv;
    return PbPlace{j, umin((uint32_t)(kv * (off - lead) * pb_inverse(w - lead)), kv - 1) / kPbUnit * kPbUnit, at};
}
// The cut before workgroup w of n on a line of `work`: rounded, but never backwards as w grows, and
// the same wherever it is worked out. part: 1.0 / n.
DS5_HD double pb_cut_at(double work, uint32_t w, uint32_t n, double part) { return w >= n ? work : floor(work * (w * part)); }
// The last workgroup whose cut is at most x (x below work).
DS5_HD uint32_t pb_last_cut(double work, uint32_t n, double part, double x) {
    uint32_t w = umin((uint32_t)(x * pb_inverse(work) * n), n - 1);
    while (w > 0 && pb_cut_at(work, w, n, part) > x) w--;
    while (w + 1 < n && pb_cut_at(work, w + 1, n, part) <= x) w++;
    return w;
}
DS5_HD double pb_snap(double work, double part, uint32_t group) {
    return fmax(floor(work * part * 0.0625), (double)group * (kPbUnit / 2));
}
// A tile's cost that lies before its positions; of tiles that several workgroups share, no more than
// leaves each of them some.
DS5_HD double pb_lead(double work, double part, uint32_t group) {
    return fmin(floor(work * part * 0.5), (double)group * kPbTileCost);
}
// The workgroups that share a line of work: kPbPiece of a row's work each at least, and the same number
// for each kv head where there are enough, so that no workgroup ends one head's tile to begin another's.
DS5_HD uint32_t pb_workgroups(double work, double inv_group, uint32_t heads, double inv_heads, uint32_t grid) {
    const double n = work * inv_group * (1.0 / kPbPiece);
    const uint32_t all = n >= (double)grid ? grid : n < 1.0 ? 1 : (uint32_t)n;
    return all > heads ? pb_over(all, inv_heads) * heads : all;
}
// Moves c on to the next tile that has rows; false where that is past the part that ends at `end`.
// at_end: the part ends inside this tile, at position end.k. seq(b) gives sequence b.
template <class Seq>
DS5_HD bool pb_next(PbCut& c, const PbCut& end, uint32_t n_seqs, uint32_t n_kv_heads, uint32_t group, Seq seq, bool& at_end) {
    while (c.kvh < n_kv_heads && (c.b >= n_seqs || c.j >= pb_tiles(seq(c.b), group))) {
        c.j = c.k = 0;
        if (++c.b >= n_seqs) {
            c.b = 0;
            c.kvh++;
        }
    }
    at_end = c.kvh == end.kvh && c.b == end.b && c.j == end.j;
    if (c.kvh >= n_kv_heads || (at_end && end.k == 0)) return false;
    return c.kvh < end.kvh || (c.kvh == end.kvh && (c.b < end.b || (c.b == end.b && c.j <= end.j)));
}
// Lane's byte offset, from the first row of a group of 16 rows of 2 D bytes, of its 16 bytes of
// direct-to-LDS load b (LDS bytes 1024 b + 16 lane of the group): 16-byte chunk c of row r lies
// in the row's slot c ^ (pb_swz of the row).
DS5_HD uint32_t pb_swz(int D, bool v, uint32_t r) {
    return v ? 4 * (D == 128 ? r & 3 : (r >> 1) & 1) : D == 128 ? r & 15 : (r >> 1) & 7;
}
DS5_HD uint32_t pb_load_off(int D, bool v, int b, int lane) {
    const uint32_t at = 1024 * b + 16 * lane, r = at / (2 * D), slot = at % (2 * D) / 16;
    return r * (2 * D) + (slot ^ pb_swz(D, v, r)) * 16;
}

}  // namespace ds5idx
