/*
 * ds5_paged_index.h -- test hooks of the paged batch's attention, as those of ds5_index.h: host
 * wrappers of the arithmetic of qw3_amd/csrc/ds5_index.hpp that paged_attention_kernel runs on
 * the device. Not part of the kernel provider; no reference counterpart.
 */
#ifndef DS5_PAGED_INDEX_H
#define DS5_PAGED_INDEX_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* paged_attention_kernel: the parts of a ragged batch over `grid` workgroups, ten words each:
 * workgroup, kv head, sequence, tile, first position, end, positions of the tile, its first query
 * row, its rows, and the last workgroup with a part of it where this one begins it and does not end
 * it (else itself); returns their number (at most `max` are written). n and before: each sequence's
 * new tokens and those before them. Byte offsets [loads][64] of a group of 16 K (v = 0) or V rows'
 * direct-to-LDS loads. */
uint32_t ds5_index_pb_parts(uint32_t n_seqs, const uint32_t* n, const uint32_t* before, uint32_t group, uint32_t n_kv_heads,
                            uint32_t grid, int whole, uint32_t max, uint32_t* out);
/* How far off, relative, the reciprocals' estimates are that ds5_index_pb_parts works from (0 at first; the
 * device's at most 2^-22). */
void ds5_index_pb_estimate(double error);
void ds5_index_pb_loads(uint32_t head_dim, int v, uint32_t* off);

#ifdef __cplusplus
}
#endif

#endif /* DS5_PAGED_INDEX_H */
