/*
 * paged_cache.h — C-ABI of the caption decoder's paged key / value cache: attention of a chunk of new
 * tokens over the cache (csrc/paged_attention.hip) and the page pool's updates (csrc/paged_cache.hip),
 * built into libmsda_hip.so.
 *
 * A cache of L layers is one buffer `data` (L, 2, pages, kv_heads, page_size, dim): keys at [:, 0],
 * values at [:, 1], page_size a power of two up to 1024.  Sequence s owns the pages table[s][0 ..] (int32, -1 behind
 * the last one) and lens[s] tokens in them; refs[x] counts the sequences that hold page x (0 = free), so
 * sequences share the pages of a common beginning.
 *
 * All functions are asynchronous on `stream`, may be captured into a graph, and return 0, else non-zero with
 * mfl_paged_last_error().  They launch on the current device, which has to be the stream's.
 */
#ifndef MFL_PAGED_CACHE_H
#define MFL_PAGED_CACHE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Attention of new tokens over one layer's pages.  Row i of sequence s sits at position p = starts[s] + i
 * (starts NULL: kv_lens[s] - the sequence's rows); query head h reads key / value head h / (heads / kv_heads).
 * Key j of s is row j % page_size of page table[s][j / page_size]; it is visible to the row when
 * j < min(kv_lens[s], width * page_size), j <= p (causal) and the page number is in [0, pages).
 *   out[row] = sum_j softmax_j(scale * q . k_j) v_j,   0 where no key is visible.
 * With k_new / v_new the chunk's own keys and values are also written to the pages, row i at position p
 * (dropped when p < 0, p >= kv_lens[s] or the page number is out of range), and read from there.
 *
 * Rows: offsets NULL — `rows` rows of every sequence, sequence s's row i at s * *_seq + i * *_row (elements);
 * offsets (n + 1, int32, ascending) — sequence s has rows offsets[s] .. offsets[s + 1] of `total` packed rows
 * *_row apart, `rows` bounds their number (further ones are neither computed nor written), and rows before
 * offsets[0] or behind offsets[n] are set to zero when zero_tail, else left as they were.  q, k_new, v_new heads are *_head apart, the last
 * dimension contiguous, all strides multiples of 16 bytes; out is contiguous.
 * dtype: 0 float32, 2 bfloat16, 3 float16.  dim <= 128, a multiple of 16 bytes.  max_kv bounds kv_lens
 * for the choice of the launch only (a larger one is still computed in full).  workspace:
 * mfl_paged_attention_workspace_bytes(args) bytes, 16-byte aligned. */
typedef struct {
  const void *q, *k_new, *v_new;
  void *k_pages, *v_pages, *out, *workspace;
  const int32_t *table, *kv_lens, *starts, *offsets;
  int64_t n, rows, total, heads, kv_heads, dim, pages, page_size, width, max_kv;
  int64_t q_seq, q_row, q_head, k_seq, k_row, k_head, v_seq, v_row, v_head;
  int64_t dtype, causal, zero_tail;
  double scale;
} mfl_paged_attention_args;

int64_t mfl_paged_attention_workspace_bytes(const mfl_paged_attention_args* args);

int mfl_paged_attention(const mfl_paged_attention_args* args, void* stream);

/* The page pool.  One call brings every row from (table, lens, refs) to a new state; row s becomes a share of
 * row parents[s] (NULL: itself; outside [0, n): an empty row), cut or grown to new_lens[s] tokens (NULL: the
 * parent's length), clamped to [0, width * page_size]:
 *   1. refs' = refs - the pages of the rows as they were + the pages the new rows keep (the first
 *      min(length of the parent, new length) tokens'); pages of refs' = 0 are free
 *   2. a row that grows from inside a page with refs' > 1 gets a copy of its own of that page's used tokens,
 *      in every layer — except the highest such row of a page that no other row keeps
 *   3. the copy's page and the pages of the new tokens are asked for in row order, within a row in that order,
 *      and the i-th asked for is the i-th lowest free page
 * If more are asked for than are free nothing changes (outputs equal inputs) and *short_out is the number
 * lacking, else 0.  Table entries behind a row's last page are -1; entries outside [0, pages) hold nothing.
 * refs may count holders outside the table.  Outputs must not overlap inputs.  data (planes, pages, heads,
 * page_size, row_bytes), planes = 2 * layers, row_bytes a multiple of 16; NULL: no data (planes ignored).
 * n <= 2^20.  workspace: mfl_pages_update_workspace_bytes(n, pages) bytes, 16-byte aligned. */
int64_t mfl_pages_update_workspace_bytes(int64_t n, int64_t pages);

int mfl_pages_update(const int32_t* table, const int32_t* lens, const int32_t* refs, const int32_t* parents,
                     const int32_t* new_lens, int64_t n, int64_t width, int64_t pages, int64_t page_size, void* data,
                     int64_t planes, int64_t heads, int64_t row_bytes, int32_t* table_out, int32_t* lens_out,
                     int32_t* refs_out, int32_t* short_out, void* workspace, void* stream);

/* Live pages (refs > 0) brought to the front: with L of them, the k-th lowest live page >= L moves to the k-th
 * lowest free page < L, in every plane; page_bytes = heads * page_size * row_bytes, a multiple of 16.
 * remap_out[x]: the new number of page x, -1 if free; table entries outside [0, pages) and of free pages
 * become -1.  live_out: L.  Outputs must not overlap inputs.  workspace:
 * mfl_pages_compact_workspace_bytes(pages) bytes. */
int64_t mfl_pages_compact_workspace_bytes(int64_t pages);

int mfl_pages_compact(const int32_t* table, int64_t entries, const int32_t* refs, int64_t pages, void* data,
                      int64_t planes, int64_t page_bytes, int32_t* table_out, int32_t* refs_out, int32_t* remap_out,
                      int32_t* live_out, void* workspace, void* stream);

/* Page src[i] copied to page dst[i] in every plane, i < count; pairs with a number outside [0, pages) are
 * skipped.  No page may be both a source and a destination, nor a destination twice. */
int mfl_pages_copy(const int32_t* src, const int32_t* dst, int64_t count, void* data, int64_t planes, int64_t pages,
                   int64_t page_bytes, void* stream);

const char* mfl_paged_last_error(void);

#ifdef __cplusplus
}
#endif

#endif
