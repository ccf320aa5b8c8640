/*
 * C ABI of the operators on the pages of a cache: giving requests the pages that they need and taking back the others, continuing
 * requests (forks, reordered beams) with the partly filled page copied, and moving the pages in use to the front.
 *
 * A block table [requests, entries] names pages 0 .. blocks - 1; any other number is an empty entry (written as -1). `counts` [blocks] says how many
 * entries name a page; a page with 0 is free. The calls keep it so; if it is not so before a call, which pages are given out is not defined, but nothing outside of the tensors
 * is accessed. Entries of a request's first ceil(length / page_rows) pages count (of lengths below 0 as of 0, behind the table as of all of it).
 *
 * All pointers in the structs are device pointers valid on the current device, except `tensors`. Functions only enqueue work on `stream` (a cudaStream_t) and never
 * synchronise; 0 is success, -1 a call outside of what is stated here (nothing is enqueued), anything else the CUDA error code of the failed enqueue.
 * `workspace` (16-byte aligned, of the size that the functions of that name give): its contents matter to nobody between calls, but calls that may run at the same time need one each.
 *
 * `status`: SPARSE_MLA_STATUS_WORDS int32 words (sparse_mla.h), set to the first report if word 0 is zero: SPARSE_MLA_STATUS_NO_PAGE, request (fork: row of table_out), entry where no free page was
 * left, whose entry stays empty; SPARSE_MLA_STATUS_BAD_PAGE, request, length for a length behind the table.
 */
#ifndef ASCENDFLOW_B200_PAGES_H_
#define ASCENDFLOW_B200_PAGES_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PAGES_MOST_BLOCKS (1 << 23)
#define PAGES_MOST_TENSORS 128

/* Tables may have up to 2^31 - 1 entries, caches up to PAGES_MOST_BLOCKS pages. table_out is table_in or disjoint from it (in `launch_pages_fork` always disjoint),
 * counts_out is counts_in or disjoint from it. */
typedef struct {
  const int32_t* table_in; /* [requests, entries] */
  int32_t* table_out;      /* resize, compact: [requests, entries]; fork: [children, entries] */
  const int32_t* counts_in; /* [blocks] */
  int32_t* counts_out;
  const int32_t* lengths;   /* [requests]; compact: unused */
  void* workspace;
  int32_t* status;
  int64_t requests, entries, blocks, page_rows;
} pages_call;

/* What lies in pages: memory of `blocks` pages of `page_bytes` each, in `rows` equal parts that stand for page_rows / rows cached rows each. */
typedef struct {
  void* memory;
  int64_t page_bytes, rows;
} pages_tensor;

/* Entries that lengths count and that are empty get the free pages of lowest number, in the order of requests and entries; pages of entries that lengths do not count are
 * given back first (their counts go down), and their entries become empty. */
int workspace_size_pages_resize(uint64_t* bytes, const pages_call* call);
int launch_pages_resize(void* stream, const pages_call* call);

/* Row i of table_out continues request parents[i]: it has the entries that this one's length counts, the others are empty; so are all of a row whose
 * parent is no request (whose length from then on is 0). A last page that is partly filled goes on in one row: the first that continues the request keeps it if its count is 1 (nobody else names it), and every
 * other gets one of the pages that are free before the call (lowest numbers first, in the order of the rows) with a copy of the filled rows in every tensor (parts that are
 * filled in part are copied whole). So rows may be appended to, also where a length is shorter than the request was when it shared its pages. counts_out counts the entries of table_out instead of those of table_in. Sources and targets of copies are different pages. */
typedef struct {
  pages_call pages;
  const int32_t* parents;      /* [children] */
  const pages_tensor* tensors; /* host memory, [tensor_count] */
  int64_t children, tensor_count;
} pages_fork_call;
int workspace_size_pages_fork(uint64_t* bytes, const pages_fork_call* call);
int launch_pages_fork(void* stream, const pages_fork_call* call);

/* With U pages in use: the k-th page in use from number U on is moved to the k-th free page in front of U, in every tensor (whole pages), counts with them. places[p] is
 * the number that page p has then, -1 for free ones; table_out has the new numbers (empty entries as they are). */
typedef struct {
  pages_call pages;
  int32_t* places;             /* [blocks] */
  const pages_tensor* tensors; /* host memory, [tensor_count] */
  int64_t tensor_count;
} pages_compact_call;
int workspace_size_pages_compact(uint64_t* bytes, const pages_compact_call* call);
int launch_pages_compact(void* stream, const pages_compact_call* call);

#ifdef __cplusplus
}
#endif
#endif /* ASCENDFLOW_B200_PAGES_H_ */
