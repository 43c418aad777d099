// Page tables of a batch over pools of cache pages, kept on the device
// (gfx950): rows forked, reordered and dropped, pages freed and handed out, the
// pools closed up.  No call waits for the device or reads it back, so a
// captured decode loop can hold them; the reference keeps one sequence and its
// pages in Python lists (src/bmx/cache/packed_streaming.py:116-267).
//
// The state: `rows` table rows of `cap` page ids, row r's first n_pages[r]
// entries its pages in order; refs[p], the uses of pool page p (one a table
// entry, and one for every holder outside the tables); and a stack of free ids,
// free[0 .. n_free), the top at its end.  One state serves the pools of all
// layers (a page id means the same page of each), of whatever page format.  The
// calls write a new state and leave the given one as it is; their buffers must
// not overlap.
#ifndef BMX_PAGES_H
#define BMX_PAGES_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define BMX_PAGES_E_INVALID 1
#define BMX_PAGES_E_WORKSPACE 2
#define BMX_PAGES_E_HIP 3

// status words of an update (device)
#define BMX_PAGES_OK 0
#define BMX_PAGES_NO_FREE 1   // fewer free pages than all rows ask for
#define BMX_PAGES_NO_ROOM 2   // a row would grow past cap

#define BMX_PAGES_MAX_POOLS 128

typedef struct bmx_pages_state {
  int32_t* table;     // device [rows][cap]
  int32_t* n_pages;   // device [rows], taken within 0..cap
  int32_t* refs;      // device [n_pool]
  int32_t* free;      // device [n_pool]
  int32_t* n_free;    // device [1], taken within 0..n_pool
} bmx_pages_state;

// New row i continues old row index[i] (forked where several do, dropped where
// none does; empty where index[i] is outside 0..rows - 1).  Then
//   refs'[p] = refs[p] - (entries p of the old rows) + (entries p of the new ones);
// pages with refs > 0 >= refs' are free: they go onto the stack in ascending
// order.  Then row i gets grow[i] more pages off the top, row 0 first, each
// with refs' = 1 -- all rows or, where the stack or some row is too short, none
// (status).  Entries past a row's pages become 0, free ids past n_free' -1.
// Entries outside the pool are copied and not counted.
typedef struct bmx_pages_update_args {
  bmx_pages_state in, out;
  int32_t rows, new_rows;   // 1..16384 each
  int32_t cap;              // entries of a row, old and new: 1..2^22
  int32_t n_pool;           // 1..2^22
  const int32_t* index;     // device [new_rows], or NULL: every row as it is (new_rows == rows)
  const int32_t* grow;      // device [new_rows] (below 0: 0), or NULL: none
  int32_t* status;          // device [1]
  void* workspace;          // bmx_pages_update_workspace_bytes(), 16-byte aligned
  size_t workspace_bytes;
} bmx_pages_update_args;

size_t bmx_pages_update_workspace_bytes(const bmx_pages_update_args* a);
int bmx_pages_update(const bmx_pages_update_args* a, void* stream);

// With n live pages (refs > 0), those at ids n and up move to the free ids below
// n, lowest to lowest, in every pool; tables, refs and the stack follow (the
// stack hands out the lowest id first).  What a page left behind stays as it
// was.  The pools are changed in place.  A holder outside the tables is not told
// its pages' new ids: one that reads them keeps them as a row of the table.
typedef struct bmx_pages_compact_args {
  bmx_pages_state in, out;
  int32_t rows, cap, n_pool;
  int32_t n_pools;                            // 0..128
  void* pools[BMX_PAGES_MAX_POOLS];           // device [n_pool][page_bytes], 16-byte aligned
  int64_t page_bytes[BMX_PAGES_MAX_POOLS];    // multiples of 16
  void* workspace;
  size_t workspace_bytes;
} bmx_pages_compact_args;

size_t bmx_pages_compact_workspace_bytes(const bmx_pages_compact_args* a);
int bmx_pages_compact(const bmx_pages_compact_args* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif
