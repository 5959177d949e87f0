// The host's side of the 4-bit paged cache: which page holds which positions of
// which row, how many rows hold a page, which pages are free.  Plain loops over the
// caller's arrays; nothing here touches the device.
#include <stdlib.h>
#include <string.h>

#include "pages4.h"

namespace tsattn {
namespace {

int32_t *row_of(const tsattn_pages4_host *h, int32_t row) { return h->table + static_cast<int64_t>(row) * h->columns; }

void let_go(tsattn_pages4_host *h, int32_t page) {
  if (--h->refs[page] == 0) h->stack[h->free++] = page;
}

int32_t take(tsattn_pages4_host *h) {
  const int32_t page = h->stack[--h->free];
  h->refs[page] = 1;
  return page;
}

int32_t pages_of(const tsattn_pages4_host *h, int64_t positions) {
  return static_cast<int32_t>((positions + h->page_size - 1) / h->page_size);
}

}  // namespace

// Pages of their own for the next `steps` positions of the rows.  A row that appends
// into a page that others hold too gets a copy of it (src -> dst); of the holders
// that all append, the last keeps the page.  Counted first, so that too few free
// pages change nothing: returns how many are needed then, else 0.
int32_t pages4_grow(tsattn_pages4_host *h, int32_t n, const int32_t *rows, int32_t steps, int32_t *src,
                    int32_t *dst, int32_t *at, int32_t *value, int32_t *copies, int32_t *sets) {
  int64_t need = 0;
  int32_t shared = 0;
  for (int32_t i = 0; i < n; ++i) {
    const int32_t len = h->lengths[rows[i]], *row = row_of(h, rows[i]);
    if (len % h->page_size) {
      const int32_t page = row[len / h->page_size];
      if (h->refs[page] > 1) {
        --h->refs[page];
        src[shared] = page;
        dst[shared++] = rows[i];  // (its row, until its copy is known)
        ++need;
      }
    }
    for (int32_t c = len / h->page_size, stop = pages_of(h, static_cast<int64_t>(len) + steps); c < stop; ++c)
      need += row[c] < 0;
  }
  if (need > h->free) {
    for (int32_t i = 0; i < shared; ++i) ++h->refs[src[i]];
    return static_cast<int32_t>(need < INT32_MAX ? need : INT32_MAX);
  }
  int32_t k = 0;
  for (int32_t i = 0; i < shared; ++i) {
    const int32_t row = dst[i], c = h->lengths[row] / h->page_size;
    dst[i] = row_of(h, row)[c] = take(h);
    at[k] = row * h->columns + c;
    value[k++] = dst[i];
  }
  for (int32_t i = 0; i < n; ++i) {
    const int32_t len = h->lengths[rows[i]];
    int32_t *row = row_of(h, rows[i]);
    for (int32_t c = len / h->page_size, stop = pages_of(h, static_cast<int64_t>(len) + steps); c < stop; ++c)
      if (row[c] < 0) {
        row[c] = take(h);
        at[k] = rows[i] * h->columns + c;
        value[k++] = row[c];
      }
  }
  *copies = shared;
  *sets = k;
  return 0;
}

// The rows end at `lengths`; pages wholly past them are given back.
void pages4_cut(tsattn_pages4_host *h, int32_t n, const int32_t *rows, const int32_t *lengths) {
  for (int32_t i = 0; i < n; ++i) {
    int32_t *row = row_of(h, rows[i]);
    for (int32_t c = pages_of(h, h->lengths[rows[i]]); c-- > pages_of(h, lengths[i]);)
      if (row[c] >= 0) {
        let_go(h, row[c]);
        row[c] = -1;
      }
    h->lengths[rows[i]] = lengths[i];
  }
}

// Row rows[i] takes over the pages and the length of rows[index[i]].  `old` has room
// for the n rows' entries and lengths.
void pages4_reorder(tsattn_pages4_host *h, int32_t n, const int32_t *rows, const int32_t *index, int32_t *old,
                    int32_t *at, int32_t *value, int32_t *sets) {
  const int32_t width = h->columns + 1;
  for (int32_t i = 0; i < n; ++i) {
    memcpy(old + static_cast<int64_t>(i) * width, row_of(h, rows[i]), sizeof(int32_t) * h->columns);
    old[static_cast<int64_t>(i) * width + h->columns] = h->lengths[rows[i]];
  }
  int32_t k = 0;
  for (int pass = 0; pass < 2; ++pass)  // (all are taken before any is let go)
    for (int32_t i = 0; i < n; ++i) {
      if (index[i] == i) continue;
      const int32_t *mine = old + static_cast<int64_t>(i) * width, *from = old + static_cast<int64_t>(index[i]) * width;
      if (pass) {
        for (int32_t c = pages_of(h, mine[h->columns]); c-- > 0;)
          if (mine[c] >= 0) let_go(h, mine[c]);
        continue;
      }
      int32_t *row = row_of(h, rows[i]);
      const int32_t had = pages_of(h, mine[h->columns]), has = pages_of(h, from[h->columns]);
      for (int32_t c = 0; c < (had > has ? had : has); ++c) {
        row[c] = from[c];
        if (from[c] < 0) continue;
        ++h->refs[from[c]];
        if (from[c] != mine[c]) {
          at[k] = rows[i] * h->columns + c;
          value[k++] = from[c];
        }
      }
      h->lengths[rows[i]] = from[h->columns];
    }
  *sets = k;
}

}  // namespace tsattn
