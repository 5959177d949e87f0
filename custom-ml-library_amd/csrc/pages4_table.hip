// The host's side of the 4-bit paged cache: which page holds which positions of
// which row, how many rows hold a page, which pages are free, which table entries
// the device's copy lacks.  Plain loops over the caller's arrays; nothing here
// touches the device.
#include <stdlib.h>
#include <string.h>

#include "pages4.h"

namespace tsattn {
namespace {

int32_t *row_of(const tsattn_pages4_host *h, int32_t row) { return h->table + static_cast<int64_t>(row) * h->columns; }

void let_go(tsattn_pages4_host *h, int32_t page) {
  if (--h->refs[page] == 0 && h->free < h->pages) h->stack[h->free++] = page;
}

int32_t take(tsattn_pages4_host *h) {
  const int32_t page = h->stack[--h->free];
  h->refs[page] = 1;
  return page;
}

int32_t pages_of(const tsattn_pages4_host *h, int64_t positions) {
  return static_cast<int32_t>((positions + h->page_size - 1) / h->page_size);
}

void put(tsattn_pages4_host *h, int32_t row, int32_t column, int32_t page) {
  const int32_t at = row * h->columns + column;
  h->table[at] = page;
  if (h->shown[at] != page && !h->dirty[at]) {
    h->dirty[at] = 1;
    h->changed[h->n_changed++] = at;
  }
}

}  // namespace

// Pages of their own for the next `steps` positions of the rows.  A row that appends
// into a page that others hold too gets a copy of it (src -> dst); of the holders
// that all append, the first keeps the page.  Counted first, so that too few free
// pages change nothing: returns how many are needed then, -1 where a free page is not
// one of the pool, else 0.  Rows give pages back last to first and take them first to
// last, so that those which are cut and grow again, or fork again, find the pages that
// the device's table shows.
int32_t pages4_grow(tsattn_pages4_host *h, int32_t n, const int32_t *rows, int32_t steps, int32_t *src,
                    int32_t *dst, int32_t *copies) {
  int64_t need = 0;
  int32_t shared = 0;
  for (int32_t i = n; i-- > 0;) {
    const int32_t len = h->lengths[rows[i]], *row = row_of(h, rows[i]);
    int32_t c = len / h->page_size;
    if (len - c * h->page_size) {
      const int32_t page = row[c++];
      if (h->refs[page] > 1) {
        --h->refs[page];
        src[shared] = page;
        dst[shared++] = rows[i];  // (its row, until its copy is known)
        ++need;
      }
    }
    need += pages_of(h, static_cast<int64_t>(len) + steps) - c;
  }
  bool known = true;
  for (int64_t i = 0; i < need && need <= h->free; ++i) {
    const int32_t page = h->stack[h->free - 1 - i];
    known = known && page >= 0 && page < h->pages;
  }
  if (need > h->free || !known) {
    for (int32_t i = 0; i < shared; ++i) ++h->refs[src[i]];
    return !known ? -1 : static_cast<int32_t>(need < INT32_MAX ? need : INT32_MAX);
  }
  *copies = shared;
  if (!need) return 0;
  for (int32_t i = shared; i-- > 0;) {
    const int32_t row = dst[i];
    dst[i] = take(h);
    put(h, row, h->lengths[row] / h->page_size, dst[i]);
  }
  for (int32_t i = 0; i < n; ++i) {
    const int32_t len = h->lengths[rows[i]];
    for (int32_t c = pages_of(h, len), stop = pages_of(h, static_cast<int64_t>(len) + steps); c < stop; ++c)
      put(h, rows[i], c, take(h));
  }
  return 0;
}

// The rows end at `lengths`; pages wholly past them are given back.
void pages4_cut(tsattn_pages4_host *h, int32_t n, const int32_t *rows, const int32_t *lengths) {
  for (int32_t i = n; i-- > 0;) {
    int32_t *row = row_of(h, rows[i]);
    if (lengths[i] == h->lengths[rows[i]]) continue;
    for (int32_t c = pages_of(h, h->lengths[rows[i]]), stop = pages_of(h, lengths[i]); c-- > stop;) {
      let_go(h, row[c]);
      row[c] = -1;
    }
    h->lengths[rows[i]] = lengths[i];
  }
}

// Row rows[i] takes over the pages and the length of rows[index[i]].  `old` has room
// for the n rows' entries and lengths.
void pages4_reorder(tsattn_pages4_host *h, int32_t n, const int32_t *rows, const int32_t *index, int32_t *old) {
  const int64_t width = h->columns + 1;
  for (int32_t i = 0; i < n; ++i) {
    memcpy(old + i * width, row_of(h, rows[i]), sizeof(int32_t) * h->columns);
    old[i * width + h->columns] = h->lengths[rows[i]];
  }
  for (int32_t i = 0; i < n; ++i) {  // (all are taken before any is let go)
    const int32_t *mine = old + i * width, *from = old + index[i] * width;
    const int32_t had = pages_of(h, mine[h->columns]), has = pages_of(h, from[h->columns]);
    for (int32_t c = 0; c < has; ++c) {
      ++h->refs[from[c]];
      if (from[c] != mine[c]) put(h, rows[i], c, from[c]);
    }
    for (int32_t c = has; c < had; ++c) row_of(h, rows[i])[c] = -1;
    h->lengths[rows[i]] = from[h->columns];
  }
  for (int32_t i = n; i-- > 0;)
    for (int32_t c = pages_of(h, old[i * width + h->columns]); c-- > 0;) let_go(h, old[i * width + c]);
}

// `to`, of n rows, holds what the rows of `from` do, its pages 0, 1, .. in the order of
// the rows: src -> dst.  `number` [from->pages] is scratch.  Returns the pages in use, and does
// nothing else if `to` has fewer.
int32_t pages4_clone(const tsattn_pages4_host *from, int32_t n, const int32_t *rows, tsattn_pages4_host *to,
                     int32_t *number, int32_t *src, int32_t *dst) {
  memset(number, 0xFF, sizeof(int32_t) * from->pages);
  int32_t k = 0;
  for (int32_t i = 0; i < n; ++i)
    for (int32_t c = 0, stop = pages_of(from, from->lengths[rows[i]]); c < stop; ++c) {
      int32_t *p = number + row_of(from, rows[i])[c];
      if (*p < 0) *p = k++;
    }
  if (k > to->pages) return k;
  memset(to->table, 0xFF, sizeof(int32_t) * to->rows * static_cast<size_t>(to->columns));
  memset(to->shown, 0xFF, sizeof(int32_t) * to->rows * static_cast<size_t>(to->columns));
  memset(to->refs, 0, sizeof(int32_t) * to->pages);
  memset(to->dirty, 0, static_cast<size_t>(to->rows) * to->columns);
  to->n_changed = 0;
  for (int32_t p = 0; p < from->pages; ++p)
    if (number[p] >= 0) src[number[p]] = p, dst[number[p]] = number[p];
  for (int32_t i = 0; i < n; ++i) {
    to->lengths[i] = from->lengths[rows[i]];
    for (int32_t c = 0, stop = pages_of(from, to->lengths[i]); c < stop; ++c) {
      const int32_t page = number[row_of(from, rows[i])[c]];
      ++to->refs[page];
      put(to, i, c, page);
    }
  }
  to->free = to->pages - k;
  for (int32_t i = 0; i < to->free; ++i) to->stack[i] = to->pages - 1 - i;
  return k;
}

// The pages in use past the first n (n: how many are in use) move into the free ones
// before: src -> dst, none both.  `number` [pages] is scratch.  Returns n.
int32_t pages4_compact(tsattn_pages4_host *h, int32_t *number, int32_t *src, int32_t *dst, int32_t *copies) {
  const int32_t n = h->pages - h->free;
  int32_t hole = 0, k = 0;
  for (int32_t p = n; p < h->pages; ++p) {
    number[p] = p;
    if (!h->refs[p]) continue;
    while (h->refs[hole]) ++hole;
    h->refs[hole] = h->refs[p];
    h->refs[p] = 0;
    src[k] = p;
    dst[k++] = number[p] = hole;
  }
  for (int32_t row = 0; k && row < h->rows; ++row)
    for (int32_t c = pages_of(h, h->lengths[row]); c-- > 0;)
      if (row_of(h, row)[c] >= n) put(h, row, c, number[row_of(h, row)[c]]);
  for (int32_t i = 0; i < h->free; ++i) h->stack[i] = h->pages - 1 - i;
  *copies = k;
  return n;
}

// The changed entries that hold another page than the device's: at, value (room for
// n_changed).  They stay among the changed ones until they are sent.
int32_t pages4_changes(const tsattn_pages4_host *h, int32_t *at, int32_t *value) {
  int32_t k = 0;
  for (int32_t i = 0; i < h->n_changed; ++i) {
    const int32_t a = h->changed[i];
    if (h->table[a] < 0 || h->table[a] == h->shown[a]) continue;
    at[k] = a;
    value[k++] = h->table[a];
  }
  return k;
}

// The device's table has what pages4_changes gave: no entry is changed.
void pages4_sent(tsattn_pages4_host *h, int32_t sets, const int32_t *at, const int32_t *value) {
  for (int32_t i = 0; i < h->n_changed; ++i) h->dirty[h->changed[i]] = 0;
  for (int32_t i = 0; i < sets; ++i) h->shown[at[i]] = value[i];
  h->n_changed = 0;
}

}  // namespace tsattn
