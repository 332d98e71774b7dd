// file_pages.h — which bytes of a mapped file the rows of a tensor lie in.  Plain C++, so that the arithmetic can be checked on its own.
#pragma once
#include <stddef.h>

struct AxFileRange { size_t first, last; };       // bytes [first, last) from the start of the mapping

// Rows [r0, r1) of `cols` numbers of `size` bytes AS THEY LIE IN THE FILE (half of what they become where F16 is converted to f32), the
// first row of the tensor at byte `at`.  `first` is rounded down to a page, as madvise wants it; nothing lies behind the file: what follows
// the mapping belongs to somebody else, and madvise would throw its contents away too.
static inline AxFileRange ax_file_rows(size_t at, size_t size, size_t cols, size_t r0, size_t r1, size_t page, size_t file_bytes) {
    AxFileRange r = { at + r0 * cols * size, at + r1 * cols * size };
    if (r.last > file_bytes) r.last = file_bytes;
    r.first -= r.first % page;
    if (r.first > r.last) r.first = r.last;
    return r;
}
