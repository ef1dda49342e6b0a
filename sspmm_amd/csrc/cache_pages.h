// Launch interface of the pages of the cache: taking, sharing, giving back, moving to the front.
#ifndef SSPMM_AMD_CACHE_PAGES_H
#define SSPMM_AMD_CACHE_PAGES_H

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace sspmm {

// refs[pages]: how many table entries name a page; free where it is not positive.  table [rows, slots].
struct PageTable {
  int32_t *refs, *table;
  int pages, rows, slots;
};
// A pool as bytes: of each page block_bytes of keys, as many of values, and scale_floats.
struct PagePool {
  unsigned char *keys, *values;
  float *scales;
  long long block_bytes;  // a multiple of 16
  int scale_floats;
};

size_t reserve_workspace_ints(int pages, int rows, int slots);  // 0: none wanted
size_t fork_workspace_ints(int rows, int count);
size_t compact_workspace_ints(int pages);

hipError_t launch_reserve_pages(const PageTable &t, const int32_t *starts, const int32_t *offsets, int page_size, int32_t *workspace, hipStream_t stream);
hipError_t launch_release_pages(const PageTable &t, int32_t *lengths, const int32_t *named, int count, hipStream_t stream);
hipError_t launch_fork_pages(const PageTable &t, const PagePool &pool, int32_t *lengths, const int32_t *parents, const int32_t *children, int count, int page_size,
                             int32_t *workspace, hipStream_t stream);
hipError_t launch_compact_pages(const PageTable &t, const PagePool &pool, int32_t *workspace, hipStream_t stream);

}  // namespace sspmm
#endif
