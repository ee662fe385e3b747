// Copies between pages of a KV cache (included by l3g_ops.cu inside namespace
// l3g).
#pragma once

// Entry i copies rows [0, rows[i]) of page src[i] to page dst[i], 16 bytes a
// thread and step.  grid (x: slices of an entry, y: entries).  Bound by memory:
// every byte is read and written once.  2048 part-filled pages (269 MB moved) in
// 48 us, 1500 whole ones (786 MB) in 127 us: 5.6 and 6.2 TB/s.  Slices of an
// entry: one 54 and 139 us, four 48 and 127, eight 50 and 124.
constexpr int COPY_SLICES = 4;
static __global__ void k_copy_pages(const uint8_t* sp, int n_src, uint8_t* dp, int n_dst,
                                    int row_bytes, const int* src, const int* dst,
                                    const int* rows, int n, int* status) {
  for (int i = blockIdx.y; i < n; i += gridDim.y) {
    const int s = src[i], d = dst[i], r = rows ? rows[i] : KV_PAGE;
    if (s < 0 || s >= n_src || d < 0 || d >= n_dst || r < 0 || r > KV_PAGE) {
      if (status && threadIdx.x == 0 && blockIdx.x == 0 && atomicCAS(status, 0, (int)ERR_PAGE) == 0)
        atomicExch(status + 1, i);
      continue;
    }
    const int4* a = reinterpret_cast<const int4*>(sp + (size_t)s * KV_PAGE * row_bytes);
    int4* b = reinterpret_cast<int4*>(dp + (size_t)d * KV_PAGE * row_bytes);
    const int m = r * (row_bytes >> 4);
    for (int e = blockIdx.x * blockDim.x + threadIdx.x; e < m; e += gridDim.x * blockDim.x)
      b[e] = a[e];
  }
}
