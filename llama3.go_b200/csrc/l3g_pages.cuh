// Copies between pages of a KV cache (included by l3g_ops.cu inside namespace
// l3g).
#pragma once

// Entry i copies rows [0, rows[i]) of page src[i] to page dst[i], 16 bytes a
// thread and step.  grid (x: slices of an entry, y: entries).  Bound by memory:
// every byte is read and written once, four loads of a thread on their way
// together (one at a time: 48 and 128 us).  2048 part-filled pages (269 MB moved)
// in 45 us, 1500 whole ones (786 MB) in 125 us: 5.9 and 6.3 TB/s.  Slices of an
// entry: two 46.6 and 127.5 us, four 45.3 and 125.0, eight 49.2 and 123.1.
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
    const int step = gridDim.x * blockDim.x;
    for (int e = blockIdx.x * blockDim.x + threadIdx.x; e < m; e += 4 * step) {
      int4 v[4];  // on their way together
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (e + u * step < m) v[u] = a[e + u * step];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (e + u * step < m) b[e + u * step] = v[u];
    }
  }
}
