// Software versions of the helpers of llama3.go_b200/csrc/l3g_tc16.cuh (same
// names and signatures) on the tensor-memory model of simt_tcgen05.h, for the
// host build of the 16-bit tensor-core kernels: tcgen05.mma kind::f16 with A
// in tensor memory (lane = row, two f16 K elements per 32-bit column) and B in
// shared memory, K-major or MN-major, 128- or 64-byte swizzle; tensor-memory loads and
// stores; asynchronous copies (done at once); register reallocation (nothing).
// Included inside namespace l3g.  Test infrastructure only.
#pragma once

template <bool ACC>
inline void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi,
                       uint32_t idesc) {
  ::simt::TensorOp op{};
  op.commit = false;
  op.d_tmem = d_tmem;
  op.adesc = a_tmem;
  op.bdesc = (uint64_t)b_hi << 32 | b_lo;
  op.idesc = idesc;
  op.accumulate = ACC;
  ::simt::queue_tensor_op(op);
}
inline bool mbar_try_wait(uint64_t* b, uint32_t parity, uint32_t) { return mbar_test(b, parity); }
inline void prefetch_l2(const void* p) {
  if (!::simt::in_global(p, 4)) ::simt::fail("prefetch outside every buffer");
}
inline bool elect_one() { return ::simt::cur()->lane == 0; }
inline uint32_t* tmem_cell(uint32_t taddr, int cols) {
  ::simt::Thread* t = ::simt::cur();
  __syncwarp();
  const uint32_t lane0 = taddr >> 16, col = taddr & 0xFFFFu;
  if (lane0 != 32u * (uint32_t)(t->warp % 4))
    ::simt::fail("tcgen05.ld/st: a warp may only address its own quarter of the lanes");
  if (col + cols > 512) ::simt::fail("tcgen05.ld/st past the last column");
  for (uint32_t u = col / 32; u <= (col + cols - 1) / 32; ++u)
    if (!(t->blk->tmem_used >> u & 1u)) ::simt::fail("tcgen05.ld/st of unallocated tensor memory");
  return &t->blk->tmem[(size_t)(lane0 + t->lane) * 512 + col];
}
inline void tmem_get32(uint32_t taddr, uint32_t* v) { memcpy(v, tmem_cell(taddr, 32), 128); }
inline void tmem_get16(uint32_t taddr, uint32_t* v) { memcpy(v, tmem_cell(taddr, 16), 64); }
inline void tmem_st16(uint32_t taddr, const uint32_t* v) { memcpy(tmem_cell(taddr, 16), v, 64); }
inline void tmem_st8(uint32_t taddr, const uint32_t* v) { memcpy(tmem_cell(taddr, 8), v, 32); }
inline void tmem_st4(uint32_t taddr, const uint32_t* v) { memcpy(tmem_cell(taddr, 4), v, 16); }
inline void tmem_wait_st() {}
inline void cp_async16(void* dst, const void* src, uint32_t bytes) {
  if (!::simt::in_smem(::simt::cur()->blk, dst, 16) || ((uintptr_t)dst & 15) ||
      ((uintptr_t)src & 15))
    ::simt::fail("cp.async: destination outside shared memory or unaligned");
  if (bytes && !::simt::in_global(src, bytes)) ::simt::fail("cp.async: source outside every buffer");
  memset(dst, 0, 16);
  if (bytes) memcpy(dst, src, bytes);
}
inline void cp_async_commit() {}
template <int N>
inline void cp_async_wait() {}
inline void fence_proxy_async_shared() {}
template <int N>
inline void regs_inc() {}
template <int N>
inline void regs_dec() {}
inline float ex2(float x) { return std::exp2(x); }

// Tensor maps are stood in for by the geometry itself, in the map's bytes
struct EmuMap {
  const uint8_t* base;
  int row_bytes, box_bytes, box_rows;  // bytes of a tensor row and of a box's row; rows of a box
  int es;
};
inline void tmap_rebase(void* map, void* stage, const CUtensorMap* tmpl, const void* base, int lane) {
  __syncwarp();
  EmuMap m;
  memcpy(&m, tmpl, sizeof m);
  m.base = static_cast<const uint8_t*>(base);
  if (lane == 0) memcpy(stage, &m, sizeof m);
  if (lane == 0) memcpy(map, &m, sizeof m);
  __syncwarp();
}
inline void tma_load_2d(void* dst, const void* map, int x, int y, uint64_t* bar) {
  EmuMap m;
  memcpy(&m, map, sizeof m);
  if ((x * m.es) % 16) ::simt::fail("tensor copy starts off a 16-byte boundary");
  const uint32_t at = smem_u32(dst);
  if (at % (8 * m.box_bytes)) ::simt::fail("tensor copy destination off its swizzle pattern");
  // swizzled as the hardware does: by address bits above the 16-byte piece
  ::simt::Runtime& r = ::simt::rt();
  ::simt::mbar(bar, "cp.async.bulk.tensor");
  ::simt::Copy c;
  c.dst = static_cast<uint8_t*>(dst);
  c.data.resize((size_t)m.box_rows * m.box_bytes);
  const uint32_t mask = m.box_bytes == 128 ? 7 : 3;
  for (int k = 0; k < m.box_rows; ++k) {
    const uint8_t* src = m.base + (size_t)(y + k) * m.row_bytes + (size_t)x * m.es;
    if (!::simt::in_global(src, m.box_bytes)) ::simt::fail("tensor copy reads outside every buffer");
    for (int b = 0; b < m.box_bytes; ++b) {
      const uint32_t lin = (uint32_t)(k * m.box_bytes + b);
      c.data[lin ^ (((lin >> 7) & mask) << 4)] = src[b];
    }
  }
  c.bar = bar;
  c.blk = ::simt::cur()->blk;
  const int d = r.randomize ? (int)(r.rng() % (uint64_t)(r.max_copy_delay + 1)) : 1;
  c.due = r.clock + 1 + (uint64_t)d * (r.threads.size() / 8 + 1);
  r.copies.push_back(std::move(c));
}
