// Software versions of the helpers of llama3.go_b200/csrc/l3g_tc16.cuh (same
// names and signatures) on the tensor-memory model of simt_tcgen05.h, for the
// host build of the 16-bit tensor-core kernels: tcgen05.mma kind::f16 with A
// in tensor memory (lane = row, two f16 K elements per 32-bit column) and B in
// shared memory, K-major or MN-major, no swizzle; tensor-memory loads and
// stores; asynchronous copies (done at once); register reallocation (nothing).
// Included inside namespace l3g.  Test infrastructure only.
#pragma once

inline void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                       uint32_t accumulate) {
  ::simt::TensorOp op{};
  op.commit = false;
  op.d_tmem = d_tmem;
  op.adesc = a_tmem;
  op.bdesc = bdesc;
  op.idesc = idesc;
  op.accumulate = accumulate;
  ::simt::queue_tensor_op(op);
}
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
inline void tmem_ld32(uint32_t taddr, uint32_t* v) { memcpy(v, tmem_cell(taddr, 32), 128); }
inline void tmem_ld16(uint32_t taddr, uint32_t* v) { memcpy(v, tmem_cell(taddr, 16), 64); }
inline void tmem_st16(uint32_t taddr, const uint32_t* v) { memcpy(tmem_cell(taddr, 16), v, 64); }
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
