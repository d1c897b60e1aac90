// TMA tile loads and the 5th-generation tensor core's instructions (tcgen05.*), one PTX
// instruction each, with the descriptors of the operand layouts the kernels use.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace wc {

// Shared-memory matrix descriptor of a K-major tile written by TMA with the 128-byte
// swizzle: rows of 128 bytes, 8-row groups 1024 bytes apart (stride byte offset), leading
// byte offset unused (1), descriptor version 1, layout type 2 (SWIZZLE_128B). The start
// address of the k-th 16-element slice of a row is the tile base + 32 k bytes.
__device__ __forceinline__ uint64_t umma_desc_sw128(uint32_t saddr) {
  return uint64_t((saddr & 0x3FFFFu) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
          smem_addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, int v,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
      "[%7];\n" ::"r"(smem_addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void umma_bf16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrives on `bar` once every tcgen05.mma this thread issued before has completed
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_addr(bar))
               : "memory");
}
// 16 consecutive fp32 columns of this thread's TMEM lane (32x32b shape, x16)
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// The MN-major operand of a TMA tile with the 128-byte swizzle has rows of 128 bytes as K indices (8-row
// groups 1024 bytes apart = stride byte offset) and 64-element MN blocks `leading` * 16 bytes apart.
// Instruction descriptor, kind::f16: fp32 accumulator, bf16 A and B, M 128; B K-major or MN-major.
__host__ __device__ constexpr uint32_t umma_idesc_bf16_m128(int N, int b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(b_mn_major) << 16) | (uint32_t(N >> 3) << 17) |
         (uint32_t(128 >> 4) << 24);
}
// A shared-memory descriptor as its address field (low word) and its constant high word: the address
// of a later slice of the same tile is a 32-bit addition away.
__device__ __forceinline__ uint32_t umma_lo(uint32_t saddr, uint32_t leading) {
  return ((saddr & 0x3FFFFu) >> 4) | (leading << 16);
}
constexpr uint32_t kUmmaHiSw128 = (1024u >> 4) | (1u << 14) | (2u << 29);  // stride 1024 bytes, version 1, 128B swizzle
// kind::f16 products of one thread, operands given by their descriptors' words
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t alo, uint32_t blo, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}\n" ::"r"(d),
      "r"(alo), "r"(blo), "r"(idesc), "r"(uint32_t(acc)), "r"(kUmmaHiSw128)
      : "memory");
}
// the same with A in tensor memory: lane = row, one 32-bit column = two consecutive bf16 K elements
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t blo, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.b32 p, %4, 0;\n mov.b64 b, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(blo), "r"(idesc), "r"(uint32_t(acc)), "r"(kUmmaHiSw128)
      : "memory");
}
// one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
#define WC_R8(a, i) "=r"((a)[i]), "=r"((a)[i + 1]), "=r"((a)[i + 2]), "=r"((a)[i + 3]), "=r"((a)[i + 4]), \
                    "=r"((a)[i + 5]), "=r"((a)[i + 6]), "=r"((a)[i + 7])
#define WC_I8(a, i) "r"((a)[i]), "r"((a)[i + 1]), "r"((a)[i + 2]), "r"((a)[i + 3]), "r"((a)[i + 4]), \
                    "r"((a)[i + 5]), "r"((a)[i + 6]), "r"((a)[i + 7])
// 32 consecutive columns of this thread's lane, complete on return
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : WC_R8(r, 0), WC_R8(r, 8), WC_R8(r, 16), WC_R8(r, 24)
      : "r"(taddr)
      : "memory");
}
// stores 32 consecutive columns; tmem_st_wait() completes them
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};\n" ::WC_I8(r, 0),
      WC_I8(r, 8), WC_I8(r, 16), WC_I8(r, 24), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::WC_I8(
          r, 0),
      WC_I8(r, 8), "r"(taddr)
      : "memory");
}
#undef WC_R8
#undef WC_I8
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
// generic-proxy shared-memory writes before this are visible to the tensor core and copy engine after it
__device__ __forceinline__ void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

}  // namespace wc
