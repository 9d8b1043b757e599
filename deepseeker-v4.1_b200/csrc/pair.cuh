// Pieces of the kernels that run on CTA pairs (tcgen05 cta_group::2): signals
// between the two CTAs, pair-wide commits, accumulator reads and result boxes.
//
// A pair is a cluster of two CTAs.  The leader (rank 0) issues the MMAs; both
// stage their halves of the operands in their own shared memory and count the
// bytes on the leader's barrier; a commit signals the same barrier of both.
#pragma once

#include <cuda.h>

#include "ptx.cuh"
#include "tc5.cuh"

namespace ds {
namespace pair {

using namespace ds::ptx;

constexpr int kBox = 4096;   // 32 lines of 128 bytes

// Allocation and release of tensor memory, by one warp of both CTAs.
__device__ __forceinline__ void alloc512(uint32_t* dst) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(dst)) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc512(uint32_t base) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(base) : "memory");
}

constexpr uint64_t kWaitNs = 2000000000ull;   // 2 s
constexpr int kErrTimeout = 2;

// Bounded wait for a phase.  The thread sleeps in try_wait and wakes as the
// phase completes; the clock and the abort flag are looked at only when that
// has run out once.  Gives up after kWaitNs or when another role has.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* err) {
  if (mbar_try_wait_sleep(bar, parity, 20000u)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait_sleep(bar, parity, 20000u)) {
    if (*abort) return false;
    if (globaltimer_ns() - t0 > kWaitNs) {
      *abort = 1;
      atomicOr(err, kErrTimeout);
      return false;
    }
  }
  return true;
}

// The same by a whole warp, with one verdict.
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, volatile int* abort, int* err) {
  return __all_sync(0xffffffffu, wait(bar, parity, abort, err));
}

// This address in the leader's shared memory.
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}

// A CTA's rows of an operand, their bytes counted on the leader's barrier.
__device__ __forceinline__ void load_box(uint8_t* dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}

// Arrives on this barrier of both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

__device__ __forceinline__ void arrive_leader(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

__device__ __forceinline__ void ld_x32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// A box of 32 lines of 128 bytes in shared memory, 16-byte pieces swizzled:
// lane = line, piece c of it.
__device__ __forceinline__ uint4* box_at(uint8_t* box, int lane, int c) {
  return reinterpret_cast<uint4*>(box + lane * 128 + ((c ^ (lane & 7)) << 4));
}

__device__ __forceinline__ void box_put(uint8_t* box, int lane, const float (&v)[32]) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *box_at(box, lane, c) = make_uint4(__float_as_uint(v[4 * c]), __float_as_uint(v[4 * c + 1]),
                                       __float_as_uint(v[4 * c + 2]), __float_as_uint(v[4 * c + 3]));
}

__device__ __forceinline__ void box_get(uint8_t* box, int lane, float (&v)[32]) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint4 w = *box_at(box, lane, c);
    v[4 * c] = __uint_as_float(w.x), v[4 * c + 1] = __uint_as_float(w.y);
    v[4 * c + 2] = __uint_as_float(w.z), v[4 * c + 3] = __uint_as_float(w.w);
  }
}

// 32 f32 columns of 32 rows (lane = row) handed out row by row, lane = column:
// single stores of any width then fall on neighbouring addresses.  A thread's
// own stores along its row made a result whose rows do not start on 16 bytes
// six times slower.  The box must not be in use.
template <typename Store>
__device__ __forceinline__ void by_rows(uint8_t* box, int lane, const float (&v)[32], Store store) {
  __syncwarp();
  box_put(box, lane, v);
  __syncwarp();
#pragma unroll 8
  for (int r = 0; r < 32; ++r)
    store(r, *reinterpret_cast<const float*>(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4));
}

// One thread: the box goes to columns x.., rows y.. (clipped to the matrix).
__device__ __forceinline__ void box_store(const CUtensorMap* map, int x, int y, const uint8_t* box) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x),
               "r"(y), "r"(smem_u32(box))
               : "memory");
}
__device__ __forceinline__ void box_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// This thread's stores but the last N have read their boxes.
template <int N>
__device__ __forceinline__ void box_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void box_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

}  // namespace pair
}  // namespace ds
