// Fifth-generation tensor cores and the copies that feed them, as inline PTX: TMEM allocation,
// loads and stores, tcgen05.mma with both operands in shared memory or the first in TMEM,
// commits to mbarriers, and tiled bulk copies (never multicast). Waits are bounded.
//
// Layouts used throughout (16-bit elements). A tile of R rows and up to 128 columns lies in
// shared memory as one or two blocks of R rows x 128 bytes (64 columns), as a tiled copy with
// the 128-byte swizzle writes them; a block starts on a 1024-byte boundary. Read along its
// columns (K-major, for x y^T) eight rows are 1024 bytes apart and 16 columns are 32 bytes;
// read along its rows (MN-major, for w y, where the rows of y are summed over) 16 rows are 2048
// bytes and the second 64 columns one block apart. An accumulator row is a TMEM lane.
#pragma once

#include <cuda.h>

#include "nt_bulk.cuh"

namespace nt {

// A wait bounded by the SM's cycle counter: the waits between warps are a few hundred cycles, and
// a read of %globaltimer costs as much (wait_stage of nt_bulk.cuh).
constexpr long long kWaitLimitCycles = 4000000000ll;   // about 2 s
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (clock64() - t0 > kWaitLimitCycles) return false;
  }
  return true;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_mbar_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
// ---- clusters --------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float load_cluster(const float* p, uint32_t rank) {
  uint32_t local = static_cast<uint32_t>(__cvta_generic_to_shared(p)), remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote));
  return v;
}

__device__ __forceinline__ float4 load_cluster4(const float* p, uint32_t rank) {
  uint32_t local = static_cast<uint32_t>(__cvta_generic_to_shared(p)), remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote));
  return v;
}
constexpr int kMaxSplits = 8;   // blocks of a portable cluster

// Four columns of a row whose parts lie in `splits` blocks from block `base` of the cluster on:
// unnormalised output at `part`, maximum and sum at `statistic`. Eight blocks' loads are issued before the first is used (one at a time they
// cost a trip to the other SM each). Adds the parts in rank order; a part of weight 0 may not be
// there.
struct JoinedRow {
  float4 o;
  float top, sum;
};
__device__ __forceinline__ JoinedRow join_row(const float* part, const float* statistic, int splits, float scale_log2,
                                             int base = 0) {
  JoinedRow r{make_float4(0.0f, 0.0f, 0.0f, 0.0f), -INFINITY, 0.0f};
  for (int k0 = 0; k0 < splits; k0 += 8) {
    float m[8], l[8];
    float4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      m[k] = -INFINITY;
      l[k] = 0.0f;
      v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (k0 + k < splits) {
        m[k] = load_cluster(statistic, base + k0 + k);
        l[k] = load_cluster(statistic + 1, base + k0 + k);
        v[k] = load_cluster4(part, base + k0 + k);
      }
    }
    float top = r.top;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, m[k]);
    const float old = r.top == -INFINITY ? 0.0f : exp2f((r.top - top) * scale_log2);
    r.top = top;
    r.sum *= old;
    if (old != 0.0f) { r.o.x *= old; r.o.y *= old; r.o.z *= old; r.o.w *= old; }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = m[k] == -INFINITY ? 0.0f : exp2f((m[k] - top) * scale_log2);
      r.sum = fmaf(l[k], f, r.sum);
      if (f != 0.0f) {
        r.o.x = fmaf(v[k].x, f, r.o.x);
        r.o.y = fmaf(v[k].y, f, r.o.y);
        r.o.z = fmaf(v[k].z, f, r.o.z);
        r.o.w = fmaf(v[k].w, f, r.o.w);
      }
    }
  }
  return r;
}

// Programmatic dependent launch: the next kernel's blocks may start from here on; wait for the end of
// the kernel before (no wait where there is no such dependence).
__device__ __forceinline__ void grid_dependents_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// One box of a 4-D tensor map (column, token, head, batch) into shared memory.
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int column, int token, int head, int batch,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(column), "r"(token), "r"(head), "r"(batch), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// ---- TMEM ----------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 or 16 consecutive columns of this thread's lane (warp w reaches lanes 32 (w % 4) ..).
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[32]) { tmem_load32(addr, r); }
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[16]) { tmem_load16(addr, r); }
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// ---- matrix instructions ---------------------------------------------------------------
// Shared-memory operand: start address, leading and stride byte offsets in units of 16 bytes,
// descriptor version 1, 128-byte swizzle.
__device__ __forceinline__ uint64_t tc_descriptor(uint32_t addr, uint32_t leading, uint32_t stride) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(stride >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// A tile of `rows` rows read along its columns, and what 16-column step k adds to its address.
__device__ __forceinline__ uint64_t tc_columns(uint32_t tile) { return tc_descriptor(tile, 16, 1024); }
__device__ __forceinline__ constexpr uint64_t tc_column_step(int rows, int k) {
  return (uint64_t)(((k >> 2) * rows * 128 + (k & 3) * 32) >> 4);
}
// The same read along its rows; 16-row step k.
__device__ __forceinline__ uint64_t tc_rows(uint32_t tile, int rows) { return tc_descriptor(tile, rows * 128, 1024); }
__device__ __forceinline__ constexpr uint64_t tc_row_step(int k) { return (uint64_t)(k * 2048 >> 4); }

// True in one lane of the (whole, converged) warp. The compiler takes code under it as one
// thread's, so the operands of the matrix instructions stay in uniform registers: under an
// ordinary lane test each instruction took about 100 cycles to issue.
__device__ __forceinline__ bool elect_one() {
  uint32_t chosen;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(chosen));
  return chosen != 0;
}

// float32 accumulator of 128 rows and n columns (a multiple of 16); a and b are both float16 or
// both bfloat16; b_rows: the second operand is read along its rows.
template <int DT>
__device__ __forceinline__ uint32_t tc_instruction(int n, bool b_rows) {
  constexpr uint32_t type = DT == NT_BF16 ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(instruction), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void tc_mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t instruction, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(instruction), "r"((uint32_t)add)
      : "memory");
}
// Arrives on `bar` once every matrix instruction this thread has issued is complete.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// Two float32 values as one register of two 16-bit ones (round to nearest even).
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (DT == NT_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <int DT>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (DT == NT_BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two float32 operations in one instruction.
struct Pair {
  uint64_t bits;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ void get(float& lo, float& hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(bits)); }
};
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}

// 2^x of two values on the FP32 pipe: x = n + f with n the nearest integer, 2^f for |f| <= 1/2 by the
// polynomial of degree 4 with the least largest relative error (2.7e-6, far below a 16-bit
// weight's own rounding), scaled by 2^n. From 2^-126, which stands for everything below, to 2^126,
// which does for everything above; NaN stays NaN.
__device__ __forceinline__ void ex2_polynomial(float& x, float& y) {
  const Pair v(min_nan(max_nan(x, -126.0f), 126.0f), min_nan(max_nan(y, -126.0f), 126.0f));
  const Pair t = add2(v, Pair(12582912.0f, 12582912.0f));   // 1.5 * 2^23: the integer ends up in the low bits
  const Pair f = add2(v, fma2(t, Pair(-1.0f, -1.0f), Pair(12582912.0f, 12582912.0f)));
  Pair p = fma2(f, Pair(0.009570100344717503f, 0.009570100344717503f), Pair(0.05591785907745361f, 0.05591785907745361f));
  p = fma2(p, f, Pair(0.240247443318367f, 0.240247443318367f));
  p = fma2(p, f, Pair(0.6931217908859253f, 0.6931217908859253f));
  p = fma2(p, f, Pair(0.9999992847442627f, 0.9999992847442627f));
  float a, b;
  t.get(a, b);
  mul2(p, Pair(__int_as_float((__float_as_int(a) << 23) + 0x3f800000), __int_as_float((__float_as_int(b) << 23) + 0x3f800000)))
      .get(x, y);
}
// Exponentials of two neighbouring columns: the special-function unit gives 16 a cycle and SM, fewer
// than the tensor cores can use, so every fourth pair goes to the FP32 pipe.
template <int PAIR>
__device__ __forceinline__ void ex2_mixed(float& x, float& y) {
  if constexpr (PAIR % 4 == 3) {
    ex2_polynomial(x, y);
  } else {
    x = ex2_approx(x);
    y = ex2_approx(y);
  }
}
// True in every thread of the barrier when `any` was in one.
__device__ __forceinline__ bool named_barrier_or(int id, int threads, bool any) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, %2, %3, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"((uint32_t)any), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}

// 32 rows of a warp, CH 16-byte vectors each, lane r holding row r, written to global memory with
// whole row segments per instruction (a lane storing its own row would touch 32 lines at a time;
// that took longer than the products of a short window). `stage`: CH * 512 bytes of this warp's.
// Rows from `rows` on and vectors from `vectors` on are not stored.
template <int CH>
__device__ __forceinline__ void stage_vector(uint8_t* stage, int lane, int k, uint4 v) {
  *reinterpret_cast<uint4*>(stage + (lane * CH + (k ^ (lane / (8 / CH) % CH))) * 16) = v;
}
template <int CH>
__device__ __forceinline__ void store_staged(const uint8_t* stage, int lane, char* dst, int64_t row_bytes, int rows, int vectors) {
  __syncwarp();
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 32 / CH) {
    const int r = r0 + lane / CH, k = lane % CH;
    if (r < rows && k < vectors)
      *reinterpret_cast<uint4*>(dst + r * row_bytes + k * 16) =
          *reinterpret_cast<const uint4*>(stage + (r * CH + (k ^ (r / (8 / CH) % CH))) * 16);
  }
  __syncwarp();
}

}  // namespace nt
