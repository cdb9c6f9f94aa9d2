// What the bf16 matrix kernels of the training operators share: copies from
// memory straight into LDS, and the operands of v_mfma_f32_32x32x16_bf16 read
// from there, as they lie or transposed.
//
// The instruction computes C[m][n] += sum over 16 k of A[m][k] B[k][n].  Lane l
// gives eight consecutive k, 8 (l / 32) ..., of row m = l % 32 of A and of column
// n = l % 32 of B, and holds of C the column n = l % 32 and the rows
// 8 (r / 4) + 4 (l / 32) + r % 4, r < 16.
#pragma once

#include "common.h"

namespace tcfp {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* lds_v4s;
typedef __attribute__((address_space(3))) uint8_t* lds_bytes;

constexpr uint32_t kOutOfRange = 0x80000000u;  // beyond every descriptor
// Largest byte span of a descriptor (offsets are 32-bit and kOutOfRange stays
// beyond it).
constexpr int64_t kMaxSpan = (int64_t(1) << 31) - (int64_t(1) << 20);

// A buffer descriptor of `bytes` bytes: loads past them give zeros.
TCFP_DEV v4i make_rsrc(const void* base, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  v4i r;
  r[0] = int(uint32_t(a));
  r[1] = int(uint32_t(a >> 32) & 0xFFFFu);
  r[2] = int(bytes);
  r[3] = 0x00020000;
  return r;
}

// 64 lanes x 16 bytes from the descriptor's offset of each lane into LDS at
// lds + 16 * lane (lds the wave's); done when vmcnt has counted it.  From inline
// assembly, as the compiler would otherwise wait for every such copy before any
// LDS read; the wait state between the write of m0 and the copy, which the
// compiler adds for instructions of its own only, is in the text.
TCFP_DEV void copy16(v4i rsrc, uint32_t off, uint32_t lds) {
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :
               : "v"(off), "s"(rsrc), "{m0}"(lds)
               : "memory");
}

// The same, 4 bytes a lane: into LDS at lds + 4 * lane.  (Its descriptor may come out
// of vector registers, which takes five wait states.)
TCFP_DEV void copy4(v4i rsrc, uint32_t off, uint32_t lds) {
#pragma unroll
  for (int i = 0; i < 4; ++i) rsrc[i] = __builtin_amdgcn_readfirstlane(rsrc[i]);
  asm volatile("s_nop 4\n\tbuffer_load_dword %0, %1, 0 offen lds"
               :
               : "v"(off), "s"(rsrc), "{m0}"(lds)
               : "memory");
}

// Hides a value's origin from the compiler, which would otherwise keep all that is
// derived from it in registers through a loop, where none are free.
TCFP_DEV int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Waits until at most N of the wave's vector memory operations are in flight and
// its LDS reads are done, then for the workgroup.
template <int N>
TCFP_DEV void wait_and_sync() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

TCFP_DEV uint32_t lds_offset(const void* p) {
  return uint32_t(reinterpret_cast<uintptr_t>((lds_bytes)(p)));
}

TCFP_DEV v8bf read16(const uint8_t* p) { return *reinterpret_cast<const v8bf*>(p); }

// Two transposing reads: lane l of a group of 16 gets column l % 16 of the
// 4 x 16 block whose rows the group's lanes point at (lane i at row i / 4,
// columns 4 (i % 4) ...).
TCFP_DEV v8bf read_transposed(const uint8_t* lo, const uint8_t* hi) {
  const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(lo));
  const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(hi));
  return __builtin_bit_cast(v8bf, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

TCFP_DEV v16f mfma(const v8bf& a, const v8bf& b, const v16f& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

TCFP_DEV uint32_t pack2(float a, float b) {
  const v2bf v = {(__bf16)a, (__bf16)b};  // round to nearest even
  return __builtin_bit_cast(uint32_t, v);
}

TCFP_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
TCFP_DEV float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

}  // namespace tcfp
