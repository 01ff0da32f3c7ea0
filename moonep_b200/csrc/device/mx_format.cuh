// Microscaled 4-bit operands: elements of E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two a byte with the
// earlier one in the low half, and one power of two per block of 32 along the reduction (E8M0: byte b stands for
// 2^(b - 127), 255 for NaN).
//
// Codes: [rows][bytes], a row padded with zeros to whole blocks (16 bytes each).  Scales: atoms of 512 bytes for 128
// rows x 4 blocks, [row atom][block atom][512], in the order in which the tensor cores take them into tensor memory: row
// r, block j at 16 (r % 32) + 4 (r / 32 % 4) + j % 4.  A matrix of token rows has its scales four times, [4][row atom][block
// atom][512]: the atoms of phase s begin at row 32 s, so that those of a tile that starts at any multiple of 32 rows
// begin with an atom.  (Tensor memory wants them so: the MMA takes them from columns that start one.)
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace mep {

constexpr int MX_BLOCK = 32;          // elements that share a scale
constexpr int MX_ATOM_ROWS = 128;
constexpr int MX_ATOM_K = 128;        // elements of a row that an atom of scales covers
constexpr int MX_ATOM_BYTES = 512;
constexpr uint32_t MX_INF = 0x7F800000u;

__host__ __device__ __forceinline__ int mx_atoms(int n) { return (n + 127) / 128; }

constexpr int MX_PHASES = 4;

// Offset of the four scales of row r (within its matrix, or counted from its phase's first) and block atom ka.
__host__ __device__ __forceinline__ long long mx_scale_offset(int r, int ka, int k_atoms) {
  return ((long long)(r >> 7) * k_atoms + ka) * MX_ATOM_BYTES + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}
// Scale byte of a block whose largest magnitude has the fp32 bits `a`: floor(log2 a) - 2, so that the block's largest
// element lands in [4, 8); what rounds to more than 6 becomes 6.  A block with an infinity or a NaN is all NaN.
__device__ __forceinline__ uint32_t mx_scale(uint32_t a) {
  if (a >= MX_INF) return 255u;
  const uint32_t e = a >> 23;
  return e > 2u ? e - 2u : 0u;
}
// 2^(127 - b), by which the block is multiplied (exact; 0 for the NaN scale, so that its codes are zeros)
__device__ __forceinline__ float mx_inverse(uint32_t b) { return b == 255u ? 0.f : __uint_as_float((254u - b) << 23); }
// 2^(b - 127) (b = 0 is a subnormal number)
__device__ __forceinline__ float mx_value(uint32_t b) {
  return __uint_as_float(b == 255u ? 0x7FC00000u : b == 0u ? 0x00400000u : b << 23);
}
// Eight values, already divided by their scale, as codes: nearest, ties to the even code, beyond 6 to 6.
__device__ __forceinline__ uint32_t mx_codes(const float* x) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return r;
}
// The value of a code (its low four bits): sign, then 0 0.5 1 1.5 2 3 4 6.  As an fp32 number the code's exponent and
// mantissa are put where fp32 has its own and rescaled by 2^126; 0.5, subnormal in either format, comes out right.
__device__ __forceinline__ float mx_element(uint32_t code) {
  return __uint_as_float(((code & 8u) << 28) | ((code & 7u) << 22)) * 0x1p126f;
}
// Four codes (the low 16 bits) as bf16, two a word: the magnitudes' bytes are looked up by byte permutations; a product
// moves the two signs of a word to bits 15 and 31.
__device__ __forceinline__ uint2 mx_bf16x4(uint32_t codes) {
  const uint32_t sel = codes & 0x7777u;
  const uint32_t high = __byte_perm(0x3F3F3F00u, 0x40404040u, sel), low = __byte_perm(0xC0800000u, 0xC0804000u, sel);
  uint2 r;
  r.x = __byte_perm(low, high, 0x5140) | ((codes & 0x88u) * 0x01001000u & 0x80008000u);
  r.y = __byte_perm(low, high, 0x7362) | ((codes & 0x8800u) * 0x00010010u & 0x80008000u);
  return r;
}

}  // namespace mep
