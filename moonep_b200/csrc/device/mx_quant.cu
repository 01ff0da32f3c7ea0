// Quantisation into microscaled 4-bit operands (mx_format.cuh) and back.  Both directions are bandwidth kernels: one
// pass, every element read and written once.  They are launched as programmatic dependents, as the product behind them
// is: a chain's kernels are in place when their predecessor ends (rows quantised and multiplied, 16 tokens: 49.7 -> 46.1 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "device/mx_format.cuh"
#include "device/sync.cuh"
#include "host/ctx.h"
#include "host/errors.h"

namespace mep {

enum { MX_BF16 = 0, MX_FP16 = 1, MX_FP32 = 2 };

__device__ __forceinline__ uint32_t mx_abs(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// Two neighbouring elements as they are stored: largest magnitudes of either side, and products with a power of two per
// side, in as few instructions as their type allows (magnitudes of 16 bits compare like integers, two at once; a bf16
// times a power of two is a bf16, exactly).
template <class T> struct __align__(2 * sizeof(T)) MxPair { T e[2]; };
template <class T> struct MxMax;         // largest magnitudes so far of the left and the right elements
template <> struct MxMax<float> {
  uint32_t a = 0u, b = 0u;
  __device__ __forceinline__ void add(const MxPair<float>& x) { a = max(a, mx_abs(x.e[0])); b = max(b, mx_abs(x.e[1])); }
  __device__ __forceinline__ uint32_t left() const { return a; }
  __device__ __forceinline__ uint32_t right() const { return b; }
};
template <class T> struct MxMax16 {
  uint32_t m = 0u;
  __device__ __forceinline__ void add(const MxPair<T>& x) { m = __vmaxu2(m, *reinterpret_cast<const uint32_t*>(&x) & 0x7FFF7FFFu); }
};
template <> struct MxMax<__nv_bfloat16> : MxMax16<__nv_bfloat16> {
  __device__ __forceinline__ uint32_t left() const { return m << 16; }
  __device__ __forceinline__ uint32_t right() const { return m & 0xFFFF0000u; }
};
template <> struct MxMax<__half> : MxMax16<__half> {
  __device__ __forceinline__ uint32_t left() const { return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m))); }
  __device__ __forceinline__ uint32_t right() const { return __float_as_uint(__half2float(__ushort_as_half((unsigned short)(m >> 16)))); }
};
__device__ __forceinline__ float2 mx_times(const MxPair<float>& x, float s, float t) { return make_float2(x.e[0] * s, x.e[1] * t); }
__device__ __forceinline__ float2 mx_times(const MxPair<__half>& x, float s, float t) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
  return make_float2(f.x * s, f.y * t);
}
__device__ __forceinline__ float2 mx_times(const MxPair<__nv_bfloat16>& x, float s, float t) {
  const __nv_bfloat162 k = __floats2bfloat162_rn(s, t), y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x), k);
  return __bfloat1622float2(y);
}

// Row of a packed pair of a gate (up = 0) and an up projection: sixteen of either in turn.
__device__ __forceinline__ int mx_pair_row(int r, int up) { return (r >> 4) * 32 + (r & 15) + 16 * up; }

struct MxQuantParams {
  const void* x;
  const void* x2;               // the up projection of a pair (x: gate), along the columns; or null
  long long batch, stride;      // elements between matrices, and between rows of x
  int mats, rows, cols;         // of x
  int out_rows;                 // rows of a matrix of the output (codes)
  int code_bytes, k_atoms, row_atoms;
  uint8_t* codes;
  uint8_t* scales;
  const int32_t* rows_ptr;      // rows of x that hold something, on the device; or null
  int phases;                   // 4: token rows, whose scales are stored at four phases
};

// Where the first four scales of row r are in phase s, the next ones 512 bytes further each; null where there is no such copy.
__device__ __forceinline__ uint32_t* mx_scale_row(const MxQuantParams& p, int mat, int r, int s) {
  if (s >= p.phases || r < 32 * s) return nullptr;
  const long long copy = p.phases == 1 ? mat : s;
  return reinterpret_cast<uint32_t*>(p.scales + copy * p.row_atoms * p.k_atoms * MX_ATOM_BYTES + mx_scale_offset(r - 32 * s, 0, p.k_atoms));
}

// Raw elements are loaded first, all of a thread's, and converted when they are there: a load beside its use in one guarded
// block made a chain of load latencies (the kernel along the columns: 925 us for 32 x 7168 x 2048 in bf16, 4.2x).
template <class T> struct __align__(16) MxEight { MxPair<T> p[4]; };

// Eight elements of a row from column c on, as they were loaded; behind the row's end zeros.
template <class T, bool VEC>
struct MxRaw {                            // rows of 16-byte pieces (cols is a multiple of 8)
  MxEight<T> v;
  __device__ __forceinline__ void load(const T* row, int c, int cols) {
    uint4* q = reinterpret_cast<uint4*>(&v);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      q[i] = c < cols ? __ldcs(reinterpret_cast<const uint4*>(row + c) + i) : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ const MxEight<T>& get() const { return v; }
};
template <class T>
struct MxRaw<T, false> {                  // rows that start anywhere: the aligned pieces they lie in, moved when they are used
  static constexpr int PIECES = sizeof(T) / 2 + 1, WORDS = 2 * sizeof(T);
  uint32_t w[4 * PIECES];
  int off;                                // bytes of the first piece in front of them
  __device__ __forceinline__ void load(const T* row, int c, int cols) {
    const uintptr_t at = (uintptr_t)(row + c), first = at & ~(uintptr_t)15;
    const int pieces = at == first ? PIECES - 1 : PIECES;
    off = (int)(at - first);
    if (first >= (uintptr_t)row && first + 16 * pieces <= (uintptr_t)(row + cols)) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const uint4 q = i < pieces ? reinterpret_cast<const uint4*>(first)[i] : make_uint4(0, 0, 0, 0);
        w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
      }
    } else {                              // (nothing outside the row is read)
      MxEight<T> v;
#pragma unroll
      for (int i = 0; i < 8; ++i) v.p[i / 2].e[i % 2] = c + i < cols ? row[c + i] : T(0.f);
#pragma unroll
      for (int i = 0; i < 4 * PIECES; ++i) w[i] = i < WORDS ? reinterpret_cast<const uint32_t*>(&v)[i] : 0u;
      off = 0;
    }
  }
  __device__ __forceinline__ MxEight<T> get() const {
    MxEight<T> v;
    uint32_t u[WORDS + 2];
#pragma unroll
    for (int i = 0; i < WORDS + 2; ++i) u[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < WORDS + 1; ++i) u[i] = off & 4 ? u[i + 1] : u[i];
#pragma unroll
    for (int i = 0; i < WORDS; ++i)
      reinterpret_cast<uint32_t*>(&v)[i] = sizeof(T) == 2 ? __funnelshift_r(u[i], u[i + 1], 8 * (off & 2)) : u[i];
    return v;
  }
};

// Along the rows.  A warp takes MXQ_DEPTH parts of 256 elements of a row, a lane eight of each: four lanes share a
// block and store its scale, a phase each.  Bound by HBM: 8192 x 7168 in bf16 30 us, 5.0 TB/s with the launch, fp32 42 us,
// 6.3.  (Sixteen elements a lane are fewer instructions, but two 16-byte accesses of a lane side by side: 14336 x 7168
// 51.6 us, 53.7; 32 x 7168 x 2048 215, 201.)  Rows of odd lengths: 8192 x 7001 in fp32 54 us, 4.8 TB/s (by elements 68), 7167 in
// bf16 45 (48).
constexpr int MXQ_WARPS = 8, MXQ_DEPTH = 4;

template <class T, bool VEC>
__global__ void __launch_bounds__(MXQ_WARPS * 32) ep_mx_quant_rows_kernel(const __grid_constant__ MxQuantParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = p.rows_ptr ? max(0, min(*p.rows_ptr, p.rows)) : p.rows;
  const unsigned lines = (unsigned)p.mats * (unsigned)rows;
  for (unsigned line = blockIdx.x * MXQ_WARPS + warp; line < lines; line += gridDim.x * MXQ_WARPS) {
    const int mat = p.mats > 1 ? (int)(line / (unsigned)rows) : 0, row = (int)(line - (unsigned)mat * (unsigned)rows);
    const T* x = (const T*)p.x + mat * p.batch + row * p.stride;
    uint8_t* codes = p.codes + ((long long)mat * p.out_rows + row) * p.code_bytes;
    uint8_t* scales = reinterpret_cast<uint8_t*>(mx_scale_row(p, mat, row, lane & 3));    // of this lane's phase, if it has one
    for (int c0 = blockIdx.y * 256 * MXQ_DEPTH; c0 < p.cols; c0 += gridDim.y * 256 * MXQ_DEPTH) {
      MxRaw<T, VEC> raw[MXQ_DEPTH];
#pragma unroll
      for (int i = 0; i < MXQ_DEPTH; ++i) raw[i].load(x, c0 + i * 256 + lane * 8, p.cols);
#pragma unroll
      for (int i = 0; i < MXQ_DEPTH; ++i) {
        if (c0 + i * 256 >= p.cols) break;          // (the same for the whole warp)
        const int c = c0 + i * 256 + lane * 8;
        const MxEight<T> u = raw[i].get();
        MxMax<T> m;
#pragma unroll
        for (int e = 0; e < 4; ++e) m.add(u.p[e]);
        uint32_t a = max(m.left(), m.right());
        a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));
        a = max(a, __shfl_xor_sync(0xffffffffu, a, 2));
        const uint32_t b = mx_scale(a);
        const float inv = mx_inverse(b);
        float v[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) *reinterpret_cast<float2*>(v + 2 * e) = mx_times(u.p[e], inv, inv);
        // (a NaN scale: zeros, whatever inf * 0 would give)
        const uint32_t q = b == 255u ? 0u : mx_codes(v);
        if (c < 2 * p.code_bytes) *reinterpret_cast<uint32_t*>(codes + c / 2) = q;
        if (scales != nullptr && c < p.k_atoms * MX_ATOM_K) scales[(c >> 7) * (long long)MX_ATOM_BYTES + (c >> 5 & 3)] = (uint8_t)b;
      }
    }
  }
}

// Along the columns: the output is the transpose.  A block takes 256 rows of x, a warp one block of 32 rows, a lane four
// columns of it (two of fp32): 256-byte pieces of x's rows.  (With 128-byte pieces of bf16 rows 3.8 TB/s; 32 x 7168 x 2048
// 314 us.)  The codes of a column meet in shared memory and leave as 128-byte rows.
constexpr int MXT_ROWS = 256;
template <class T> constexpr int mxt_pairs() { return sizeof(T) == 2 ? 2 : 1; }

template <class T, bool VEC>
__global__ void __launch_bounds__(256, 2) ep_mx_quant_cols_kernel(const __grid_constant__ MxQuantParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int NP = mxt_pairs<T>(), COLS = 64 * NP;
  struct __align__(8) Piece { MxPair<T> p[NP]; };
  __shared__ __align__(16) uint8_t s_codes[COLS * 128];
  __shared__ __align__(4) uint8_t s_scale[COLS][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r0 = blockIdx.y * MXT_ROWS, c0 = blockIdx.x * COLS;
  // (a pair's last turn of sixteen is stored whole: zeros behind the last column)
  const bool pair = p.x2 != nullptr;
  const int cols = pair ? (p.cols + 15) & ~15 : p.cols;
  for (int z = blockIdx.z; z < (pair ? 2 : 1) * p.mats; z += gridDim.z) {
    const int up = z >= p.mats ? 1 : 0, m = z - up * p.mats;
    const int c = c0 + 2 * NP * lane, rw = r0 + warp * MX_BLOCK;
    const T* x = (const T*)(up ? p.x2 : p.x) + m * p.batch + (long long)rw * p.stride + c;
    auto out_row = [&](int n) { return pair ? mx_pair_row(c0 + n, up) : c0 + n; };
    Piece raw[MX_BLOCK];
#pragma unroll
    for (int i = 0; i < MX_BLOCK; ++i) {
      const T* e = x + i * p.stride;
      if constexpr (VEC) {             // (the number of columns is a multiple of a lane's)
        const uint2 q = rw + i < p.rows && c < p.cols ? __ldcs(reinterpret_cast<const uint2*>(e)) : make_uint2(0, 0);
        raw[i] = *reinterpret_cast<const Piece*>(&q);
      } else {
#pragma unroll
        for (int j = 0; j < 2 * NP; ++j) raw[i].p[j / 2].e[j % 2] = rw + i < p.rows && c + j < p.cols ? e[j] : T(0.f);
      }
    }
#pragma unroll
    for (int h = 0; h < NP; ++h) {
      MxMax<T> top;
#pragma unroll
      for (int i = 0; i < MX_BLOCK; ++i) top.add(raw[i].p[h]);
      const uint32_t b0 = mx_scale(top.left()), b1 = mx_scale(top.right());
      const float inv0 = mx_inverse(b0), inv1 = mx_inverse(b1);
      uint32_t q[2][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float u[8], v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 f = mx_times(raw[8 * j + i].p[h], inv0, inv1);
          u[i] = f.x; v[i] = f.y;
        }
        q[0][j] = b0 == 255u ? 0u : mx_codes(u);
        q[1][j] = b1 == 255u ? 0u : mx_codes(v);
      }
      // (16-byte pieces of a row in an order by column: neighbouring lanes' fall into different banks)
      const int n = 2 * NP * lane + 2 * h;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<uint4*>(s_codes + (n + i) * 128 + (warp ^ (lane & 7)) * 16) = make_uint4(q[i][0], q[i][1], q[i][2], q[i][3]);
      s_scale[n][warp] = (uint8_t)b0;
      s_scale[n + 1][warp] = (uint8_t)b1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < COLS * 8; i += 256) {       // 16 bytes of a column's codes
      const int n = i >> 3, k = r0 / 2 + (i & 7) * 16;
      if (c0 + n < cols && k < p.code_bytes)
        *reinterpret_cast<uint4*>(p.codes + ((long long)m * p.out_rows + out_row(n)) * p.code_bytes + k) =
            *reinterpret_cast<const uint4*>(s_codes + n * 128 + ((i & 7) ^ (n / (2 * NP) & 7)) * 16);
    }
    for (int i = threadIdx.x; i < 2 * COLS * p.phases; i += 256) {
      const int n = (i >> 1) % COLS, ka = r0 / MX_ATOM_K + (i & 1);
      uint32_t* scales = c0 + n < cols && ka < p.k_atoms ? mx_scale_row(p, m, out_row(n), i / (2 * COLS)) : nullptr;
      if (scales != nullptr) scales[(long long)ka * (MX_ATOM_BYTES / 4)] = *reinterpret_cast<const uint32_t*>(&s_scale[n][4 * (i & 1)]);
    }
    __syncthreads();
  }
}

struct MxDequantParams {
  const uint8_t* codes;
  const uint8_t* scales;
  int mats, rows, cols;         // of the values; `rows` of gate or up where they are a packed pair, which has both mats times
  int in_rows, code_bytes, k_atoms, row_atoms;
  void* out;                    // [mats][rows][cols]
  const int32_t* rows_ptr;
  int pair;                     // the values of the gate projections, then of the up projections
};

// A lane takes eight values of a row, a warp MXD_DEPTH times 256.  Bound by HBM (6.0 TB/s); the values' bytes are looked
// up, which takes half the instructions of computing them.  (By the conversions of
// ep_mx_dgrad_kernel: 5.8 TB/s.  Sixteen values a lane: 4.3.)  Rows of odd lengths have their eights where the output is
// aligned and compute them, 3.1 - 3.4 TB/s (by elements 1.4; looked up, with two scales a pair, 2.8 - 3.0).
constexpr int MXD_DEPTH = 8;

template <class T, bool VEC>
__global__ void __launch_bounds__(MXQ_WARPS * 32) ep_mx_dequant_kernel(const __grid_constant__ MxDequantParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = p.rows_ptr ? max(0, min(*p.rows_ptr, p.rows)) : p.rows;
  const unsigned lines = (unsigned)(p.pair ? 2 * p.mats : p.mats) * (unsigned)rows;
  for (unsigned line = blockIdx.x * MXQ_WARPS + warp; line < lines; line += gridDim.x * MXQ_WARPS) {
    const int out_mat = lines > (unsigned)rows ? (int)(line / (unsigned)rows) : 0, row = (int)(line - (unsigned)out_mat * (unsigned)rows);
    const int up = out_mat >= p.mats ? 1 : 0, mat = out_mat - up * p.mats;
    const int r = p.pair ? mx_pair_row(row, up) : row;
    const uint8_t* codes = p.codes + ((long long)mat * p.in_rows + r) * p.code_bytes;
    const uint8_t* scales = p.scales + (long long)mat * p.row_atoms * p.k_atoms * MX_ATOM_BYTES + mx_scale_offset(r, 0, p.k_atoms);
    T* out = (T*)p.out + ((long long)out_mat * p.rows + row) * p.cols;
    if constexpr (!VEC) {        // rows start anywhere: eights begin where the output is aligned, their codes lie in two words
      constexpr int DEPTH = MXD_DEPTH / 2;
      const int first = -(int)((uintptr_t)out / sizeof(T) % 8);
      for (int c0 = first + blockIdx.y * 256 * DEPTH + lane * 8; c0 < p.cols; c0 += gridDim.y * 256 * DEPTH) {
        uint32_t code[DEPTH][2], b[DEPTH][2];
#pragma unroll
        for (int i = 0; i < DEPTH; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {        // the word with the first of the eight and the next; the first one's scale and the last one's
            const int c = c0 + i * 256, w = (c >> 3) + h, e = min(max(c + 7 * h, 0), p.cols - 1);
            code[i][h] = w >= 0 && 4 * w < p.code_bytes ? reinterpret_cast<const uint32_t*>(codes)[w] : 0u;
            b[i][h] = scales[(long long)(e >> 7) * MX_ATOM_BYTES + (e >> 5 & 3)];
          }
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
          const int c = c0 + i * 256;
          if (c >= p.cols) break;
          const uint32_t q = __funnelshift_r(code[i][0], code[i][1], 4 * (c & 7));
          const float s0 = mx_value(b[i][0]), s1 = mx_value(b[i][1]);
          const int of_first = 32 - (c & 31);        // so many have the first scale
          MxEight<T> v;
#pragma unroll
          for (int e = 0; e < 8; ++e) v.p[e / 2].e[e % 2] = T(mx_element(q >> (4 * e)) * (e < of_first ? s0 : s1));
          if (c >= 0 && c + 8 <= p.cols) {
#pragma unroll
            for (int e = 0; e < (int)sizeof(T) / 2; ++e) __stcs(reinterpret_cast<uint4*>(out + c) + e, reinterpret_cast<const uint4*>(&v)[e]);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (c + e >= 0 && c + e < p.cols) out[c + e] = v.p[e / 2].e[e % 2];
          }
        }
      }
    } else
    for (int c0 = blockIdx.y * 256 * MXD_DEPTH + lane * 8; c0 < p.cols; c0 += gridDim.y * 256 * MXD_DEPTH) {
      uint32_t code[MXD_DEPTH], b[MXD_DEPTH];
#pragma unroll
      for (int i = 0; i < MXD_DEPTH; ++i) {
        const int c = c0 + i * 256;
        code[i] = c < p.cols ? __ldcs(reinterpret_cast<const uint32_t*>(codes + c / 2)) : 0u;
        b[i] = c < p.cols ? scales[(long long)(c >> 7) * MX_ATOM_BYTES + (c >> 5 & 3)] : 0u;
      }
#pragma unroll
      for (int i = 0; i < MXD_DEPTH; ++i) {
        const int c = c0 + i * 256;
        if (c >= p.cols) break;
        const float s = mx_value(b[i]);
        if constexpr (sizeof(T) == 2) {
          const __nv_bfloat162 s2 = __float2bfloat162_rn(s);
          const uint2 lo = mx_bf16x4(code[i]), hi = mx_bf16x4(code[i] >> 16);
          uint4 q = make_uint4(lo.x, lo.y, hi.x, hi.y);
          __nv_bfloat162* v = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = __hmul2(v[e], s2);
          __stcs(reinterpret_cast<uint4*>(out + c), q);
        } else {
          float4 v[2];
          float* f = reinterpret_cast<float*>(v);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = mx_element(code[i] >> (4 * e)) * s;
          __stcs(reinterpret_cast<float4*>(out + c), v[0]);
          __stcs(reinterpret_cast<float4*>(out + c) + 1, v[1]);
        }
      }
    }
  }
}

// Blocks for so many rows (one a warp) of so many parts: enough for a few rounds of the device, columns shared out only
// where the rows are too few for that.
static dim3 mx_grid(long long lines, int parts) {
  const long long most = 148 * 16;
  const long long x = (lines + MXQ_WARPS - 1) / MXQ_WARPS;
  long long y = x >= most ? 1 : most / x;
  if (y > parts) y = parts;
  return dim3((unsigned)(x < most ? x : most), (unsigned)y);
}

template <class T>
static int mx_quant(MxQuantParams& p, bool along_cols, cudaStream_t stream) {
  const bool rows16 = (uintptr_t)p.x % 16 == 0 && (p.stride * sizeof(T)) % 16 == 0 && (p.batch * sizeof(T)) % 16 == 0 && p.cols % 8 == 0;
  constexpr int lane_cols = 2 * mxt_pairs<T>(), block_cols = 32 * lane_cols;
  const bool pieces = ((uintptr_t)p.x | (uintptr_t)p.x2) % 8 == 0 && p.stride % lane_cols == 0 && p.batch % lane_cols == 0 && p.cols % lane_cols == 0;
  if (along_cols) {
    const dim3 grid((unsigned)((p.cols + block_cols - 1) / block_cols), (unsigned)((p.rows + MXT_ROWS - 1) / MXT_ROWS),
                    (unsigned)(p.mats < 32767 ? (p.x2 ? 2 : 1) * p.mats : 65534));
    if (grid.y > 65535) return fail(-5, "mx quantise: %d rows are too many along the last but one axis", p.rows);
    MEP_CUDA_OK(launch_chained(pieces ? (const void*)ep_mx_quant_cols_kernel<T, true> : (const void*)ep_mx_quant_cols_kernel<T, false>,
                               grid, dim3(256), 0, stream, p, 0, 1));
  } else {
    const dim3 grid = mx_grid((long long)p.mats * p.rows, (p.k_atoms * MX_ATOM_K + 256 * MXQ_DEPTH - 1) / (256 * MXQ_DEPTH));
    MEP_CUDA_OK(launch_chained(rows16 ? (const void*)ep_mx_quant_rows_kernel<T, true> : (const void*)ep_mx_quant_rows_kernel<T, false>,
                               grid, dim3(MXQ_WARPS * 32), 0, stream, p, 0, 1));
  }
  return 0;
}

}  // namespace mep

using namespace mep;

extern "C" {

// x [mats][rows][cols] of `type` (bf16, fp16, fp32), `batch` and `stride` elements apart.  along_cols = 0: blocks along the
// columns, output rows are x's; 1: blocks along the rows, output rows are x's columns.  out_rows: rows of an output matrix.
// phases = 4 (one matrix): scales for token rows, else 1.  x2 (along_cols = 1): the up projection packed with x, the gate.
// rows_ptr: rows of x that hold something, on the device; or null.
struct MxQuantDesc {
  const void *x, *x2;
  void *codes, *scales;
  const int32_t* rows_ptr;
  int64_t batch, stride;
  int32_t type, mats, rows, cols, along_cols, out_rows, phases, unused;
};
// The values [mats][rows][cols] in bf16, or fp32; of a pair [2][mats][rows][cols].
struct MxDequantDesc {
  const void *codes, *scales;
  void* out;
  const int32_t* rows_ptr;
  int32_t mats, rows, cols, pair, in_rows, fp32;
};

int mep_mx_quant_desc_bytes() { return (int)(sizeof(MxQuantDesc) << 16 | sizeof(MxDequantDesc)); }

int mep_mx_quantize(const MxQuantDesc* d, cudaStream_t stream) {
  if (d->mats < 0 || d->rows < 0 || d->cols < 0 || d->cols > 0x7F000000 || (int64_t)d->mats * d->rows > 0x7FFFFFFF)
    return fail(-1, "mx quantise: %d x %d x %d elements", d->mats, d->rows, d->cols);
  const bool along_cols = d->along_cols != 0;
  if (d->x2 && (!along_cols || d->phases != 1)) return fail(-2, "mx quantise: a pair is packed along the columns");
  if (along_cols && d->rows_ptr) return fail(-2, "mx quantise: a device row count goes with blocks along the rows");
  if (d->phases != 1 && (d->phases != MX_PHASES || d->mats > 1))
    return fail(-4, "mx quantise: %d phases of %d matrices", d->phases, d->mats);
  if (d->mats == 0 || d->rows == 0 || d->cols == 0) return 0;
  MxQuantParams p;
  const int K = along_cols ? d->rows : d->cols;
  p.x = d->x; p.x2 = d->x2; p.batch = d->batch; p.stride = d->stride; p.mats = d->mats; p.rows = d->rows; p.cols = d->cols;
  p.out_rows = d->out_rows; p.code_bytes = (K + MX_BLOCK - 1) / MX_BLOCK * (MX_BLOCK / 2);
  p.k_atoms = mx_atoms(K); p.row_atoms = mx_atoms(d->out_rows);
  p.codes = (uint8_t*)d->codes; p.scales = (uint8_t*)d->scales; p.rows_ptr = d->rows_ptr; p.phases = d->phases;
  if (d->type == MX_BF16) return mx_quant<__nv_bfloat16>(p, along_cols, stream);
  if (d->type == MX_FP16) return mx_quant<__half>(p, along_cols, stream);
  if (d->type == MX_FP32) return mx_quant<float>(p, along_cols, stream);
  return fail(-3, "mx quantise: unknown type %d", d->type);
}

int mep_mx_dequantize(const MxDequantDesc* d, cudaStream_t stream) {
  if (d->mats < 0 || d->rows < 0 || d->cols < 0 || d->cols > 0x7F000000 || (d->pair ? 2 : 1) * (int64_t)d->mats * d->rows > 0x7FFFFFFF)
    return fail(-1, "mx dequantise: %d x %d x %d elements", d->mats, d->rows, d->cols);
  if (d->mats == 0 || d->rows == 0 || d->cols == 0) return 0;
  MxDequantParams p;
  p.codes = (const uint8_t*)d->codes; p.scales = (const uint8_t*)d->scales; p.mats = d->mats; p.rows = d->rows; p.cols = d->cols;
  p.in_rows = d->in_rows; p.code_bytes = (d->cols + MX_BLOCK - 1) / MX_BLOCK * (MX_BLOCK / 2);
  p.k_atoms = mx_atoms(d->cols); p.row_atoms = mx_atoms(d->in_rows);
  p.out = d->out; p.rows_ptr = d->rows_ptr; p.pair = d->pair;
  const dim3 grid = mx_grid((d->pair ? 2ll : 1ll) * d->mats * d->rows, (d->cols + 256 * MXD_DEPTH - 1) / (256 * MXD_DEPTH));
  const bool vec = d->cols % 8 == 0 && (uintptr_t)d->out % 16 == 0;
  const void* kern = d->fp32 ? (vec ? (const void*)ep_mx_dequant_kernel<float, true> : (const void*)ep_mx_dequant_kernel<float, false>)
                             : (vec ? (const void*)ep_mx_dequant_kernel<__nv_bfloat16, true> : (const void*)ep_mx_dequant_kernel<__nv_bfloat16, false>);
  MEP_CUDA_OK(launch_chained(kern, grid, dim3(MXQ_WARPS * 32), 0, stream, p, 0, 1));
  return 0;
}

}  // extern "C"
