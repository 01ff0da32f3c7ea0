// Grouped product of microscaled 4-bit operands (mx_format.cuh) on the tensor cores' block-scaled form,
// tcgen05.mma.kind::mxf4.block_scale: C[rows of g] = A[rows of g] * W[g]^T, fp32 sums, computed as C^T = W[g] * A^T
// like ep_token_gemm_kernel (token_gemm.cuh): the weights' rows take the fixed M side (256 a CTA pair), the tokens N.
//
// In bytes a tile is what it is there: a k-step of the MMA reads 32 bytes of an operand row (64 elements instead of
// 16 of bf16) and takes as long, so a stage of 128 bytes a row feeds four MMAs and the same ring carries four times the
// operations.  What is new are the scales.  They lie in memory in the atoms that tensor memory takes (128 rows x 4
// blocks), come with their stage by TMA, and tcgen05.cp puts them into tensor memory in front of the stage's MMAs; both
// run in the tensor core's order, and two sets of columns are used in turn.  In a pair either CTA has the scales of its
// own 128 weight rows and those of all tokens.
//
// Tensor memory: two accumulators of 224 columns and two sets of 24 for scales.  (256 tokens a tile would leave no
// room for scales beside a second accumulator.)
// Token tiles start at multiples of 32 rows of the whole tensor, whatever row a group starts at: then a tile's scales
// are whole atoms of one of their four phases.  Rows of a neighbouring group in a tile are computed and not stored.
//
// What bounds it: short groups the stream of the weights (16 tokens, 32 experts, 7168 -> 2 x 2048: 83 us, 6.0 TB/s; a launch has
// 5 us before its first bytes and after its last), long ones the operand bytes that L2 and the SMs exchange, 11 - 13
// TB/s, and in a long run the power cap (8192 x 7168 x 4096 82 us, 5.9 PFLOP/s; 91 at 1.3 - 1.6 GHz).  Measured and worse: two
// token tiles that share staged weights, three quarters of the bytes, but weights that wait for the second tile are slots
// with nothing in flight (118 us); weights in one contiguous piece a k-block (the same).
//   warp 0  TMA producer
//   warp 1  MMA issuer
//   warps 2..  epilogue, two or three sets of four, as in ep_token_gemm_kernel
//
// SwiGLU: gate and up columns come packed in turns of 16 rows, so that a warp's 32 rows of tensor memory hold both of 16
// activations: read as two fragments of 16 rows, gate and up of an element meet in one thread's registers, in fp32.
// The activation is rounded to bf16 and, if it is the next product's operand, quantised while it is in shared memory.
// Backward: the same product again, with the gradients of gate and up computed where the forward pass has the
// activation.  Gate and up are then neither kept between the passes nor rounded: a quarter of a bf16 product's time for
// four bytes an element of either.
#pragma once

#include "device/mx_format.cuh"

namespace mep {

enum { MX_EPI_BF16 = 0, MX_EPI_SWIGLU = 1, MX_EPI_SWIGLU_SAVE = 2, MX_EPI_SWIGLU_BWD = 3 };

constexpr int MXG_MAX_N = 224;                   // tokens of a tile, at most
constexpr int MXG_BK = 256;                      // elements of a k-block: 128 bytes a row
constexpr int MXG_W_BYTES = 128 * 128;
constexpr int MXG_S_BYTES = 2 * MX_ATOM_BYTES;   // scales of 128 rows and one k-block
constexpr int MXG_BOXES = 5;
__host__ __device__ constexpr int mxg_box_rows(int b) { return b == 0 ? 16 : b == 4 ? MXG_MAX_N / 2 : 32 * b; }
// A stage: weights, half of the tokens (whole swizzle atoms), scales of the weights and of all tokens.
constexpr int MXG_T_BYTES = MXG_MAX_N / 2 * 128, MXG_T_ATOMS = (MXG_MAX_N + 127) / 128;
constexpr int MXG_STAGE = MXG_W_BYTES + MXG_T_BYTES + MXG_S_BYTES * (1 + MXG_T_ATOMS);
static_assert(MXG_T_BYTES % 1024 == 0 && MXG_STAGE % 1024 == 0, "swizzle atoms");
constexpr uint32_t MXG_SCALES_AT = 2 * MXG_MAX_N;
constexpr uint32_t MXG_SCALE_COLS = 24;             // columns of tensor memory of a set: 8 of weights, 16 of tokens
static_assert(MXG_SCALES_AT + 2 * MXG_SCALE_COLS <= 512, "tensor memory");

struct MxParams {
  CUtensorMap w, ws;               // weights' codes, 128-byte x 128-row boxes; scales, two atoms a box
  CUtensorMap tok[MXG_BOXES], ts;  // token rows in boxes of 16, 32, 64, 96, 112 rows; scales
  const int32_t* cu_seqlens;
  const int32_t* pads;
  int ngroups, total_rows, K;
  int w_rows, w_atoms;             // rows and row atoms of a group's weights
  int t_atoms;                     // row atoms of a phase of the tokens' scales
  int N;                           // output columns
  __nv_bfloat16* out;              // y or act, or null
  __nv_bfloat16 *gate, *up;
  uint8_t *codes, *scales;         // act quantised, or null (scales at four phases, out_atoms row atoms each)
  int code_bytes, k_atoms, out_atoms;      // of act
  int vec_out;
  const float* row_scale;
  const float* d_act;              // backward: gradient of the activation, [total_rows][N]
  int zero_tail;                   // rows behind the last group become zeros
  int check_groups;                // a group whose rows are no multiple of 64 is recorded in `status`
  float* d_scale;                  // parts of the scales' gradients, [CTA's columns][total_rows], or null
  long long ldc;
  int32_t* status;
  unsigned long long timeout_ns;
};

// Sets of four epilogue warps.  (Gate and up of the decoder's experts, 32768 rows, 2048 -> 768: two sets 86 us, three 78;
// backward 125, 117.  Four cost a slot of the ring: 32 x 1024 rows, 7168 -> 2048 324 us, 338.  Plain products, whose
// epilogue is shorter: two 207 us, three 211.)
template <int EPI> constexpr int mxg_sets() { return EPI == MX_EPI_SWIGLU || EPI == MX_EPI_SWIGLU_BWD ? 3 : 2; }
template <int EPI> constexpr int mxg_threads() { return 64 + mxg_sets<EPI>() * 128; }
// Shared memory that the kernel declares itself: staged tokens, group tables, scales of two tiles, barriers (rounded up).
template <int EPI> constexpr int mxg_token_row() { return (EPI == MX_EPI_SWIGLU_SAVE ? 384 : EPI == MX_EPI_SWIGLU ? 128 : 256) + 16; }
template <int EPI> constexpr int mxg_static_smem() {
  return mxg_sets<EPI>() * TG_CHUNK * mxg_token_row<EPI>() + (3 * MAX_GROUPS + 1) * 4 + (EPI == MX_EPI_BF16 ? 8 : mxg_sets<EPI>() * 128 * 4) +
         (EPI == MX_EPI_SWIGLU_BWD ? mxg_sets<EPI>() * 4 * TG_CHUNK * 4 : 0) + 512;
}

// Stages: as many as the device's shared memory has room for beside these.  (Short groups do not gain from smaller stages,
// of 64 tokens, and nine of them: 32 groups of 1 to 64 rows, 7168 -> 2 x 2048 96 - 98 us, 98 - 100; 128, 2048 -> 2 x 768 53 - 55, 51 - 55.)
template <int EPI> constexpr int mxg_stages() { return (227 * 1024 - 1024 - mxg_static_smem<EPI>()) / MXG_STAGE; }

struct MxTile {
  int g, row0, n;          // first row (a multiple of 32), tokens computed (a multiple of 32)
  int lo, hi, zero_to;     // rows stored: [lo, hi); this tile also zeroes the rows [hi, zero_to)
  int m;                   // first weight row
};

// D (+)= A * B with one E8M0 scale per 32 elements; A and B E2M1, K = 64; issued by one thread for the pair.
__device__ __forceinline__ void umma_mxf4_2cta(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                               uint32_t scale_a, uint32_t scale_b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)
      : "memory");
}
// An atom of scales (32 rows of 16 bytes) from shared memory into four columns of tensor memory, in every warp's quarter;
// in both CTAs of the pair, each from its own shared memory.
__device__ __forceinline__ void tmem_cp_scales_2cta(uint32_t tmem_dst, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem_dst), "l"(desc) : "memory");
}
// Unswizzled rows of 16 bytes: groups of eight rows 128 bytes apart.
__device__ __forceinline__ uint64_t make_scale_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr >> 4) & 0x3FFF) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
// kind::mxf4: bits 4..5 scale byte of B, 7..9 A format and 10..11 B format (1 = E2M1), 17..22 N >> 3, 23 scale format
// (1 = E8M0), 24..28 M >> 4, 29..30 scale byte of A.
__host__ __device__ constexpr uint32_t make_instr_desc_mxf4(int M, int N, int scale_byte) {
  return ((uint32_t)scale_byte << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) |
         ((uint32_t)(M >> 4) << 24) | ((uint32_t)scale_byte << 29);
}

// 1 / (1 + e^-x).  Its relative error is that of __expf where x is negative, 2^-23 (2 + 1.2 |x|) or so, and far below the
// bf16 rounding of what it goes into.  (With the exact division gate and up of the decoder's experts, whose
// epilogue is as long as their reduction, took 134 us, so 86.)
__device__ __forceinline__ float mx_sigmoid(float x) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + __expf(-x)));
  return r;
}

template <int EPI>
__global__ void __launch_bounds__(mxg_threads<EPI>(), 1)
ep_mx_gemm_kernel(const __grid_constant__ MxParams p) {
  constexpr int SETS = mxg_sets<EPI>();
  constexpr int NST = mxg_stages<EPI>(), STAGE = MXG_STAGE;
  constexpr bool GATED = EPI != MX_EPI_BF16, SAVE = EPI == MX_EPI_SWIGLU_SAVE, BWD = EPI == MX_EPI_SWIGLU_BWD;
  constexpr int TOK_ROW = mxg_token_row<EPI>();     // bytes of a staged token
  const int crank = (int)cluster_cta_rank();
  const int work_id0 = (int)(blockIdx.x >> 1), work_stride = (int)(gridDim.x >> 1);
  extern __shared__ uint8_t smem_dyn[];
  __shared__ __align__(8) uint64_t full[NST];
  __shared__ __align__(8) uint64_t empty[NST];
  __shared__ __align__(8) uint64_t acc_full[2];
  __shared__ __align__(8) uint64_t acc_empty[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ int s_end[MAX_GROUPS], s_span[MAX_GROUPS];
  __shared__ int s_prefix[MAX_GROUPS + 1];
  __shared__ __align__(128) uint8_t s_stage[SETS][TG_CHUNK * TOK_ROW];
  __shared__ float s_part[BWD ? SETS : 1][BWD ? 4 : 1][BWD ? TG_CHUNK : 1];     // sums over a quarter's columns
  // row scales of a set's tokens in the present tile, chunk by chunk.  A set's own: it may be a whole tile ahead of another
  __shared__ float s_scale[GATED ? SETS : 1][GATED ? 128 : 1];

  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  uint8_t* stages = (uint8_t*)(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  volatile int* abortp = &s_abort;

  if (warp == 0) {
    if (lane == 0) {
      // both CTAs' loads count on the leader's full barrier, on which only its producer arrives
      for (int s = 0; s < NST; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
      for (int a = 0; a < 2; ++a) { mbar_init(&acc_full[a], 1); mbar_init(&acc_empty[a], 8 * SETS); }
      mbar_fence_init();
      s_abort = 0;
    }
    if (lane == 1) { tma_prefetch_desc(&p.w); tma_prefetch_desc(&p.ws); }
    if (lane == 2) { tma_prefetch_desc(&p.ts); tma_prefetch_desc(&p.tok[0]); }
  }
  if (warp == 1) { tmem_alloc2(&s_tmem, 512); tmem_relinquish2(); }
  pdl_wait();               // nothing of this is read from memory; what follows is
  // Group tables: ends, and rows with tokens counted from the multiple of 32 at or before the first.  (One round of loads
  // for all groups, 1 us; the padding ranges looked up in the scan below and again for every tile cost 2 - 4 us a launch.)
  for (int g = tid; g < p.ngroups; g += mxg_threads<EPI>()) {
    // (no row outside the tensors is stored, whatever cu_seqlens says)
    auto clamped = [&](int end) { return min(max(end, 0), p.total_rows); };
    const int start = g == 0 || p.cu_seqlens == nullptr ? 0 : clamped(p.cu_seqlens[g - 1]);
    const int end = clamped(p.cu_seqlens != nullptr ? p.cu_seqlens[g] : p.total_rows);
    s_end[g] = end;
    if constexpr (EPI == MX_EPI_BF16) {
      // (one that ends where the tensors do has nothing behind it that the weight grads could read)
      if (p.check_groups && blockIdx.x == 0 && (end - start) % 64 != 0 && end != p.total_rows && p.status != nullptr &&
          atomicCAS(p.status, 0, (int)ST_BAD_INDEX) == 0) {
        p.status[1] = KID_MX_GEMM;
        p.status[4] = g;
        p.status[5] = end - start;
      }
    }
    // (a group of nothing but padding: negative, of one row, for a tile that writes the zeros)
    const int tokens = end > start ? group_tokens(p, g, start, end) : 0;
    s_span[g] = tokens > 0 ? (start & 31) + tokens : end > start ? -((start & 31) + 1) : 0;
  }
  __syncthreads();
  if (warp == 0) {      // exclusive prefix of token tiles per group
    int run = 0;
    for (int g0 = 0; g0 < p.ngroups; g0 += 32) {
      const int g = g0 + lane;
      const int nt = g < p.ngroups ? (abs(s_span[g]) + MXG_MAX_N - 1) / MXG_MAX_N : 0;
      int incl = nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (g < p.ngroups) s_prefix[g] = run + incl - nt;
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) s_prefix[p.ngroups] = run;
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = s_tmem;

  const int m_tiles = (p.w_rows + 255) / 256;
  const long long total_tiles = (long long)s_prefix[p.ngroups] * m_tiles;
  // Tile `id`, for a whole warp; ids only grow, and g is where the warp's last tile was.
  auto get = [&](long long id, int& g) {
    while (true) {      // the first group behind g that starts beyond id, 32 at a time
      const int i = g + 1 + lane;
      const uint32_t beyond = __ballot_sync(0xffffffffu, i >= p.ngroups || (long long)s_prefix[i] * m_tiles > id);
      if (beyond != 0u) { g += __ffs(beyond) - 1; break; }
      g += 32;
    }
    MxTile t;
    t.g = g;
    const int nt = s_prefix[g + 1] - s_prefix[g];
    const int local = (int)(id - (long long)s_prefix[g] * m_tiles);
    const int mi = local / nt, ti = local - mi * nt;       // tiles that share weights are neighbours
    const int start = g == 0 ? 0 : s_end[g - 1], end = s_end[g];
    const int span = s_span[g], length = abs(span), valid = span < 0 ? start : start + length - (start & 31);
    t.n = ((length + nt - 1) / nt + 31) & ~31;
    t.row0 = (start & ~31) + ti * t.n;
    t.lo = max(t.row0, start);
    t.hi = max(t.lo, min(t.row0 + t.n, valid));
    t.zero_to = ti == nt - 1 ? end : 0;
    t.m = mi * 256;
    return t;
  };
  const int num_kb = (p.K + MXG_BK - 1) / MXG_BK;
  auto warp_wait = [&](uint64_t* bar, uint32_t parity, int where) {
    return __all_sync(0xffffffffu, gemm_wait(bar, parity, abortp, p, where)) != 0;
  };
  // (the same in every lane: said so, see ep_token_gemm_kernel)
  auto uniform = [&](int v) { return __shfl_sync(0xffffffffu, v, 0); };

  if (warp == 0) {
    // ================= TMA producer =================
    const bool issue = elect_one();
    int at = 0;
    RingSlot st;
    bool ok = true;
    for (long long id = work_id0; id < total_tiles && ok; id += work_stride) {
      const MxTile t = get(id, at);
      const int n = uniform(t.n), row0 = uniform(t.row0), g = uniform(t.g), m = uniform(t.m);
      const int box = n / 2 <= 16 ? 0 : (n / 2 + 31) / 32;
      const int atoms = (n + 127) / 128;       // row atoms that hold the tokens' scales
      const CUtensorMap* tmap = &p.tok[0] + box;
      const uint32_t bytes = 2u * (uint32_t)(MXG_W_BYTES + mxg_box_rows(box) * 128 + (1 + atoms) * MXG_S_BYTES);
      const int wrow = g * p.w_rows + m + 128 * crank, watom = g * p.w_atoms + m / 128 + crank;
      const int trow = row0 + crank * (n / 2), tatom = (row0 >> 5 & 3) * p.t_atoms + (row0 >> 7);
      for (int kb = 0; kb < num_kb; ++kb, st.next(NST)) {
        const int s = st.slot;
        ok = warp_wait(&empty[s], st.parity ^ 1u, 1);
        if (!ok) break;
        if (!issue) continue;
        uint8_t* sw = stages + (size_t)s * STAGE;
        uint8_t* ss = sw + MXG_W_BYTES + MXG_T_BYTES;
        const uint32_t bar = mapa_u32(&full[s], 0);
        if (crank == 0) mbar_expect_tx(&full[s], bytes);
        tma_load_2d_pair(sw, &p.w, kb * 128, wrow, bar);
        tma_load_2d_pair(sw + MXG_W_BYTES, tmap, kb * 128, trow, bar);
        tma_load_2d_pair(ss, &p.ws, kb * 256, watom, bar);
        for (int a = 0; a < atoms; ++a) tma_load_2d_pair(ss + (1 + a) * MXG_S_BYTES, &p.ts, kb * 256, tatom + a, bar);
      }
    }
  } else if (warp == 1) {
    // ================= MMA issuer (the leader issues for both CTAs of the pair) =================
    if (crank == 0) {
      const bool issue = elect_one();
      const uint64_t desc_w = make_smem_desc(smem_u32(stages), 16, 1024);
      const uint64_t desc_t = make_smem_desc(smem_u32(stages) + MXG_W_BYTES, 16, 1024);
      const uint64_t desc_s = make_scale_desc(smem_u32(stages) + MXG_W_BYTES + MXG_T_BYTES);
      RingSlot st;
      int tile_n = 0, at = 0;
      uint32_t set = 0;
      bool ok = true;
      for (long long id = work_id0; id < total_tiles && ok; id += work_stride, ++tile_n) {
        const int n = uniform(get(id, at).n);
        const uint32_t idesc0 = make_instr_desc_mxf4(256, n, 0), idesc2 = make_instr_desc_mxf4(256, n, 2);
        const int acc = tile_n & 1;
        if (!warp_wait(&acc_empty[acc], ((uint32_t)(tile_n >> 1) & 1u) ^ 1u, 2)) break;
        tc_fence_after();
        const uint32_t tacc = tmem_base + (uint32_t)acc * MXG_MAX_N;
        uint32_t add = 0u;
        for (int kb = 0; kb < num_kb; ++kb, st.next(NST), set ^= MXG_SCALE_COLS) {
          const int s = st.slot;
          ok = warp_wait(&full[s], st.parity, 3);
          if (!ok) break;
          tc_fence_after();
          if (issue) {
            const uint32_t off = (uint32_t)(s * (STAGE >> 4));
            const uint64_t da = desc_w + off, db = desc_t + off, ds = desc_s + off;
            const uint32_t tsa = tmem_base + MXG_SCALES_AT + set, tsb = tsa + 8;
            // (row atoms behind a short tile's tokens are copied as they lie there: nothing is multiplied by them.  With
            // the number of atoms as the loop's bound the issuer was what the kernel waited for: 8192 x 7168 x 4096 90 us, 82)
#pragma unroll
            for (int j = 0; j < 2; ++j) {        // block atoms of the k-block
              tmem_cp_scales_2cta(tsa + 4 * j, ds + j * (MX_ATOM_BYTES >> 4));
#pragma unroll
              for (int a = 0; a < MXG_T_ATOMS; ++a)
                tmem_cp_scales_2cta(tsb + 8 * j + 4 * a, ds + (((1 + a) * MXG_S_BYTES + j * MX_ATOM_BYTES) >> 4));
            }
            // 64 elements each: two of an atom row's four scales
            umma_mxf4_2cta(tacc, da, db, idesc0, tsa, tsb, add);
            umma_mxf4_2cta(tacc, da + 2, db + 2, idesc2, tsa, tsb, 1u);
            umma_mxf4_2cta(tacc, da + 4, db + 4, idesc0, tsa + 4, tsb + 8, 1u);
            umma_mxf4_2cta(tacc, da + 6, db + 6, idesc2, tsa + 4, tsb + 8, 1u);
            umma_commit_2cta(&empty[s], 3);
          }
          add = 1u;
        }
        if (!ok) break;
        if (issue) umma_commit_2cta(&acc_full[acc], 3);
      }
    }
  } else {
    // ========= epilogue: sets of four warps, each warp one quarter of the CTA's weight rows =========
    const int q = warp & 3, set = (warp - 2) >> 2;
    const int te = tid - 64 - set * 128;                    // 0..127
    const int step = SETS * TG_CHUNK;
    int tile_n = 0, at = 0;
    uint8_t* const sb = s_stage[set];
    // this thread's row of the matrices that its warp stores: token 8 (lane / 16) + lane % 8, columns 8 (lane / 8 % 2)
    const uint32_t st_addr = smem_u32(sb) + (uint32_t)((8 * (lane >> 4) + (lane & 7)) * TOK_ROW + q * (GATED ? 32 : 64) +
                                                       ((lane >> 3) & 1) * 16);
    const bool vec_ok = p.vec_out != 0;
    for (long long id = work_id0; id < total_tiles; id += work_stride, ++tile_n) {
      const MxTile t = get(id, at);
      const int acc = tile_n & 1;
      // this set's chunks start at tokens first, first + step, ...; the sets change places from tile to tile, so that
      // tiles of few tokens keep all of them busy
      const int first = (set + tile_n) % SETS * TG_CHUNK, my_tok = (te >> 5) * step + first + (te & 31);
      if constexpr (GATED) {
        // (published by epilogue_all() below; the set's last reads of the tile before were in front of its last epilogue_sync())
        static_assert(4 * SETS * TG_CHUNK >= MXG_MAX_N, "a thread has one token of its set at most");
        const int r = t.row0 + my_tok;
        if (my_tok < t.n) s_scale[set][te] = r >= t.lo && r < t.hi && p.row_scale != nullptr ? p.row_scale[r] : 1.f;
      }
      // the gradients that meet a chunk's fragments: columns 8 half + lane / 4 of the quarter, tokens 8 j + 2 (lane % 4)
      // and the next at [4 j + 2 half]; on their way before the fragments are
      float da[BWD ? 16 : 1];
      auto load_gradients = [&](int c) {
        if constexpr (BWD) {
          const int col = t.m / 2 + 64 * crank + q * 16 + (lane >> 2);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int row = t.row0 + c + 8 * (i >> 2) + 2 * (lane & 3) + (i & 1), x = col + 8 * (i >> 1 & 1);
            da[i] = row >= t.lo && row < t.hi && x < p.N ? __ldg(p.d_act + (long long)row * p.ldc + x) : 0.f;
          }
        }
      };
      if (first < t.n) load_gradients(first);
      const bool have = gemm_wait(&acc_full[acc], (uint32_t)(tile_n >> 1) & 1u, abortp, p, 4);
      __syncwarp();
      if (!epilogue_all(set, have)) break;
      tc_fence_after();
      const uint32_t tacc = tmem_base + (uint32_t)acc * MXG_MAX_N + ((uint32_t)(q * 32) << 16);
      uint32_t r[32];
      auto release_acc = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (crank != 0) mbar_arrive_remote(&acc_empty[acc], 0);
          else mbar_arrive(&acc_empty[acc]);
        }
      };
      // the two scales of this CTA's 64 activations of a row: four of its eight threads store one phase each
      auto store_scales = [&](int row, uint32_t both) {
        const int s = te & 7, at = row - 32 * s, k = t.m / 2 + 64 * crank;
        if (s < MX_PHASES && at >= 0 && (k >> 7) < p.k_atoms)
          *reinterpret_cast<uint16_t*>(p.scales + (long long)s * p.out_atoms * p.k_atoms * MX_ATOM_BYTES +
                                       mx_scale_offset(at, k >> 7, p.k_atoms) + (k >> 5 & 3)) = (uint16_t)both;
      };
      // A chunk's staged columns, from byte `at` of a token's row on, to rows of dst that start anywhere: neighbouring
      // threads store neighbouring elements.  (Eight a thread: 8192 x 7168 -> 2047 90 us, so 57; 49 for 2048.)
      auto store_elements = [&](__nv_bfloat16* dst, int at, int c) {
        constexpr int W = GATED ? 64 : 128;
        const int f = te & (W - 1), col = (GATED ? t.m / 2 : t.m) + W * crank + f;
        if (dst == nullptr || col >= p.N) return;
#pragma unroll 1
        for (int k = te / W; k < TG_CHUNK; k += 128 / W) {
          const int row = t.row0 + c + k;
          if (row >= t.lo && row < t.hi) dst[(long long)row * p.ldc + col] = *reinterpret_cast<const __nv_bfloat16*>(sb + k * TOK_ROW + at + f * 2);
        }
      };
      if (first < t.n) {
        tmem_ld_16x256_x4(tacc + first, r);
        tmem_ld_16x256_x4(tacc + first + (16u << 16), r + 16);
      } else {
        release_acc();
      }
#pragma unroll 1
      for (int c = first, own = 0; c < t.n; c += step, own += TG_CHUNK) {      // own: counted over the set's tokens
        __syncwarp();
        tmem_ld_wait();
        uint32_t pk[16];       // [16-row half][token block][lower, upper 8 rows]
        uint32_t pa[8];        // activations [token block][lower, upper 8 columns]
        auto pack = [](float a, float b) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
          return *reinterpret_cast<const uint32_t*>(&h);
        };
        if constexpr (BWD) {
          const int col = t.m / 2 + 64 * crank + q * 16 + (lane >> 2);
          float part[8];       // of token [2 j + e], over this thread's two columns
#pragma unroll
          for (int i = 0; i < 8; ++i) part[i] = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float dg[2], du[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float g = __uint_as_float(r[2 * i + e]), u = __uint_as_float(r[16 + 2 * i + e]);
              const float sig = mx_sigmoid(g), d = da[2 * i + e];
              const float ds = d * s_scale[set][own + 8 * (i >> 1) + 2 * (lane & 3) + e];
              // (columns behind the last have whatever lies behind the weights)
              part[2 * (i >> 1) + e] += col + 8 * (i & 1) < p.N ? d * (g * sig) * u : 0.f;
              dg[e] = ds * u * (sig * (1.f + g * (1.f - sig)));
              du[e] = ds * (g * sig);
            }
            pk[i] = pack(dg[0], dg[1]);
            pk[8 + i] = pack(du[0], du[1]);
          }
          if (p.d_scale != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) part[i] += __shfl_xor_sync(0xffffffffu, part[i], o);
              if (lane < 4) s_part[set][q][8 * (i >> 1) + 2 * lane + (i & 1)] = part[i];
            }
          }
          if (c + step < t.n) load_gradients(c + step);
        } else if constexpr (GATED) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float a[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float g = __uint_as_float(r[2 * i + e]), u = __uint_as_float(r[16 + 2 * i + e]);
              a[e] = g * mx_sigmoid(g) * u * s_scale[set][own + 8 * (i >> 1) + 2 * (lane & 3) + e];
            }
            pa[i] = pack(a[0], a[1]);
          }
        }
        if constexpr (EPI == MX_EPI_BF16 || SAVE) {
#pragma unroll
          for (int i = 0; i < 16; ++i) pk[i] = pack(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
        }
        if (c + step < t.n) {            // the next 32 tokens travel while these leave
          tmem_ld_16x256_x4(tacc + c + step, r);
          tmem_ld_16x256_x4(tacc + c + step + (16u << 16), r + 16);
        } else {
          release_acc();
        }
        __syncwarp();
        if constexpr (GATED && !BWD) {
#pragma unroll
          for (int j = 0; j < 4; j += 2)
            stmatrix_x4_trans(st_addr + (uint32_t)(j * 8 * TOK_ROW), pa[2 * j], pa[2 * j + 1], pa[2 * j + 2], pa[2 * j + 3]);
        }
        if constexpr (!GATED || SAVE || BWD) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; j += 2)
              stmatrix_x4_trans(st_addr + (uint32_t)(j * 8 * TOK_ROW + (SAVE ? 128 * (1 + h) : BWD ? 128 * h : h * 32)),
                                pk[8 * h + 2 * j], pk[8 * h + 2 * j + 1], pk[8 * h + 2 * j + 2], pk[8 * h + 2 * j + 3]);
        }
        __syncwarp();
        epilogue_sync(set);
        if (!vec_ok) {
          store_elements(BWD ? p.gate : p.out, 0, c);
          if constexpr (SAVE) { store_elements(p.gate, 128, c); store_elements(p.up, 256, c); }
          if constexpr (BWD) store_elements(p.up, 128, c);
        }
        if constexpr (BWD) {
          const int f = (te & 7) * 8, col0 = t.m / 2 + 64 * crank + f;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int k = (te >> 3) + 16 * i, row = t.row0 + c + k;
            if (!vec_ok || row < t.lo || row >= t.hi || col0 >= p.N) continue;
            const long long off = (long long)row * p.ldc + col0;
            store8(p.gate + off, *reinterpret_cast<const uint4*>(sb + k * TOK_ROW + f * 2), p.N - col0, true);
            store8(p.up + off, *reinterpret_cast<const uint4*>(sb + k * TOK_ROW + 128 + f * 2), p.N - col0, true);
          }
          if (p.d_scale != nullptr && te < TG_CHUNK) {
            const int row = t.row0 + c + te;
            if (row >= t.lo && row < t.hi)
              p.d_scale[(long long)(t.m / 128 + crank) * p.total_rows + row] =
                  (s_part[set][0][te] + s_part[set][1][te]) + (s_part[set][2][te] + s_part[set][3][te]);
          }
        } else if constexpr (GATED) {
          const int f = (te & 7) * 8, col0 = t.m / 2 + 64 * crank + f;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int k = (te >> 3) + 16 * i, row = t.row0 + c + k;
            const bool mine = row >= t.lo && row < t.hi;
            const uint4 a4 = *reinterpret_cast<const uint4*>(sb + k * TOK_ROW + f * 2);
            const long long off = (long long)row * p.ldc + col0;
            if (vec_ok && mine && col0 < p.N) {
              if (p.out) store8(p.out + off, a4, p.N - col0, true);
              if constexpr (SAVE) {
                if (p.gate) store8(p.gate + off, *reinterpret_cast<const uint4*>(sb + k * TOK_ROW + 128 + f * 2), p.N - col0, true);
                if (p.up) store8(p.up + off, *reinterpret_cast<const uint4*>(sb + k * TOK_ROW + 256 + f * 2), p.N - col0, true);
              }
            }
            if (p.codes != nullptr) {      // four neighbouring threads hold a block, eight a row's two
              uint32_t w[4] = {a4.x, a4.y, a4.z, a4.w}, top = 0u;
              if (col0 + 8 > p.N) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  w[j] &= (col0 + 2 * j < p.N ? 0xFFFFu : 0u) | (col0 + 2 * j + 1 < p.N ? 0xFFFF0000u : 0u);
              }
#pragma unroll
              for (int j = 0; j < 4; ++j) top = __vmaxu2(top, w[j] & 0x7FFF7FFFu);
              uint32_t a = max(top << 16, top & 0xFFFF0000u);
              a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));
              a = max(a, __shfl_xor_sync(0xffffffffu, a, 2));
              const uint32_t b = mx_scale(a);
              const __nv_bfloat162 inv = __float2bfloat162_rn(mx_inverse(b));
              float v[8];
#pragma unroll
              for (int j = 0; j < 4; ++j)       // (exact: a power of two)
                *reinterpret_cast<float2*>(v + 2 * j) = __bfloat1622float2(__hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]), inv));
              const uint32_t both = __shfl_sync(0xffffffffu, b, lane & 24) | __shfl_sync(0xffffffffu, b, (lane & 24) + 4) << 8;
              if (mine) {
                if (col0 < 2 * p.code_bytes)
                  *reinterpret_cast<uint32_t*>(p.codes + (long long)row * p.code_bytes + col0 / 2) = b == 255u ? 0u : mx_codes(v);
                store_scales(row, both);
              }
            }
          }
        } else {
          const int f = (te & 15) * 8, col0 = t.m + 128 * crank + f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = (te >> 4) + 8 * i, row = t.row0 + c + k;
            if (!vec_ok || row < t.lo || row >= t.hi || col0 >= p.N) continue;
            store8(p.out + (long long)row * p.ldc + col0, *reinterpret_cast<const uint4*>(sb + k * TOK_ROW + f * 2), p.N - col0, true);
          }
        }
        epilogue_sync(set);              // every row of the set's buffer has been read: it may be filled again
      }
      {      // padding rows that no tile computes
        constexpr int V = GATED ? 8 : 16;                    // vectors of this CTA's columns in a row
        const int f = (te & (V - 1)) * 8, col0 = (GATED ? t.m / 2 : t.m) + V * 8 * crank + f;
        for (int row = t.hi + (te + 128 * set) / V; row < t.zero_to; row += 128 * SETS / V) {
          const uint4 zero = make_uint4(0, 0, 0, 0);
          const long long off = (long long)row * p.ldc + col0;
          if constexpr (BWD) {
            if (p.d_scale != nullptr && (te & 7) == 0) p.d_scale[(long long)(t.m / 128 + crank) * p.total_rows + row] = 0.f;
          }
          if (col0 < p.N) {
            if (p.out) store8(p.out + off, zero, p.N - col0, vec_ok);
            if constexpr (SAVE || BWD) {
              if (p.gate) store8(p.gate + off, zero, p.N - col0, vec_ok);
              if (p.up) store8(p.up + off, zero, p.N - col0, vec_ok);
            }
          }
          if constexpr (GATED) {
            if (p.codes != nullptr) {
              if (col0 < 2 * p.code_bytes) *reinterpret_cast<uint32_t*>(p.codes + (long long)row * p.code_bytes + col0 / 2) = 0u;
              store_scales(row, 0u);
            }
          }
        }
      }
    }
  }
  if constexpr (EPI == MX_EPI_BF16) {
    if (p.zero_tail && warp >= 2) {      // a warp a row
      const int warps = 4 * SETS;
      for (int row = s_end[p.ngroups - 1] + (int)blockIdx.x * warps + warp - 2; row < p.total_rows; row += (int)gridDim.x * warps)
        for (int c = lane * 8; c < p.N; c += 256) store8(p.out + (long long)row * p.ldc + c, make_uint4(0, 0, 0, 0), p.N - c, p.vec_out != 0);
    }
  }
  pdl_launch_dependents();   // (a kernel that waits for this one may take what room there is beside the last tiles)
  // ---- teardown: everything joins, in-flight work is given time to land on an abort ----------
  tc_fence_before();
  __syncthreads();
  if (s_abort) {
    unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) { }
  }
  cluster_sync_all();        // neither CTA leaves while its peer may still touch it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc2(tmem_base, 512);
  }
}

// Sums of the parts above, in their order.
__global__ void __launch_bounds__(256) ep_mx_sum_parts_kernel(const float* __restrict__ parts, int n, int rows,
                                                              const int32_t* __restrict__ rows_ptr, float* __restrict__ sum) {
  const int r = blockIdx.x * 256 + threadIdx.x, used = rows_ptr ? min(*rows_ptr, rows) : rows;
  if (r >= rows) return;
  float s = 0.f;
  if (r < used)
    for (int i = 0; i < n; ++i) s += parts[(long long)i * rows + r];
  sum[r] = s;
}

}  // namespace mep
