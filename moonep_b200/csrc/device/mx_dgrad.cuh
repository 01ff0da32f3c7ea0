// Token-major grouped products of bf16 rows with microscaled 4-bit weights (mx_format.cuh) whose blocks lie along the
// OUTPUT columns: the gradients of the products of mx_gemm.cuh with respect to their rows.  C[rows of g] = A W[g], W[g]
// [K][columns]; computed as C^T = W^T A^T like ep_token_gemm_kernel, in bf16: a scale is shared by neighbouring columns, not
// along the reduction, so the block-scaled MMA cannot take them.
//
// Four warps read the codes of a k-block (64 weight rows x 128 columns a CTA, 4 KB) from shared memory and write the bf16
// operand of the MMA: every code's value times its scale is a bf16, exactly.  What this saves are the bf16 weights in memory,
// two bytes an element written and read again.  For each k-block a chain of waits, loads, arithmetic and stores, whose turns
// four teams of four warps take; long groups are bound by the MMAs (and the power cap), short ones by this chain.  2 x 768 ->
// 2048 of 128 groups of 256 rows, in us: one team 379, two 240, three 207; with fewer instructions a code 166; with a warp of its own
// for the codes, which runs ahead of the tokens' slots, 151 (two teams 164, four 150; 32 x 64 rows, 2 x 2048 -> 7168: two 322,
// three 304 - 343, four 280 - 312).  Against the product of bf16 weights and the time to make them: 92 us, 115 + 121 (2048 -> 768);
// 150, 174 + 178 (2 x 768 -> 2048); 280 - 312, 313 + 399 (32 x 64 rows, 2 x 2048 -> 7168); 1300 - 1740, 1260 + 420 (32 x 1024).
// One group of 8192 rows, where a weight is decoded for each of its 32 token tiles: 113 - 171, 103 - 155 + 12 (by the clock).
// A chain of slots:
//   warp 0       TMA producer of the token rows (counted on the leader's barrier, for both CTAs)
//   warp 1       MMA issuer: waits for the pair's tokens and for both CTAs' eight decoding warps
//   warp 2       TMA producer of the codes (on this CTA's own barriers)
//   warps 3..18  decode, four teams of four that take k-blocks in turn: 16 weight rows a warp, eight columns a lane and step
//   warps 19..26 epilogue, two sets of four, as in ep_token_gemm_kernel
// Weight rows behind the reduction's end are decoded as zeros (what lies there may be a NaN).
#pragma once

#include <type_traits>

#include "device/mx_format.cuh"

namespace mep {

constexpr int MXD_SLOTS = 5;                          // of tokens and decoded weights
constexpr int MXD_CODE_SLOTS = 8;
constexpr int MXD_T_BYTES = 128 * 128, MXD_W_BYTES = BM * BK * 2;
constexpr int MXD_CODE_BYTES = BK * BM / 2, MXD_CODE_SLOT = MXD_CODE_BYTES + MX_ATOM_BYTES;     // codes, and their atom of scales
constexpr int MXD_DECODERS = 4, MXD_TEAMS = 4;        // warps that decode a k-block, and teams of them that take turns
// A team waits for every MXD_TEAMS-th use of the rings, and a wait knows phases by their parity alone: a warp that waits for one
// has to have waited for the one before, on the same barrier.  So code slots, and the barriers that free the other slots, are
// multiples of the teams in number.
static_assert(MXD_CODE_SLOTS % MXD_TEAMS == 0, "a code slot belongs to one team");
constexpr int MXD_EMPTY = MXD_SLOTS * MXD_TEAMS;
constexpr int MXD_THREADS = 96 + MXD_TEAMS * MXD_DECODERS * 32 + TG_SETS * 128;
constexpr int MXD_SMEM = MXD_SLOTS * (MXD_T_BYTES + MXD_W_BYTES) + MXD_CODE_SLOTS * MXD_CODE_SLOT + 1024;

struct MxDgradParams {
  CUtensorMap tok[2][TG_BOXES];    // token rows of a segment, boxes of 64 elements x 32, 64, 96, 128 rows
  CUtensorMap codes, scales;       // 64-byte x 16-row boxes; atoms
  const int32_t* cu_seqlens;
  const int32_t* pads;
  int ngroups, total_rows, N, K;   // K: weight rows a segment multiplies
  int nseg;                        // 2: a packed pair, gate rows first
  int w_rows;                      // stored rows of a group
  int row_atoms;                   // of a group's scales
  void* out;                       // bf16, or fp32 (F32)
  long long ldc;
  int vec_out;
  int32_t* status;
  unsigned long long timeout_ns;
};

// The bf16 values of eight codes with one scale, exactly (the smallest is 2^-128): word i holds those of codes i and i + 4, an
// order that costs no more than to move bits (in the codes' own order a byte's two halves go different ways).  A code's sign and its
// exponent and mantissa are put where bf16 has its own, by a product with two bits set; the exponent then lacks 126, 0.5 is a
// subnormal number in either format, and one bf16 product makes up for that and applies the scale: 2^126 2^(byte - 127).  Bytes
// from 128 on need more than bf16's exponents hold and take a second one (BIG).  The logical instructions bound the decoding
// (half the rate of products), which is why shifts are products here.  (By conversions, two codes an instruction: 177 us for
// 2 x 768 -> 2048; bytes looked up as in ep_mx_dequant_kernel: 186.)
// scale: the byte, twice, in the words' halves.
template <bool BIG>
__device__ __forceinline__ uint4 mx_values8(uint32_t codes, uint32_t scale) {
  auto pair = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
  constexpr uint32_t LOW = 0x000F000Fu, HIGH = 0x00F000F0u, KEEP = 0x81C081C0u;
  const uint32_t rest = codes >> 8;
  const uint32_t w[4] = {(codes & LOW) * 0x1040u & KEEP, (codes & HIGH) * 0x104u & KEEP, (rest & LOW) * 0x1040u & KEEP,
                         (rest & HIGH) * 0x104u & KEEP};
  alignas(16) __nv_bfloat162 v[4];
  const uint32_t b = scale & 255u;
  const __nv_bfloat162 factor = pair(BIG ? (min(b, 128u) + 126u) * 0x00800080u : scale * 128u + 0x3F003F00u);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __hmul2(pair(w[i]), factor);
  if constexpr (BIG) {
    const __nv_bfloat162 more = pair((b == 255u ? 0x7FC0u : (max(b, 128u) - 1u) << 7) * 0x00010001u);       // (255: NaN)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __hmul2(v[i], more);
  }
  return *reinterpret_cast<const uint4*>(v);
}
// Where the value at position i of eight stands in that order, and eight bf16 in it back in their own.
__device__ __forceinline__ int mx_column(int i) { return (i & 1) * 4 + (i >> 1); }
__device__ __forceinline__ uint4 mx_in_order(uint4 q) {
  return make_uint4(__byte_perm(q.x, q.y, 0x5410), __byte_perm(q.z, q.w, 0x5410), __byte_perm(q.x, q.y, 0x7632),
                    __byte_perm(q.z, q.w, 0x7632));
}

template <bool F32>
__global__ void __launch_bounds__(MXD_THREADS, 1)
ep_mx_dgrad_kernel(const __grid_constant__ MxDgradParams p) {
  constexpr int NST = MXD_SLOTS, NC = MXD_CODE_SLOTS;
  const int crank = (int)cluster_cta_rank();
  const int work_id0 = (int)(blockIdx.x >> 1), work_stride = (int)(gridDim.x >> 1);
  extern __shared__ uint8_t smem_dyn[];
  __shared__ __align__(8) uint64_t t_full[NST], w_full[NST], empty[MXD_EMPTY];   // (k-block n frees its slot at empty[n % MXD_EMPTY])
  __shared__ __align__(8) uint64_t c_full[NC], c_empty[NC];
  __shared__ __align__(8) uint64_t acc_full[2], acc_empty[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ int s_end[MAX_GROUPS], s_valid[MAX_GROUPS];
  __shared__ int s_prefix[MAX_GROUPS + 1];
  __shared__ __align__(128) uint8_t s_stage[TG_SETS][F32 ? 16 : TG_CHUNK * TG_STAGE_ROW];

  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  uint8_t* t_slots = (uint8_t*)(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
  uint8_t* w_slots = t_slots + NST * MXD_T_BYTES;
  uint8_t* c_slots = w_slots + NST * MXD_W_BYTES;
  volatile int* abortp = &s_abort;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < NST; ++s) { mbar_init(&t_full[s], 1); mbar_init(&w_full[s], 2 * MXD_DECODERS); }
    for (int s = 0; s < MXD_EMPTY; ++s) mbar_init(&empty[s], 1);
    for (int s = 0; s < NC; ++s) { mbar_init(&c_full[s], 1); mbar_init(&c_empty[s], MXD_DECODERS); }
    for (int a = 0; a < 2; ++a) { mbar_init(&acc_full[a], 1); mbar_init(&acc_empty[a], 8 * TG_SETS); }
    mbar_fence_init();
    s_abort = 0;
  }
  if (warp == 1) { tmem_alloc2(&s_tmem, 512); tmem_relinquish2(); }
  pdl_wait();
  for (int g = tid; g < p.ngroups; g += MXD_THREADS) {
    auto clamped = [&](int end) { return min(max(end, 0), p.total_rows); };
    const int start = g == 0 || p.cu_seqlens == nullptr ? 0 : clamped(p.cu_seqlens[g - 1]);
    const int end = clamped(p.cu_seqlens != nullptr ? p.cu_seqlens[g] : p.total_rows);
    s_end[g] = end;
    const int tokens = end > start ? group_tokens(p, g, start, end) : 0;
    s_valid[g] = end > start && tokens == 0 ? -1 : tokens;       // (-1: nothing but padding, a tile that writes the zeros)
  }
  __syncthreads();
  if (warp == 0) {      // exclusive prefix of token tiles per group
    int run = 0;
    for (int g0 = 0; g0 < p.ngroups; g0 += 32) {
      const int g = g0 + lane;
      const int nt = g < p.ngroups ? token_tiles(abs(s_valid[g])) : 0;
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

  const int m_tiles = (p.N + 255) / 256;
  const long long total_tiles = (long long)s_prefix[p.ngroups] * m_tiles;
  // Tile `id`, for a whole warp; ids only grow, and g is where the warp's last tile was.
  auto get = [&](long long id, int& g) {
    while (true) {
      const int i = g + 1 + lane;
      const uint32_t beyond = __ballot_sync(0xffffffffu, i >= p.ngroups || (long long)s_prefix[i] * m_tiles > id);
      if (beyond != 0u) { g += __ffs(beyond) - 1; break; }
      g += 32;
    }
    TokenTile t;
    t.g = g;
    const int nt = s_prefix[g + 1] - s_prefix[g];
    const int local = (int)(id - (long long)s_prefix[g] * m_tiles);
    const int mi = local / nt, ti = local - mi * nt;       // tiles that share weights are neighbours
    const int start = g == 0 ? 0 : s_end[g - 1], end = s_end[g];
    t.n = ((abs(s_valid[g]) + nt - 1) / nt + 31) & ~31;
    t.row0 = start + ti * t.n;
    t.rows = max(0, min(t.n, start + max(s_valid[g], 0) - t.row0));      // (the padding rows of its last 32 are computed, not stored)
    t.zero_to = ti == nt - 1 ? end : 0;
    t.m0 = mi * 256;
    t.alloc = t.g_local = 0;
    return t;
  };
  const int kb_per_seg = (p.K + BK - 1) / BK, num_kb = p.nseg * kb_per_seg;
  auto warp_wait = [&](uint64_t* bar, uint32_t parity, int where) {
    return __all_sync(0xffffffffu, gemm_wait(bar, parity, abortp, p, where)) != 0;
  };
  auto uniform = [&](int v) { return __shfl_sync(0xffffffffu, v, 0); };
  // First stored row of the 16 that hold weight rows k .. k + 15 (k a multiple of 16) of a segment.
  auto stored_row = [&](int seg, int k) { return p.nseg == 1 ? k : 2 * k + 16 * seg; };

  // The barrier of the k-block a ring's turn before: the first turn waits for nothing.
  RingSlot first_free;
  first_free.slot = MXD_EMPTY - NST;

  if (warp == 0) {
    // ================= TMA producer: tokens =================
    const bool issue = elect_one();
    int at = 0;
    RingSlot st, free = first_free;
    bool ok = true;
    for (long long id = work_id0; id < total_tiles && ok; id += work_stride) {
      const TokenTile t = get(id, at);
      const int n = uniform(t.n), trow = uniform(t.row0) + crank * (n / 2), box = (n / 2 + 31) / 32;
      const uint32_t bytes = 2u * (uint32_t)(box * 32 * 128);
      for (int seg = 0; seg < p.nseg && ok; ++seg)
        for (int kb = 0; kb < kb_per_seg; ++kb, st.next(NST), free.next(MXD_EMPTY)) {
          ok = warp_wait(&empty[free.slot], free.parity ^ 1u, 1);
          if (!ok) break;
          if (issue) {
            if (crank == 0) mbar_expect_tx(&t_full[st.slot], bytes);
            tma_load_2d_pair(t_slots + st.slot * MXD_T_BYTES, &p.tok[seg][box - 1], kb * BK, trow, mapa_u32(&t_full[st.slot], 0));
          }
        }
    }
  } else if (warp == 2) {
    // ================= TMA producer: codes =================
    const bool issue = elect_one();
    int at = 0;
    RingSlot ct;
    bool ok = true;
    for (long long id = work_id0; id < total_tiles && ok; id += work_stride) {
      const TokenTile t = get(id, at);
      const int g = uniform(t.g), m0 = uniform(t.m0);
      for (int seg = 0; seg < p.nseg && ok; ++seg)
        for (int kb = 0; kb < kb_per_seg; ++kb, ct.next(NC)) {
          ok = warp_wait(&c_empty[ct.slot], ct.parity ^ 1u, 5);
          if (!ok) break;
          if (issue) {
            uint8_t* dst = c_slots + ct.slot * MXD_CODE_SLOT;
            mbar_expect_tx(&c_full[ct.slot], MXD_CODE_SLOT);
#pragma unroll
            for (int j = 0; j < BK / 16; ++j)
              tma_load_2d(dst + j * 16 * 64, &p.codes, m0 / 2 + 64 * crank, g * p.w_rows + stored_row(seg, kb * BK + 16 * j),
                          &c_full[ct.slot]);
            tma_load_2d(dst + MXD_CODE_BYTES, &p.scales, (m0 / 128 + crank) * 128, g * p.row_atoms + (stored_row(seg, kb * BK) >> 7),
                        &c_full[ct.slot]);
          }
        }
    }
  } else if (warp == 1) {
    // ================= MMA issuer (the leader issues for both CTAs of the pair) =================
    if (crank == 0) {
      const bool issue = elect_one();
      const uint64_t desc_w = make_smem_desc(smem_u32(w_slots), 8192, 1024), desc_t = make_smem_desc(smem_u32(t_slots), 16, 1024);
      RingSlot st;
      int used = 0, tile_n = 0, at = 0;
      bool ok = true;
      for (long long id = work_id0; id < total_tiles && ok; id += work_stride, ++tile_n) {
        const uint32_t idesc = make_instr_desc_bf16(256, uniform(get(id, at).n), true, false);
        const int acc = tile_n & 1;
        if (!warp_wait(&acc_empty[acc], ((uint32_t)(tile_n >> 1) & 1u) ^ 1u, 2)) break;
        tc_fence_after();
        const uint32_t tacc = tmem_base + (uint32_t)acc * TG_MAX_N;
        uint32_t add = 0u;
        for (int kb = 0; kb < num_kb; ++kb, st.next(NST), used = used + 1 == MXD_EMPTY ? 0 : used + 1) {
          ok = warp_wait(&t_full[st.slot], st.parity, 3) && warp_wait(&w_full[st.slot], st.parity, 6);
          if (!ok) break;
          tc_fence_after();
          if (issue) {
            const uint64_t da = desc_w + (uint32_t)(st.slot * (MXD_W_BYTES >> 4)), db = desc_t + (uint32_t)(st.slot * (MXD_T_BYTES >> 4));
            umma_bf16_2cta(tacc, da, db, idesc, add);
#pragma unroll
            for (int kk = 1; kk < BK / 16; ++kk) umma_bf16_2cta(tacc, da + kk * 128, db + kk * 2, idesc, 1u);
            umma_commit_2cta(&empty[used], 3);
          }
          add = 1u;
        }
        if (!ok) break;
        if (issue) umma_commit_2cta(&acc_full[acc], 3);
      }
    }
  } else if (warp < 3 + MXD_TEAMS * MXD_DECODERS) {
    // ================= decode: 16 rows of the k-block a warp, in steps of four rows x 64 columns =================
    const int team = (warp - 3) / MXD_DECODERS, dw = (warp - 3) % MXD_DECODERS, chunk = lane & 7, sub = lane >> 3;
    const uint32_t scale_bytes = 0x4040u + 0x0101u * (uint32_t)(chunk >> 2);
    RingSlot st, ct, free = first_free;
    for (int i = 0; i < team; ++i) { st.next(NST); ct.next(NC); free.next(MXD_EMPTY); }
    int kb = team;
    bool ok = true;
    for (long long id = work_id0; id < total_tiles && ok; id += work_stride, kb -= num_kb) {
      for (; kb < num_kb; kb += MXD_TEAMS) {
        const int seg = kb >= kb_per_seg ? 1 : 0, k = (kb - seg * kb_per_seg) * BK + 16 * dw;
        ok = warp_wait(&c_full[ct.slot], ct.parity, 7) && warp_wait(&empty[free.slot], free.parity ^ 1u, 8);
        if (!ok) break;
        const uint8_t* src = c_slots + ct.slot * MXD_CODE_SLOT;
        uint8_t* dst = w_slots + st.slot * MXD_W_BYTES + (16 * dw + sub) * 128;
        uint32_t code[8], sc[4];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          code[i] = *reinterpret_cast<const uint32_t*>(src + (16 * dw + sub + (i >> 1) * 4) * 64 + (i & 1) * 32 + chunk * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {        // the four scales of this lane's rows
          const int r = stored_row(seg, k) + 4 * j + sub;
          sc[j] = *reinterpret_cast<const uint32_t*>(src + MXD_CODE_BYTES + (r & 31) * 16 + ((r >> 5) & 3) * 4);
        }
        if (k + 16 > p.K) {        // rows behind the reduction's end: zeros, with a scale of 1
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (k + 4 * j + sub >= p.K) { sc[j] = 0x7F7F7F7Fu; code[2 * j] = code[2 * j + 1] = 0u; }
        }
        auto decode = [&](auto big) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {        // rows 4 (i / 2) + sub, columns 64 (i % 2) + 8 chunk
            const int j = i >> 1, b = i & 1, row = 4 * j + sub;
            *reinterpret_cast<uint4*>(dst + b * 8192 + j * 4 * 128 + ((chunk ^ ((16 * dw + row) & 7)) << 4)) =
                mx_values8<decltype(big)::value>(code[i], __byte_perm(sc[j], 0u, scale_bytes + 0x0202 * b));
          }
        };
        if (((sc[0] | sc[1] | sc[2] | sc[3]) & 0x80808080u) == 0u) decode(std::false_type{});
        else decode(std::true_type{});
        // The fence has this CTA's stores in its shared memory, where its own tensor core reads them, before the arrival leaves;
        // what the leader learns of is an order, it reads none of these bytes itself.  (A release at cluster scope by a thread
        // that does nothing else, acquired by the issuer, takes some 1500 cycles a k-block: 2 x 768 -> 2048 of 128 groups of 256
        // rows 141 us, 381; 32 x 1024 rows, 2 x 2048 -> 7168 1261 - 1376, 3100.)
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&c_empty[ct.slot]);
          if (crank == 0) mbar_arrive(&w_full[st.slot]);
          else mbar_arrive_remote(&w_full[st.slot], 0);
        }
#pragma unroll
        for (int i = 0; i < MXD_TEAMS; ++i) { st.next(NST); ct.next(NC); free.next(MXD_EMPTY); }
      }
    }
  } else {
    // ========= epilogue: two sets of four warps, each warp one quarter of the tile's columns =========
    const int ew = warp - 3 - MXD_TEAMS * MXD_DECODERS, q = warp & 3, set = ew >> 2;
    const int te = (ew & 3) * 32 + lane;                    // 0..127
    const int first = set * TG_CHUNK, step = TG_SETS * TG_CHUNK;
    int tile_n = 0, at = 0;
    uint8_t* const sb = s_stage[set];
    const uint32_t st_addr = smem_u32(sb) + (uint32_t)((8 * (lane >> 4) + (lane & 7)) * TG_STAGE_ROW + q * 64 + ((lane >> 3) & 1) * 16);
    const bool vec_ok = p.vec_out != 0;
    for (long long id = work_id0; id < total_tiles; id += work_stride, ++tile_n) {
      const TokenTile t = get(id, at);
      const int acc = tile_n & 1;
      const bool have = gemm_wait(&acc_full[acc], (uint32_t)(tile_n >> 1) & 1u, abortp, p, 4);
      __syncwarp();
      if (!epilogue_all(set, have)) break;
      tc_fence_after();
      const uint32_t tacc = tmem_base + (uint32_t)acc * TG_MAX_N + ((uint32_t)(q * 32) << 16);
      uint32_t r[32];
      auto release_acc = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (crank != 0) mbar_arrive_remote(&acc_empty[acc], 0);
          else mbar_arrive(&acc_empty[acc]);
        }
      };
      if constexpr (F32) {
        // thread = output column: a warp's 32 columns of a token leave as one 128-byte line
        const int col = t.m0 + 128 * crank + q * 32 + (lane & 24) + mx_column(lane & 7);
#pragma unroll 1
        for (int c = first; c < t.n; c += step) {
          __syncwarp();
          tmem_ld_32x32(tacc + c, r);
          tmem_ld_wait();
          if (c + step >= t.n) release_acc();
          float* o = (float*)p.out + (long long)(t.row0 + c) * p.ldc + col;
#pragma unroll
          for (int i = 0; i < TG_CHUNK; ++i)
            if (c + i < t.rows && col < p.N) o[i * p.ldc] = __uint_as_float(r[i]);
        }
        if (first >= t.n) release_acc();
      } else {
        __nv_bfloat16* const out = (__nv_bfloat16*)p.out;
        if (first < t.n) {
          tmem_ld_16x256_x4(tacc + first, r);
          tmem_ld_16x256_x4(tacc + first + (16u << 16), r + 16);
        } else {
          release_acc();
        }
#pragma unroll 1
        for (int c = first; c < t.n; c += step) {
          __syncwarp();
          tmem_ld_wait();
          uint32_t pk[16];       // [16-column half][token block][lower, upper 8 columns]
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
            pk[i] = *reinterpret_cast<const uint32_t*>(&h);
          }
          if (c + step < t.n) {            // the next 32 tokens travel while these leave
            tmem_ld_16x256_x4(tacc + c + step, r);
            tmem_ld_16x256_x4(tacc + c + step + (16u << 16), r + 16);
          } else {
            release_acc();
          }
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; j += 2)
              stmatrix_x4_trans(st_addr + (uint32_t)(j * 8 * TG_STAGE_ROW + h * 32),
                                pk[8 * h + 2 * j], pk[8 * h + 2 * j + 1], pk[8 * h + 2 * j + 2], pk[8 * h + 2 * j + 3]);
          __syncwarp();
          epilogue_sync(set);
          const int f = (te & 15) * 8, col0 = t.m0 + 128 * crank + f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = (te >> 4) + 8 * i;
            if (c + k >= t.rows || col0 >= p.N) continue;
            store8(out + (long long)(t.row0 + c + k) * p.ldc + col0,
                   mx_in_order(*reinterpret_cast<const uint4*>(sb + k * TG_STAGE_ROW + f * 2)), p.N - col0, vec_ok);
          }
          epilogue_sync(set);              // every row of the set's buffer has been read: it may be filled again
        }
        {      // padding rows that no tile computes
          const int f = (te & 15) * 8, col0 = t.m0 + 128 * crank + f;
          if (col0 < p.N)
            for (int row = t.row0 + t.rows + (te + 128 * set) / 16; row < t.zero_to; row += 128 * TG_SETS / 16)
              store8(out + (long long)row * p.ldc + col0, make_uint4(0, 0, 0, 0), p.N - col0, vec_ok);
        }
      }
    }
    if constexpr (!F32) {      // rows behind the last group
      const int warps = 4 * TG_SETS;
      for (int row = s_end[p.ngroups - 1] + (int)blockIdx.x * warps + ew; row < p.total_rows; row += (int)gridDim.x * warps)
        for (int c = lane * 8; c < p.N; c += 256)
          store8((__nv_bfloat16*)p.out + (long long)row * p.ldc + c, make_uint4(0, 0, 0, 0), p.N - c, vec_ok);
    }
  }
  pdl_launch_dependents();
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

}  // namespace mep
