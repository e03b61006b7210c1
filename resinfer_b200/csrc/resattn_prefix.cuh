// ResAttn decode for a batch that shares a prefix: the prefix part.  Included by resattn.cu behind resattn_pv.cuh, inside
// namespace ri::<anon>::tcattn.
//
// All query heads of all sequences that read one KV head are rows of one problem, R = batch x group rows against the
// prefix's tokens, so the prefix crosses HBM once instead of once per sequence.  A CTA (one per SM) takes a tile of 128
// rows, one KV head and a range of the prefix (its split) in steps of 128 tokens (head_dim 256: 64):
//
//   S[128 rows x step]  = Qbase . K^T + Qres . K^T   tcgen05.mma kind::mxf4nvf4.block_scale, codes and E4M3 scales as stored
//   P = 2^(S scale - m)                              one row per softmax thread, rounded to FP16
//   O[128 rows x D]    += P . V                      tcgen05.mma kind::f16, P from tensor memory, V expanded to FP16 (exact)
//
// and leaves the unnormalised partial (o, l, m) of its rows; the launch behind it (resattn_tail_kernel: the sequences' own
// tokens) adds the partials of all splits.  The statistics m, l and the accumulator o stay in FP32; the maximum of a row is
// only raised when a score exceeds it by more than 2^8, so o is rarely rescaled.  FP16 holds the code x block scale products
// exactly and P with 11 bits.
//
// Rows shorter than the prefix are masked at their own length; rows beyond the batch have length zero.  What no row of the
// tile attends to may be unwritten: its scores are masked and its V is taken as zeros.
//
// What bounds it: the special function unit, 16 exponentials a cycle and SM -- 1024 cycles for 128 x 128 scores, against
// 512 + 256 for the two products -- and, close behind, issue slots and the latencies of the chain scores -> P -> product.
// So the two softmax groups run free of each other: a group takes a step's exponentials with the maximum that it knows,
// raised where the step itself shows a row grown beyond 2^8 times it; what the other group raised meanwhile is seen once the
// products of the step in front are complete, and P is then scaled by the difference -- exactly down to FP16's smallest
// normal number, maxima being whole powers of two; below it a P of at most 2^-14 loses last bits.  (Waiting for the other group's maximum first, or taking turns at the exponentials, cost more than it hid; so did a
// polynomial in the place of an eighth, a quarter or half of the exponentials: 128 steps 121, 139, 146 us against 119.)
// Measured (differences of two lengths, back to back, 1.93 GHz): a step of 128 x 128 0.89 us with pages of 128 tokens, 1720
// cycles, the special function unit busy for 59 % and the tensor cores for 43 to 50 %; 0.93 us with pages of 32, 0.96 with
// pages of 16; head_dim 256 (128 x 64) 0.86.  Before the first step 4 us (the query's codes 2), behind the last 3.  64
// sequences of 64 heads over 8 behind 32768 tokens and no further ones, in four pieces on 128 SMs: 69 us with the launch that
// merges, 0.99 PFLOP/s of the two products.
//
// Roles (16 warps):
//   0-3, 4-7   softmax, thread = row (tensor-memory lane); the first group takes the even steps, the second the odd ones
//   8-11       V conversion: codes x scales -> FP16 in the 128-byte-swizzled N-major operand layout
//   12, 13     one thread each issues the scores' and the P.V products; warp 12 lays K's scales out for them
//   14, 15     copies of codes (tiled TMA in the operand swizzle) and of scales (bulk), one lane per run of tokens that lie
//              together in a page.  Small copies are what pages of 16 and 32 tokens cost: with V among them, all from one warp, a
//              step took 1.8 us, from two warps 1.17; there the conversion warps load V themselves (0.96).
// Every wait is bounded.  A role whose wait expires sets the abort flag and leaves its loop (the scores': issues nothing more),
// the others follow at their next wait that is not over, and none begins a copy or a product after that.  What is in flight
// then is waited for whatever the flag says (px_drain): the products by a commit of their own, the copies by the barriers
// that count their bytes.  So all roles meet at the end, nothing outlives the CTA, and the status word is set.
template <int D>
struct PxCfg {
  static constexpr int kStep = D == 128 ? 128 : 64;            // tokens per step
  static constexpr int kRows = 128;
  static constexpr int kFirstConv = 8, kConv = 4, kQkWarp = 12, kPvWarp = 13, kProdWarp = 14;
  static constexpr int kThreads = 512;
  static constexpr int kStages = 4;
  static constexpr int kMma = D / 64;
  static constexpr int kRowBytes = D / 2;
  static constexpr int kSfPerRow = D / 16;
  static constexpr int kDBlocks = D / 64;
  // shared memory: Q codes and scales (base, residue), V tiles, stages
  static constexpr int kQBytes = kRows * kRowBytes;
  static constexpr int kQsfBytes = kMma * 512;
  static constexpr int kOffQsf = 2 * kQBytes;
  static constexpr int kOffV = kOffQsf + 2 * kQsfBytes;        // a multiple of 1024
  static constexpr int kVBytes = kStep * D * 2;
  static constexpr int kOffStage = kOffV + 2 * kVBytes;
  static constexpr int kKBytes = kStep * kRowBytes;
  static constexpr int kSfBytes = kStep * kSfPerRow;
  static constexpr int kStgV = kKBytes, kStgKsf = 2 * kKBytes, kStgKraw = kStgKsf + kMma * 512, kStgVsf = kStgKraw + kSfBytes;
  static constexpr int kStageBytes = (kStgVsf + kSfBytes + 1023) / 1024 * 1024;
  static constexpr int kSmemBytes = kOffStage + kStages * kStageBytes + 1024;
  // tensor memory columns: accumulator, scores (one buffer per softmax group), P, query scales, K scales (two sets)
  static constexpr int kColO = 0, kColS = D, kColP = kColS + 2 * kStep, kColSfq = kColP + kStep / 2, kColSfk = kColSfq + 8 * kMma;
  static constexpr int kTmemCols = 512;
  static_assert(kColSfk + 8 * kMma <= kTmemCols && kOffV % 1024 == 0, "layout");
};

// D[128 x N] += A[128 x 16, tensor memory] . B[16 x N, shared memory], FP16 operands
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// 32 lanes x 32 columns without waiting for the data (tmem_wait_ld below)
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// waits for this thread's loads; r is an operand so that nothing reads it earlier
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A wait that ends when the phase is complete (true), or when the kernel has given up (false, see above).  Short on purpose:
// there are a dozen of them in loops that run side by side.  With mbar_wait inside, 64 sequences behind 32768 tokens took
// 103.0 us instead of 101.1 before the roles looked at the results, and 106.6 instead of 102.4 since.
__device__ __forceinline__ bool px_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int site) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_hint(bar, parity, 20000u)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > kWaitLimitCycles) {
      *abort_flag = site;                                      // which wait gave up (reported in the status word)
      return false;
    }
  }
  return true;
}
// ... for all lanes of a warp alike
__device__ __forceinline__ bool px_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int site) {
  return __all_sync(0xffffffffu, px_wait(bar, parity, abort_flag, site));
}
// A wait for what is in flight at the end, bounded, but not cut short by the abort flag.
__device__ __forceinline__ void px_drain(uint32_t bar, uint32_t parity, volatile int* abort_flag, int site) {
  if (mbar_try(bar, parity)) return;
  const long long t0 = clock64();
  while (!mbar_try_hint(bar, parity, 20000u)) {
    if (clock64() - t0 > kWaitLimitCycles) {
      *abort_flag = site;
      return;
    }
  }
}

// two FP32 operations per instruction; a pair is (low, high) of a 64-bit register
__device__ __forceinline__ uint64_t pair64(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ void unpair64(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// NaN if one of them is.  The maxima of partials are joined so: a partial's m is -inf where it attends to nothing and holds
// no data, and NaN where it attends to scores of NaN alone, from which no maximum is found -- which has to reach the output
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// A block of the query as NVFP4 and the NVFP4 of what that leaves, global scale 1.  quant_mext16 takes the residue with a
// twice rounded reciprocal for the scale; here it is the scale itself, so that the residue is exact (a bf16 value minus
// code x scale fits FP32) and one that lies on a border between two codes, which bf16 values do often, goes to the even
// one.  Against attention over q + residues in 64 bits: 2.0e-3 with the reciprocal (single rows 2e-2), 2.5e-4 without.
// A NaN does not count for the block's magnitude and 16 of them have scale zero, there as here.
// (Products, differences and maxima in pairs: the prologue of 128 rows is bound by its instructions.)
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float absmax16(const float (&x)[16]) {
  float a = max3(fabsf(x[0]), fabsf(x[1]), fabsf(x[2])), b = max3(fabsf(x[3]), fabsf(x[4]), fabsf(x[5]));
  a = max3(a, fabsf(x[6]), fabsf(x[7]));
  b = max3(b, fabsf(x[8]), fabsf(x[9]));
  a = max3(a, fabsf(x[10]), fabsf(x[11]));
  b = max3(b, fabsf(x[12]), fabsf(x[13]));
  return max3(max3(a, b, 0.f), fabsf(x[14]), fabsf(x[15]));
}
__device__ __forceinline__ uint2 codes16(const float (&x)[16], float mult) {
  const uint64_t m2 = pair64(__float_as_uint(mult), __float_as_uint(mult));
  float lo[8], hi[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    unpair64(mul2(pair64(__float_as_uint(x[i]), __float_as_uint(x[i + 1])), m2), lo[i], lo[i + 1]);
    unpair64(mul2(pair64(__float_as_uint(x[8 + i]), __float_as_uint(x[9 + i])), m2), hi[i], hi[i + 1]);
  }
  return make_uint2(cvt_e2m1x8(lo), cvt_e2m1x8(hi));
}
__device__ __forceinline__ BlockQ quant_query16(const float (&x)[16]) {
  BlockQ q;
  q.base = codes16(x, nvfp4_scale(absmax16(x), 1.0f, &q.sf));
  const float s = decode_e4m3(q.sf);
  const uint64_t s2 = pair64(__float_as_uint(-s), __float_as_uint(-s));
  float r[16], hat[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    e2m1x8_to_float(h ? q.base.y : q.base.x, hat);             // by shifts: see expand8_packed in resattn_tail.cuh
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      unpair64(fma2(pair64(__float_as_uint(hat[i]), __float_as_uint(hat[i + 1])), s2, pair64(__float_as_uint(x[8 * h + i]), __float_as_uint(x[8 * h + i + 1]))),
               r[8 * h + i], r[8 * h + i + 1]);
  }
  q.res = codes16(r, nvfp4_scale(absmax16(r), 1.0f, &q.sf_res));
  return q;
}

// VDIRECT: the conversion warps load V's codes and scales from the pool into registers, a step ahead, instead of from the stages
template <int D, bool VDIRECT>
__global__ void __launch_bounds__(PxCfg<D>::kThreads, 1) resattn_prefix_kernel(const __grid_constant__ CUtensorMap k_map,
                                                                                  const __grid_constant__ CUtensorMap v_map,
                                                                                  const __grid_constant__ AttnParams p, int run) {
  using C = PxCfg<D>;
  constexpr int S = C::kStages, kStep = C::kStep;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[S], bar_empty[S];
  __shared__ __align__(8) uint64_t bar_sfull[2], bar_sfree[2], bar_pready[2], bar_pvdone[2], bar_vready[2], bar_vfree[2];
  __shared__ __align__(8) uint64_t bar_end[2];                 // all scores' products have ended, all P.V products
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  __shared__ volatile int copied[2];                           // steps whose codes (scales) have been asked for
  __shared__ float row_m[C::kRows], row_l[C::kRows];           // running maxima; row sums of the second group
  __shared__ int nan_from[C::kSfPerRow];                       // the first token whose V has a NaN scale in a block, INT_MAX without one
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x, hkv = blockIdx.y % p.hkv, row0 = (blockIdx.y / p.hkv) * C::kRows;
  const int G = p.group, rows = p.batch * G;

  // Everything this kernel reads was written before the launch in front of it ended, and the launch behind it may start
  // only now: it therefore may read the same inputs without a wait of its own (it waits before it reads the partials).
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int n_steps = (p.prefix_len + kStep - 1) / kStep;
  const int s_begin = min(split * p.steps_per_split, n_steps);
  const int steps = min(s_begin + p.steps_per_split, n_steps) - s_begin;

  if (split == 0 && blockIdx.y == 0 && p.splits > 1)           // tickets of the launch behind this one
    for (int i = threadIdx.x; i < p.batch * p.hkv; i += blockDim.x) p.split_counter[i] = 0;

  if (steps <= 0) {                                            // more pieces than steps: empty partials, and nothing is begun
    const int row = row0 + threadIdx.x;
    if (threadIdx.x < C::kRows && row < rows) {
      const int64_t slot = (int64_t(p.splits + split) * p.batch + row / G) * p.hq + hkv * G + row % G;
      p.l_part[slot] = 0.f;
      p.m_part[slot] = -INFINITY;
    }
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 2);                    // codes, scales
      mbar_init(smem_u32(&bar_empty[s]), VDIRECT ? 1 : C::kConv + 1); // conversion warps + the commit of the scores' MMAs
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&bar_sfull[s]), 1);
      mbar_init(smem_u32(&bar_sfree[s]), 4);
      mbar_init(smem_u32(&bar_pready[s]), 4);
      mbar_init(smem_u32(&bar_pvdone[s]), 1);
      mbar_init(smem_u32(&bar_vready[s]), C::kConv);
      mbar_init(smem_u32(&bar_vfree[s]), 1);
      mbar_init(smem_u32(&bar_end[s]), 1);
    }
    abort_flag = 0;
#pragma unroll
    for (int i = 0; i < C::kSfPerRow; ++i) nan_from[i] = 0x7fffffff;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == C::kQkWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_slot)), "r"(C::kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  __syncthreads();                                             // the barriers exist: the copies may begin
  uint8_t* stage0 = smem + C::kOffStage;
  // test: the first CTA's `role` gives up in front of a step
  auto last_step = [&](int role) {
    const int step = p.expire - (role << 26);
    return step >= 0 && step < steps && blockIdx.x == 0 && blockIdx.y == 0 ? step : steps;
  };
  int longest = 0;                                             // V conversion: of the lengths of the tile's sequences, two per lane
  if (warp >= C::kFirstConv && warp < C::kQkWarp) {
    static_assert(C::kRows / 4 + 1 <= 64, "groups of four heads and more");
    const int b0 = row0 / G + lane, b_end = (min(row0 + C::kRows, rows) - 1) / G + 1;
    if (b0 < b_end) longest = __ldg(p.seq_lens + b0);
    if (b0 + 32 < b_end) longest = max(longest, __ldg(p.seq_lens + b0 + 32));
  }
  if (warp < C::kProdWarp) {
    // -------------------------------------------------------------- query prologue: NVFP4 and its NVFP4 residue
    constexpr int kThr = C::kProdWarp * 32, kBlocks = C::kRows * C::kSfPerRow, kIt = (kBlocks + kThr - 1) / kThr;
    uint4 x[kIt][2];                                           // a block of 16 values each; all loads in flight together
#pragma unroll
    for (int it = 0; it < kIt; ++it) {
      const int i = threadIdx.x + it * kThr, row = row0 + i / C::kSfPerRow;
      x[it][0] = x[it][1] = make_uint4(0, 0, 0, 0);
      if (i < kBlocks && row < rows) {
        const int b = row / G, g = row - b * G;
        const uint4* src = reinterpret_cast<const uint4*>(p.q + (int64_t(b) * p.hq + hkv * G + g) * D + (i % C::kSfPerRow) * 16);
        x[it][0] = __ldg(src);
        x[it][1] = __ldg(src + 1);
      }
    }
#pragma unroll 1
    for (int it = 0; it < kIt; ++it) {
      const int i = threadIdx.x + it * kThr;
      if (i >= kBlocks) break;
      const int r = i / C::kSfPerRow, blk = i % C::kSfPerRow;
      uint4 lo = x[0][0], hi = x[0][1];
#pragma unroll
      for (int k = 1; k < kIt; ++k)
        if (it == k) lo = x[k][0], hi = x[k][1];
      const uint32_t u[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      float v[16];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[2 * k] = __uint_as_float(u[k] << 16);
        v[2 * k + 1] = __uint_as_float(u[k] & 0xFFFF0000u);
      }
      BlockQ bq{};                                             // rows behind the batch: zero
      if (row0 + r < rows) bq = quant_query16(v);
      const uint32_t off = swz_off<D>(r, blk * 8);
      *reinterpret_cast<uint2*>(smem + off) = bq.base;
      *reinterpret_cast<uint2*>(smem + C::kQBytes + off) = bq.res;
      const uint32_t so = C::kOffQsf + (blk >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (blk & 3);
      smem[so] = bq.sf;
      smem[so + C::kQsfBytes] = bq.sf_res;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    asm volatile("bar.sync 15, %0;" ::"n"(kThr) : "memory");
    tc_fence_after();
  }
  const uint32_t tmem_base = tmem_slot;

  if (warp < C::kFirstConv) {
    // ============================================================ softmax warps
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const int grp = warp >> 2, quarter = warp & 3;
    const uint32_t lane_base = tmem_base + (uint32_t(quarter * 32) << 16);
    const uint32_t s_col = lane_base + C::kColS + grp * kStep;
    const uint32_t b_sfull = smem_u32(&bar_sfull[grp]), b_sfree = smem_u32(&bar_sfree[grp]), b_pready = smem_u32(&bar_pready[grp]);
    const uint32_t b_pvdone = smem_u32(&bar_pvdone[grp ^ 1]);  // of the steps of the other group, in front of this group's
    const int r = quarter * 32 + lane, row = row0 + r;
    int lim = 0;
    if (row < rows) lim = min(max(__ldg(p.seq_lens + row / G), 0), p.prefix_len);
    const int lim_max = __reduce_max_sync(0xffffffffu, lim);
    const float scale = p.score_scale_log2;
    float m = -INFINITY, l = 0.f;                              // this group's: the row's maximum as it last knew it, its row sum
    if (grp == 0) row_m[r] = -INFINITY;                        // steps in which no lane's maximum moves leave it so
    if (lim_max <= s_begin * kStep) {
      // none of these rows reaches the split's tokens: their P is zero throughout
      if (grp == 0) {
        uint32_t z[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) z[i] = 0;
#pragma unroll
        for (int c = 0; c < kStep / 2; c += 32) tmem_st32(lane_base + C::kColP + c, z);
        tmem_wait_st();
        tc_fence_before();
      }
      for (int j = grp, k = 0; j < steps; j += 2, ++k) {
        if (!px_wait_warp(b_sfull, k & 1, &abort_flag, 5)) break;
        if (j > 0 && !px_wait_warp(b_pvdone, ((j - 1) >> 1) & 1, &abort_flag, 7)) break;
        if (lane == 0) {
          mbar_arrive(b_sfree);
          mbar_arrive(b_pready);
        }
      }
    } else {
      for (int j = grp, k = 0; j < steps; j += 2, ++k) {
        const int left = lim - (s_begin + j) * kStep;          // of this row's tokens, from this step on
        if (!px_wait_warp(b_sfull, k & 1, &abort_flag, 5)) break;
        tc_fence_after();
        if (__any_sync(0xffffffffu, left < kStep)) {           // a row ends here: its scores beyond are -inf
#pragma unroll 1
          for (int c = 0; c < kStep; c += 16) {
            float t[16];
            tmem_ld16(s_col + c, t);
#pragma unroll
            for (int i = 0; i < 16; ++i) t[i] = c + i < left ? t[i] : -INFINITY;
            tmem_st16f(s_col + c, t);
          }
          tmem_wait_st();
        }
        uint32_t s[kStep / 32][32];
#pragma unroll
        for (int c = 0; c < kStep / 32; ++c) tmem_ld32_async(s_col + 32 * c, s[c]);
#pragma unroll
        for (int c = 0; c < kStep / 32; ++c) tmem_wait_ld(s[c]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(b_sfree);                   // step j+2's scores may overwrite S
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kStep; i += 2)
          m4[(i >> 1) & 3] = max3(m4[(i >> 1) & 3], __uint_as_float(s[i >> 5][i & 31]), __uint_as_float(s[i >> 5][(i & 31) + 1]));
        const float mx = max3(fmaxf(m4[0], m4[1]), m4[2], m4[3]) * scale;   // scale > 0
        const float m_try = mx > m + kLazyThreshold ? ceilf(mx) : m;
        const float mu = m_try == -INFINITY ? 0.f : m_try;     // a row with nothing to attend to yet
        const uint64_t scale2 = pair64(__float_as_uint(scale), __float_as_uint(scale));
        const uint64_t mu2 = pair64(__float_as_uint(-mu), __float_as_uint(-mu));
        uint64_t sum[2] = {0, 0};
        uint32_t pk[kStep / 2];
#pragma unroll
        for (int i = 0; i < kStep / 2; ++i) {
          float a, b;
          unpair64(fma2(pair64(s[i >> 4][(2 * i) & 31], s[i >> 4][(2 * i + 1) & 31]), scale2, mu2), a, b);
          a = fast_exp2(a);
          b = fast_exp2(b);
          sum[i & 1] = add2(sum[i & 1], pair64(__float_as_uint(a), __float_as_uint(b)));
          pk[i] = h2_bits(__floats2half2_rn(a, b));
        }
        float l_step;
        {
          float a, b;
          unpair64(add2(sum[0], sum[1]), a, b);
          l_step = a + b;
        }
        float before = -INFINITY;
        if (j > 0) {                                           // P is free, the accumulator and row_m those of step j-1
          if (!px_wait_warp(b_pvdone, ((j - 1) >> 1) & 1, &abort_flag, 7)) break;
          tc_fence_after();
          before = row_m[r];
        }
        if (__any_sync(0xffffffffu, m_try != before || m != before)) {   // a maximum has moved, here or in the other group
          const float now = mx > before + kLazyThreshold ? ceilf(mx) : before;
          const float f_o = before == -INFINITY ? 0.f : fast_exp2(before - now);
          const float f_p = m_try == -INFINITY ? 0.f : fast_exp2(m_try - now);   // powers of two, 1 at most 2^8
          l *= m == -INFINITY ? 0.f : fast_exp2(m - now);
          l_step *= f_p;
          const __half2 f2 = __float2half2_rn(f_p);
#pragma unroll
          for (int i = 0; i < kStep / 2; ++i) pk[i] = h2_bits(__hmul2(bits_h2(pk[i]), f2));
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              float o[16];
              tmem_ld16(lane_base + C::kColO + c, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= f_o;
              tmem_st16f(lane_base + C::kColO + c, o);
            }
          }
          m = now;
          row_m[r] = now;
        }
        l += l_step;
#pragma unroll
        for (int c = 0; c < kStep / 2; c += 32) tmem_st32(lane_base + C::kColP + c, pk + c);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(b_pready);
      }
    }
    // ---------------------------------------------------------------- the rows' partials: half of the columns per group
    px_wait(smem_u32(&bar_pvdone[(steps - 1) & 1]), ((steps - 1) >> 1) & 1, &abort_flag, 12);
    float m_end = lim_max > s_begin * kStep ? row_m[r] : -INFINITY;   // ordered by the products in between
    l = m == -INFINITY ? 0.f : l * fast_exp2(m - m_end);
    if (m_end == -INFINITY && lim > s_begin * kStep) m_end = __int_as_float(0x7fffffff);   // see max_nan
    if (grp == 1) row_l[r] = l;
    asm volatile("bar.sync %0, 64;" ::"r"(9 + quarter) : "memory");
    if (__any_sync(0xffffffffu, row < rows)) {                 // whole warps: the loads from tensor memory are collective
      const int b = row / G, g = row - b * G;
      const int64_t slot = (int64_t(p.splits + split) * p.batch + b) * p.hq + hkv * G + g;
      if (grp == 0 && row < rows) {
        p.l_part[slot] = m_end == -INFINITY ? 0.f : l + row_l[r];
        p.m_part[slot] = m_end;
      }
      if (__any_sync(0xffffffffu, row < rows && m_end != -INFINITY)) {
        tc_fence_after();
#pragma unroll 1
        for (int c = grp * (D / 2); c < (grp + 1) * (D / 2); c += 16) {
          float o[16];
          tmem_ld16(lane_base + C::kColO + c, o);
          if (row < rows) {
            if (lim > nan_from[c / 16])
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __int_as_float(0x7fffffff);
            float* dst = p.o_part + slot * D + c;              // 32-byte aligned: whole sectors
#pragma unroll
            for (int i = 0; i < 16; i += 8)
              asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                           ::"l"(dst + i), "f"(o[i]), "f"(o[i + 1]), "f"(o[i + 2]), "f"(o[i + 3]), "f"(o[i + 4]), "f"(o[i + 5]),
                             "f"(o[i + 6]), "f"(o[i + 7]) : "memory");
          }
        }
        tc_fence_before();
      }
    }
  } else if (warp < C::kQkWarp) {
    // ============================================================ V conversion warps: 32 tokens x 64 head-dim values each
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    const int cw = warp - C::kFirstConv;
    constexpr int kUnits = kStep / 32 * C::kDBlocks / C::kConv;   // 32 tokens x 64 values each, of the same tokens
    static_assert(kUnits == 2 && C::kDBlocks % 2 == 0, "64 bytes of codes a thread");
    const int tok = 32 * (cw * kUnits / C::kDBlocks) + lane, dblk0 = cw * kUnits % C::kDBlocks;
    // Tokens that none of the tile's rows attends to need not have been written: whatever lies there, V is 0 (0 x P = 0)
    const int v_len = min(__reduce_max_sync(0xffffffffu, longest), p.prefix_len);
    uint4 n0[kUnits], n1[kUnits];                              // VDIRECT: the next step's
    uint2 nsf = make_uint2(0, 0);
    int pages[3] = {};                                         // table entries of steps j + 1, j + 2, j + 3
    auto page_of = [&](int j) -> int {
      const int t = (s_begin + j) * kStep + tok;
      return j < steps && t < v_len ? __ldg(p.prefix_table + (p.page_shift >= 0 ? t >> p.page_shift : t / p.page_size)) : 0;
    };
    auto row_of = [&](int j, int entry) -> int64_t {           // the token's row: page, and row of the page
      const int t = (s_begin + j) * kStep + tok;
      return min(max(int64_t(entry), int64_t(0)), p.num_pages - 1) << 32 |
             uint32_t(hkv * p.page_size + (p.page_shift >= 0 ? (t & (p.page_size - 1)) : t % p.page_size));
    };
    auto codes_at = [&](int64_t row) { return p.v_data + (row >> 32) * p.code_page_stride + (row & 0xffffffff) * C::kRowBytes + dblk0 * 32; };
    auto scales_at = [&](int64_t row) { return p.v_sf + (row >> 32) * p.sf_page_stride + (row & 0xffffffff) * C::kSfPerRow + dblk0 * 4; };
    auto fetch_l2 = [&](int j, int entry) {                    // a step's latency does not cover the HBM's
      if (j < steps && (s_begin + j) * kStep + tok < v_len) {
        const int64_t row = row_of(j, entry);
        asm volatile("prefetch.global.L2 [%0];" ::"l"(codes_at(row)));
        asm volatile("prefetch.global.L2 [%0];" ::"l"(codes_at(row) + 32));
        asm volatile("prefetch.global.L2 [%0];" ::"l"(scales_at(row)));
      }
    };
    auto load = [&](int j, int entry) {
      const int t = (s_begin + j) * kStep + tok;
      nsf = make_uint2(0, 0);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) n0[u] = n1[u] = make_uint4(0, 0, 0, 0);
      if (j < steps && t < v_len) {
        const int64_t row = row_of(j, entry);
        const uint4* src = reinterpret_cast<const uint4*>(codes_at(row));
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          n0[u] = __ldg(src + 2 * u);
          n1[u] = __ldg(src + 2 * u + 1);
        }
        nsf = __ldg(reinterpret_cast<const uint2*>(scales_at(row)));
      }
    };
    // A NaN scale would reach every row of the tile, 0 x NaN, also those that end before its token: the block is taken as zeros,
    // and the rows that attend to it get their NaN at the end.  (Where it is looked for, and how much code that adds to the
    // loop, matters by 2 to 4 %: in front of the wait for the operand's buffer, and short, with scales that are in registers
    // already, behind it and unrolled with those from the stages.  So placed it costs nothing to 0.8 %.)
    constexpr int kNanUnroll = VDIRECT ? 1 : 4;
    auto has_nan = [](uint32_t scales) { return (((scales & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0; };
    auto take_out_nans = [&](uint32_t& scales, int j, int dblk) {
      const uint32_t nans = ((scales & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
#pragma unroll kNanUnroll
      for (int i = 0; i < 4; ++i)
        if (nans >> (8 * i + 7) & 1) atomicMin(&nan_from[dblk * 4 + i], (s_begin + j) * kStep + tok);
      scales &= ~((nans >> 7) * 0xFFu);
    };
    if constexpr (VDIRECT) {
      const int first = page_of(0);
#pragma unroll
      for (int k = 0; k < 3; ++k) pages[k] = page_of(k + 1);
      load(0, first);
      fetch_l2(1, pages[0]);
      fetch_l2(2, pages[1]);
    }
    for (int j = 0, stg = 0, ph = 0; j < steps; ++j, stg = (stg + 1 == S ? 0 : stg + 1), ph ^= (stg == 0)) {
      const int vb = j & 1;
      uint4 c0[kUnits], c1[kUnits];
      uint32_t sfw[kUnits];
      if constexpr (VDIRECT) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          c0[u] = n0[u];
          c1[u] = n1[u];
          sfw[u] = u ? nsf.y : nsf.x;
        }
        load(j + 1, pages[0]);
        fetch_l2(j + 3, pages[2]);
        pages[0] = pages[1];
        pages[1] = pages[2];
        pages[2] = page_of(j + 4);
      } else {
        if (!px_wait_warp(smem_u32(&bar_full[stg]), ph, &abort_flag, 6)) break;
        const uint8_t* st = stage0 + stg * C::kStageBytes;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          const int dblk = dblk0 + u;
          c0[u] = c1[u] = make_uint4(0, 0, 0, 0);
          sfw[u] = 0;
          if ((s_begin + j) * kStep + tok < v_len) {
            const uint8_t* src = st + C::kStgV;
            c0[u] = *reinterpret_cast<const uint4*>(src + swz_off<D>(tok, 32 * dblk));
            c1[u] = *reinterpret_cast<const uint4*>(src + swz_off<D>(tok, 32 * dblk + 16));
            sfw[u] = *reinterpret_cast<const uint32_t*>(st + C::kStgVsf + tok * C::kSfPerRow + dblk * 4);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_empty[stg])); // the codes are in registers: the stage may be refilled
      }
      if constexpr (VDIRECT) {
        if (has_nan(sfw[0]) | has_nan(sfw[1])) {
          take_out_nans(sfw[0], j, dblk0);
          take_out_nans(sfw[1], j, dblk0 + 1);
        }
      }
      if (j >= 2 && !px_wait_warp(smem_u32(&bar_vfree[vb]), ((j >> 1) - 1) & 1, &abort_flag, 11)) break;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int dblk = dblk0 + u;
        if constexpr (!VDIRECT)
          if (has_nan(sfw[u])) take_out_nans(sfw[u], j, dblk);
        const uint32_t words[8] = {c0[u].x, c0[u].y, c0[u].z, c0[u].w, c1[u].x, c1[u].y, c1[u].z, c1[u].w};
        uint32_t lo, hi, sc2[4];                               // the four block scales as FP16 pairs (s, s)
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi) : "r"(sfw[u]));
        sc2[0] = __byte_perm(lo, 0, 0x1010); sc2[1] = __byte_perm(lo, 0, 0x3232);
        sc2[2] = __byte_perm(hi, 0, 0x1010); sc2[3] = __byte_perm(hi, 0, 0x3232);
        const uint32_t dst0 = smem_u32(smem + C::kOffV + vb * C::kVBytes + dblk * (kStep * 128) + (tok >> 3) * 1024 + (tok & 7) * 128) |
                              ((tok & 7) << 4);
#pragma unroll
        for (int w8 = 0; w8 < 8; ++w8) {                       // one 16-byte chunk = 8 FP16 per code word
          uint32_t h0, h1, h2, h3;
          asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
              "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
              "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
              : "=r"(h0), "=r"(h1), "=r"(h2), "=r"(h3) : "r"(words[w8]));
          const __half2 s2 = bits_h2(sc2[w8 >> 1]);
          const uint32_t o0 = h2_bits(__hmul2(bits_h2(h0), s2)), o1 = h2_bits(__hmul2(bits_h2(h1), s2));
          const uint32_t o2 = h2_bits(__hmul2(bits_h2(h2), s2)), o3 = h2_bits(__hmul2(bits_h2(h3), s2));
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst0 ^ (w8 << 4)), "r"(o0), "r"(o1), "r"(o2), "r"(o3) : "memory");
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_vready[vb]));
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == C::kQkWarp) {
      // ============================================================ scores
      const uint32_t idesc_qk = (1u << 7) | (1u << 10) | (uint32_t(kStep >> 3) << 17) | (uint32_t(C::kRows >> 4) << 24);
      constexpr uint32_t kSbo = 8 * C::kRowBytes, kLayout = D == 128 ? 4u : 2u;
      const uint64_t q_desc = desc_kmajor(smem_u32(smem), kSbo, kLayout);
      const uint64_t k_desc0 = desc_kmajor(smem_u32(stage0), kSbo, kLayout), ksf_desc0 = desc_sf(smem_u32(stage0) + C::kStgKsf);
      const uint32_t sfq = tmem_base + C::kColSfq;
      // Each lane remembers its own waits, and the one that issues stops by what it saw: agreeing on it here, a step in the chain
      // of the scores, cost 1 us of 64 steps
      bool go = true;
      if (elect_one()) {
#pragma unroll
        for (int i = 0; i < 2 * C::kMma; ++i)                  // the query scales, once
          tmem_cp_sf(sfq + 4 * i, desc_sf(smem_u32(smem) + C::kOffQsf + i * 512));
      }
      __syncwarp();
      const int stop = last_step(0);
      for (int j = 0, stg = 0, ph = 0; j < stop; ++j, stg = (stg + 1 == S ? 0 : stg + 1), ph ^= (stg == 0)) {
        const int sb = j & 1;
        go = go && px_wait(smem_u32(&bar_full[stg]), ph, &abort_flag, 3);
        {                                                      // [token][group] -> [group of 64 values][32 rows][4 quarters] words
          uint8_t* st = stage0 + stg * C::kStageBytes;
#pragma unroll
          for (int q = 0; q < kStep / 32; ++q) {
            const uint32_t* raw = reinterpret_cast<const uint32_t*>(st + C::kStgKraw + (32 * q + lane) * C::kSfPerRow);
#pragma unroll
            for (int i = 0; i < C::kMma; ++i) *reinterpret_cast<uint32_t*>(st + C::kStgKsf + 512 * i + lane * 16 + q * 4) = raw[i];
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        if (j >= 2) go = go && px_wait(smem_u32(&bar_sfree[sb]), ((j >> 1) - 1) & 1, &abort_flag, 4);
        tc_fence_after();
        __syncwarp();
        if (elect_one() && go) {
          const uint64_t k_desc = k_desc0 + uint64_t((stg * C::kStageBytes) >> 4), ksf_desc = ksf_desc0 + uint64_t((stg * C::kStageBytes) >> 4);
          const uint32_t sfk = tmem_base + C::kColSfk + sb * 4 * C::kMma;
#pragma unroll
          for (int i = 0; i < C::kMma; ++i) tmem_cp_sf(sfk + 4 * i, ksf_desc + uint64_t((i * 512) >> 4));
#pragma unroll
          for (int i = 0; i < 2 * C::kMma; ++i)                // base, then residue
            mma_fp4<false>(tmem_base + C::kColS + sb * kStep, q_desc + uint64_t(((i / C::kMma) * C::kQBytes >> 4) + 2 * (i % C::kMma)),
                           k_desc + uint64_t(2 * (i % C::kMma)), idesc_qk, sfq + 4 * i, sfk + 4 * (i % C::kMma), i > 0 ? 1u : 0u);
          mma_commit(smem_u32(&bar_sfull[sb]));
          mma_commit(smem_u32(&bar_empty[stg]));               // the K codes and scales of the stage have been read
        }
        __syncwarp();
      }
      if (stop < steps) abort_flag = 3;
      if (elect_one()) {
        mma_commit(smem_u32(&bar_end[0]));
        px_drain(smem_u32(&bar_end[0]), 0, &abort_flag, 17);
      }
      __syncwarp();
    } else if (warp == C::kPvWarp) {
      // ============================================================ P.V: a thread of another warp, so that the next scores do not
      // stand in line behind the exponentials
      // kind::f16: FP32 accumulate, FP16 x FP16, A from tensor memory, B N-major (bit 16), N = D, M = 128
      const uint32_t idesc_pv = (1u << 4) | (1u << 16) | (uint32_t(D >> 3) << 17) | (uint32_t(C::kRows >> 4) << 24);
      if (elect_one()) {
        // B = V: N-major, 128-byte swizzle: 64-d blocks 128 bytes x step apart (leading offset), 8-token groups 1 KB apart
        const uint64_t v_desc0 = desc_full(smem_u32(smem + C::kOffV), kStep * 128, 1024, 2);
        const int stop = last_step(1);
        for (int j = 0; j < stop; ++j) {
          const int vb = j & 1;
          const uint64_t v_desc = v_desc0 + uint64_t((vb * C::kVBytes) >> 4);
          if (!px_wait(smem_u32(&bar_vready[vb]), (j >> 1) & 1, &abort_flag, 8) ||
              !px_wait(smem_u32(&bar_pready[vb]), (j >> 1) & 1, &abort_flag, 9)) break;
          tc_fence_after();
#pragma unroll
          for (int k16 = 0; k16 < kStep / 16; ++k16)
            mma_f16_ts(tmem_base + C::kColO, tmem_base + C::kColP + 8 * k16, v_desc + uint64_t((k16 * 2048) >> 4), idesc_pv,
                       (j > 0 || k16 > 0) ? 1u : 0u);
          mma_commit(smem_u32(&bar_pvdone[vb]));
          mma_commit(smem_u32(&bar_vfree[vb]));
        }
        if (stop < steps) abort_flag = 8;
        mma_commit(smem_u32(&bar_end[1]));
        px_drain(smem_u32(&bar_end[1]), 0, &abort_flag, 13);
      }
      __syncwarp();
    } else {
      const bool codes = warp == C::kProdWarp;
      // ============================================================ copies: lane i fetches the i-th run of a step.  `run` tokens
      // (a power of two up to the step, dividing the page size) lie together in a page.
      const int runs = kStep / run;
      auto lookup = [&](int j) -> int {
        const int t0 = (s_begin + j) * kStep + lane * run;
        if (lane >= runs || j >= steps || t0 >= p.prefix_len) return 0;
        return __ldg(p.prefix_table + (p.page_shift >= 0 ? t0 >> p.page_shift : t0 / p.page_size));
      };
      int page_next = lookup(0), armed = 0;
      const int stop = last_step(codes ? 2 : 3);
      for (int j = 0, stg = 0, ph = 0; j < stop; ++j, stg = (stg + 1 == S ? 0 : stg + 1), ph ^= (stg == 0)) {
        const int t0 = (s_begin + j) * kStep + lane * run;
        const int64_t page = min(max(int64_t(page_next), int64_t(0)), p.num_pages - 1);
        page_next = lookup(j + 1);
        const int in_row = hkv * p.page_size + (p.page_shift >= 0 ? (t0 & (p.page_size - 1)) : t0 % p.page_size);
        if (j >= S && !px_wait_warp(smem_u32(&bar_empty[stg]), ph ^ 1, &abort_flag, 14)) break;
        const uint32_t st = smem_u32(stage0 + stg * C::kStageBytes), full = smem_u32(&bar_full[stg]);
        if (lane == 0) {                                       // whole runs, also the one in which the prefix ends
          const int live = min(runs, (p.prefix_len - (s_begin + j) * kStep + run - 1) / run);
          mbar_expect_tx(full, live * run * (VDIRECT ? 1 : 2) * (codes ? C::kRowBytes : C::kSfPerRow));
        }
        __syncwarp();
        if (lane < runs && t0 < p.prefix_len) {
          const int row = lane * run;
          if (codes) {
            tma_load_3d(st + row * C::kRowBytes, &k_map, 0, in_row, int(page), full);
            if constexpr (!VDIRECT) tma_load_3d(st + C::kStgV + row * C::kRowBytes, &v_map, 0, in_row, int(page), full);
          } else {
            const int64_t sf = page * p.sf_page_stride + int64_t(in_row) * C::kSfPerRow;
            bulk_load_1d(st + C::kStgKraw + row * C::kSfPerRow, p.k_sf + sf, run * C::kSfPerRow, full);
            if constexpr (!VDIRECT) bulk_load_1d(st + C::kStgVsf + row * C::kSfPerRow, p.v_sf + sf, run * C::kSfPerRow, full);
          }
        }
        armed = j + 1;
      }
      // The last stages' data have arrived before the CTA ends.  After a step that only one of the two warps has armed -- at
      // most S of them, since a stage is refilled only when both have filled it, and none unless the kernel gives up -- the
      // other arrives in its place, so that the phase counts the bytes to its end.
      if (stop < steps) abort_flag = 14;
      if (lane == 0) copied[codes ? 0 : 1] = armed;
      asm volatile("bar.sync 14, 64;" ::: "memory");
      const int most = max(armed, copied[codes ? 1 : 0]);
      if (lane == 0)
        for (int j = armed; j < most; ++j) mbar_arrive(smem_u32(&bar_full[j % S]));
      for (int j = max(most - S, 0); j < most; ++j) px_drain(smem_u32(&bar_full[j % S]), (j / S) & 1, &abort_flag, 15);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && abort_flag != 0 && p.status) atomicExch(p.status, 1 + int(blockIdx.y) + (abort_flag << 16));
  if (warp == C::kQkWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::kTmemCols) : "memory");
  }
}

template <int D, bool VDIRECT>
int launch_prefix_form(const AttnParams& p, int prefix_splits, int run, cudaStream_t st) {
  using C = PxCfg<D>;
  static bool attr_done[64] = {};
  int dev = 0;
  RI_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) dev = 0;
  if (!attr_done[dev]) {
    RI_CUDA(cudaFuncSetAttribute(resattn_prefix_kernel<D, VDIRECT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
    RI_CUDA(cudaFuncSetAttribute(resattn_prefix_kernel<D, VDIRECT>, cudaFuncAttributePreferredSharedMemoryCarveout, 100));
    attr_done[dev] = true;
  }
  CUtensorMap k_map{}, v_map{};
  const int64_t page_rows = int64_t(p.hkv) * p.page_size;
  int s = make_pool_map<D>(&k_map, p.k_data, p.num_pages, page_rows, p.code_page_stride, run);
  if (s) return s;
  if constexpr (!VDIRECT) {
    s = make_pool_map<D>(&v_map, p.v_data, p.num_pages, page_rows, p.code_page_stride, run);
    if (s) return s;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(prefix_splits, p.hkv * ((p.batch * p.group + C::kRows - 1) / C::kRows));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, resattn_prefix_kernel<D, VDIRECT>, k_map, v_map, p, run), "shared-prefix attention launch");
}

// the first launch of a shared-prefix decode.  V by way of the stages, or directly, us for 512 rows and 16384 tokens in two
// pieces, caches cold: head_dim 128 pages of 16 90 / 74, of 32 77 / 73, of 64 71.6 / 73.3, of 128 68 / 73; head_dim 256 pages
// of 16 148 / 152, of 128 137 / 149.  A TMA copy of 16 or 32 rows takes 150 cycles whatever it holds, and V is half of them.
template <int D>
int launch_prefix(const AttnParams& p, int prefix_splits, cudaStream_t st) {
  int run = 16;                                                // tokens that lie together: divides the page size and the step
  while (run < PxCfg<D>::kStep && p.page_size % (2 * run) == 0) run *= 2;
  if constexpr (D == 128)
    if (run <= 32) return launch_prefix_form<D, true>(p, prefix_splits, run, st);
  return launch_prefix_form<D, false>(p, prefix_splits, run, st);
}
