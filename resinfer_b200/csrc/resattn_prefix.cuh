// ResAttn decode for a batch that shares a prefix: the prefix part.  Included by resattn.cu behind resattn_pv.cuh, inside
// namespace ri::<anon>::tcattn.
//
// All query heads of all sequences that read one KV head are rows of one problem, R = batch x group rows against the
// prefix's tokens, so the prefix crosses HBM once instead of once per sequence.  A CTA takes NT tiles of 128 rows, one KV
// head and a range of the prefix (its split) in steps of 64 tokens:
//
//   S[128 rows x 64]  = Qbase . K^T + Qres . K^T   tcgen05.mma kind::mxf4nvf4.block_scale, codes and E4M3 scales as stored
//   P = 2^(S scale - m)                            one row per softmax thread, rounded to FP16
//   O[128 rows x D]  += P . V                      tcgen05.mma kind::f16, P from tensor memory, V expanded to FP16 (exact)
//
// and leaves the unnormalised partial (o, l, m) of its rows; the launch behind it (resattn_pv_kernel's TAIL form: the
// sequences' own tokens) adds the partials of all splits.  The statistics m, l and the accumulator o stay in FP32; the
// maximum of a row is only raised when a score exceeds it by more than 2^8, so o is rarely rescaled.  FP16 holds the
// code x block scale products exactly and P with 11 bits.
//
// Rows shorter than the prefix are masked at their own length; rows beyond the batch have length zero.
//
// Roles:
//   softmax     four warps per row tile, thread = row (tensor-memory lane)
//   conversion  four warps: V codes x scales -> FP16 in the 128-byte-swizzled N-major operand layout, once for all row tiles
//   issue       one thread per row tile: K scales shared -> tensor memory, scores of step j+1 before the P.V of step j
//   copies      two warps of cp.async, 32 tokens of a step each: pages of 16 tokens and up
// Every wait is bounded.  A role whose wait expires sets the abort flag, which ends all other waits at once, and runs on
// through its loop (every address is in bounds whatever the data), so all roles meet at the end and the status word is set.
template <int D, int NT_>
struct PxCfg {
  static constexpr int NT = NT_;                               // row tiles of a CTA
  static constexpr int kStep = 64;                             // tokens per step
  static constexpr int kRows = 128;
  static constexpr int kFirstConv = 4 * NT, kFirstIssue = kFirstConv + 4, kFirstProd = kFirstIssue + 2;
  static constexpr int kThreads = (kFirstProd + 2) * 32;       // 12 or 16 warps: whole warpgroups
  static constexpr int kCtasPerSm = D == 128 && NT == 1 ? 2 : 1;
  static constexpr int kStages = kCtasPerSm == 2 ? 4 : 6;
  static constexpr int kMma = D / 64;
  static constexpr int kRowBytes = D / 2;
  static constexpr int kSfPerRow = D / 16;
  static constexpr int kDBlocks = D / 64;
  // shared memory: per row tile Q codes (base, residue) and Q scales (base, residue); V tiles; stages
  static constexpr int kQBytes = kRows * kRowBytes;
  static constexpr int kQsfBytes = kMma * 512;
  static constexpr int kOffQsf = 2 * kQBytes, kQTile = 2 * kQBytes + 2 * kQsfBytes;     // multiples of 1024
  static constexpr int kVBytes = kStep * D * 2;
  static constexpr int kOffV = NT * kQTile;
  static constexpr int kOffStage = kOffV + 2 * kVBytes;
  static constexpr int kKBytes = kStep * kRowBytes;
  static constexpr int kStgV = kKBytes, kStgKsf = 2 * kKBytes, kStgVsf = kStgKsf + kMma * 512;
  static constexpr int kStageBytes = (kStgVsf + kStep * kSfPerRow + 1023) / 1024 * 1024;
  static constexpr int kSmemBytes = kOffStage + kStages * kStageBytes + 1024;
  // tensor memory columns of a row tile: accumulator, scores, P, query scales, K scales (two sets)
  static constexpr int kColO = 0, kColS = D, kColP = D + 64, kColSfq = D + 96, kColSfk = kColSfq + 8 * kMma;
  static constexpr int kTileCols = D == 128 ? 256 : 512;
  static constexpr int kTmemCols = NT * kTileCols;
  static_assert(kColSfk + 8 * kMma <= kTileCols && kTmemCols <= 512 && kQTile % 1024 == 0, "layout");
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
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A wait that returns when the phase is complete, or when the kernel has given up (see above).
__device__ __forceinline__ void px_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int site) {
  if (mbar_try(bar, parity)) return;
  if (*abort_flag) return;
  mbar_wait(bar, parity, abort_flag, site);
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

template <int D, int NT>
__global__ void __launch_bounds__(PxCfg<D, NT>::kThreads, PxCfg<D, NT>::kCtasPerSm)
resattn_prefix_kernel(const __grid_constant__ AttnParams p) {
  using C = PxCfg<D, NT>;
  constexpr int S = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[S], bar_empty[S];
  __shared__ __align__(8) uint64_t bar_sfull[NT], bar_sfree[NT], bar_pready[NT], bar_pvdone[NT], bar_vready[2], bar_vfree[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x, hkv = blockIdx.y % p.hkv, row0 = (blockIdx.y / p.hkv) * (NT * C::kRows);
  const int G = p.group, rows = p.batch * G;

  // Everything this kernel reads was written before the launch in front of it ended, and the launch behind it may start
  // only now: it therefore may read the same inputs without a wait of its own (it waits before it reads the partials).
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int n_steps = (p.prefix_len + C::kStep - 1) / C::kStep;
  const int s_begin = min(split * p.steps_per_split, n_steps);
  const int steps = min(s_begin + p.steps_per_split, n_steps) - s_begin;

  if (split == 0 && blockIdx.y == 0 && p.splits > 1)           // tickets of the launch behind this one
    for (int i = threadIdx.x; i < p.batch * p.hkv; i += blockDim.x) p.split_counter[i] = 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 64);
      mbar_init(smem_u32(&bar_empty[s]), 4 + NT);              // conversion warps + the commits of the scores' MMAs
    }
    for (int t = 0; t < NT; ++t) {
      mbar_init(smem_u32(&bar_sfull[t]), 1);
      mbar_init(smem_u32(&bar_sfree[t]), 4);
      mbar_init(smem_u32(&bar_pready[t]), 4);
      mbar_init(smem_u32(&bar_pvdone[t]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&bar_vready[s]), 4);
      mbar_init(smem_u32(&bar_vfree[s]), NT);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == C::kFirstIssue) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_slot)), "r"(C::kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // ---------------------------------------------------------------- query prologue: NVFP4 and its NVFP4 residue
  for (int i = threadIdx.x; i < NT * C::kRows * C::kSfPerRow; i += blockDim.x) {
    const int rr = i / C::kSfPerRow, blk = i % C::kSfPerRow, row = row0 + rr;
    const int r = rr & (C::kRows - 1);
    BlockQ bq{};
    if (row < rows) {
      const int b = row / G, g = row - b * G;
      float v[16];
      load16(p.q + (int64_t(b) * p.hq + hkv * G + g) * D + blk * 16, v);
      bq = quant_mext16(v, 1.0f, 1.0f);
    }
    uint8_t* tile = smem + (rr / C::kRows) * C::kQTile;
    const uint32_t off = swz_off<D>(r, blk * 8);
    *reinterpret_cast<uint2*>(tile + off) = bq.base;
    *reinterpret_cast<uint2*>(tile + C::kQBytes + off) = bq.res;
    const uint32_t so = C::kOffQsf + (blk >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (blk & 3);
    tile[so] = bq.sf;
    tile[so + C::kQsfBytes] = bq.sf_res;
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  uint8_t* stage0 = smem + C::kOffStage;

  if (warp < C::kFirstConv) {
    // ============================================================ softmax warps
    if constexpr (C::kCtasPerSm == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    const int tile = warp >> 2, quarter = warp & 3;
    const uint32_t lane_base = tmem_base + tile * C::kTileCols + (uint32_t(quarter * 32) << 16);
    const uint32_t b_sfull = smem_u32(&bar_sfull[tile]), b_sfree = smem_u32(&bar_sfree[tile]);
    const uint32_t b_pready = smem_u32(&bar_pready[tile]), b_pvdone = smem_u32(&bar_pvdone[tile]);
    const int row = row0 + warp * 32 + lane;
    int lim = 0;
    if (row < rows) lim = min(max(__ldg(p.seq_lens + row / G), 0), p.prefix_len);
    const int lim_min = __reduce_min_sync(0xffffffffu, lim), lim_max = __reduce_max_sync(0xffffffffu, lim);
    const float scale = p.score_scale_log2;
    float m = -INFINITY, l = 0.f;
    if (lim_max <= s_begin * C::kStep) {
      // none of this warp's rows reaches the split's tokens: their P is zero throughout
      uint32_t z[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) z[i] = 0;
      tmem_st32(lane_base + C::kColP, z);
      tmem_wait_st();
      tc_fence_before();
      for (int j = 0; j < steps; ++j) {
        px_wait(b_sfull, j & 1, &abort_flag, 5);
        if (j > 0) px_wait(b_pvdone, (j - 1) & 1, &abort_flag, 7);
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(b_sfree);
          mbar_arrive(b_pready);
        }
      }
    } else {
      for (int j = 0; j < steps; ++j) {
        px_wait(b_sfull, j & 1, &abort_flag, 5);
        __syncwarp();
        tc_fence_after();
        uint32_t s[2][32];
        tmem_ld32_async(lane_base + C::kColS, s[0]);
        tmem_ld32_async(lane_base + C::kColS + 32, s[1]);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(b_sfree);                   // the next scores may overwrite S
        const int tok0 = (s_begin + j) * C::kStep;
        if (tok0 + C::kStep > lim_min) {
#pragma unroll
          for (int i = 0; i < 64; ++i)
            if (tok0 + i >= lim) s[i >> 5][i & 31] = 0xff800000u;   // -inf
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 64; i += 2)
          m4[(i >> 1) & 3] = max3(m4[(i >> 1) & 3], __uint_as_float(s[i >> 5][i & 31]), __uint_as_float(s[i >> 5][(i & 31) + 1]));
        const float mx = max3(fmaxf(m4[0], m4[1]), m4[2], m4[3]) * scale;   // scale > 0
        bool pv_seen = j == 0;
        if (__any_sync(0xffffffffu, mx > m + kLazyThreshold)) {
          const float nw = fmaxf(m, mx);
          const float f = m == -INFINITY ? 0.f : fast_exp2(m - nw);
          m = nw;
          l *= f;
          if (j > 0) {                                         // rescale this row's accumulator in place
            px_wait(b_pvdone, (j - 1) & 1, &abort_flag, 7);
            __syncwarp();
            pv_seen = true;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              float o[16];
              tmem_ld16(lane_base + C::kColO + c, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= f;
              tmem_st16f(lane_base + C::kColO + c, o);
            }
            tmem_wait_st();
          }
        }
        const float mu = m == -INFINITY ? 0.f : m;             // a row with nothing to attend to yet
        uint32_t pk[32];
        const uint64_t scale2 = pair64(__float_as_uint(scale), __float_as_uint(scale));
        const uint64_t mu2 = pair64(__float_as_uint(-mu), __float_as_uint(-mu));
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float a, b;
          unpair64(fma2(pair64(s[i >> 4][(2 * i) & 31], s[i >> 4][(2 * i + 1) & 31]), scale2, mu2), a, b);
          a = fast_exp2(a);
          b = fast_exp2(b);
          sum[i & 1] = add2(sum[i & 1], pair64(__float_as_uint(a), __float_as_uint(b)));
          pk[i] = h2_bits(__floats2half2_rn(a, b));
        }
        {
          float a, b;
          unpair64(add2(sum[0], sum[1]), a, b);
          l += a + b;
        }
        if (!pv_seen) {
          px_wait(b_pvdone, (j - 1) & 1, &abort_flag, 7);
          __syncwarp();
        }
        tc_fence_after();
        tmem_st32(lane_base + C::kColP, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(b_pready);
      }
    }
    // ---------------------------------------------------------------- the rows' partials
    if (steps > 0) px_wait(b_pvdone, (steps - 1) & 1, &abort_flag, 12);
    __syncwarp();
    if (__any_sync(0xffffffffu, row < rows)) {                 // whole warps: the loads from tensor memory are collective
      const int b = row / G, g = row - b * G;
      const int64_t slot = (int64_t(p.splits + split) * p.batch + b) * p.hq + hkv * G + g;
      if (row < rows) {
        p.l_part[slot] = m == -INFINITY ? 0.f : l;
        p.m_part[slot] = m;
      }
      if (__any_sync(0xffffffffu, row < rows && m != -INFINITY)) {
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          float o[16];
          tmem_ld16(lane_base + C::kColO + c, o);
          if (row < rows) {
            float4* dst = reinterpret_cast<float4*>(p.o_part + slot * D + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
        tc_fence_before();
      }
    }
  } else if (warp < C::kFirstIssue) {
    // ============================================================ V conversion warps
    if constexpr (C::kCtasPerSm == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    const int cw = warp - C::kFirstConv;
    constexpr int kPer = C::kDBlocks / 2;                      // d-blocks a thread converts
    const int tok = 32 * (cw & 1) + lane;
    for (int j = 0, stg = 0, ph = 0; j < steps; ++j, stg = (stg + 1 == S ? 0 : stg + 1), ph ^= (stg == 0)) {
      const int vb = j & 1;
      px_wait(smem_u32(&bar_full[stg]), ph, &abort_flag, 6);
      const uint8_t* st = stage0 + stg * C::kStageBytes;
      const bool valid = (s_begin + j) * C::kStep + tok < p.prefix_len;
      uint4 c0[kPer], c1[kPer];
      uint32_t sfw[kPer];
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const int dblk = (cw >> 1) * kPer + u;
        c0[u] = c1[u] = make_uint4(0, 0, 0, 0);
        sfw[u] = 0;
        if (valid) {
          const uint8_t* src = st + C::kStgV;
          c0[u] = *reinterpret_cast<const uint4*>(src + swz_off<D>(tok, 32 * dblk));
          c1[u] = *reinterpret_cast<const uint4*>(src + swz_off<D>(tok, 32 * dblk + 16));
          sfw[u] = *reinterpret_cast<const uint32_t*>(st + C::kStgVsf + tok * C::kSfPerRow + dblk * 4);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_empty[stg]));   // the codes are in registers: the stage may be refilled
      if (j >= 2) px_wait(smem_u32(&bar_vfree[vb]), ((j >> 1) - 1) & 1, &abort_flag, 11);
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        const int dblk = (cw >> 1) * kPer + u;
        const uint32_t words[8] = {c0[u].x, c0[u].y, c0[u].z, c0[u].w, c1[u].x, c1[u].y, c1[u].z, c1[u].w};
        uint32_t lo, hi, sc2[4];                               // the four block scales as FP16 pairs (s, s)
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi) : "r"(sfw[u]));
        sc2[0] = __byte_perm(lo, 0, 0x1010); sc2[1] = __byte_perm(lo, 0, 0x3232);
        sc2[2] = __byte_perm(hi, 0, 0x1010); sc2[3] = __byte_perm(hi, 0, 0x3232);
        const uint32_t dst0 = smem_u32(smem + C::kOffV + vb * C::kVBytes + dblk * (C::kStep * 128) + (tok >> 3) * 1024 + (tok & 7) * 128) |
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
    if constexpr (C::kCtasPerSm == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp < C::kFirstIssue + NT) {
      // ============================================================ issue: one thread per row tile
      const int tile = warp - C::kFirstIssue;
      const uint32_t idesc_qk = (1u << 7) | (1u << 10) | (uint32_t(C::kStep >> 3) << 17) | (uint32_t(C::kRows >> 4) << 24);
      // kind::f16: FP32 accumulate, FP16 x FP16, A from tensor memory, B N-major (bit 16), N = D, M = 128
      const uint32_t idesc_pv = (1u << 4) | (1u << 16) | (uint32_t(D >> 3) << 17) | (uint32_t(C::kRows >> 4) << 24);
      constexpr uint32_t kSbo = 8 * C::kRowBytes, kLayout = D == 128 ? 4u : 2u;
      if (elect_one()) {
        const uint32_t tm = tmem_base + tile * C::kTileCols, sfq = tm + C::kColSfq;
        const uint32_t q_addr = smem_u32(smem) + tile * C::kQTile;
        const uint64_t qb_desc = desc_kmajor(q_addr, kSbo, kLayout), qr_desc = desc_kmajor(q_addr + C::kQBytes, kSbo, kLayout);
        const uint32_t b_sfull = smem_u32(&bar_sfull[tile]), b_sfree = smem_u32(&bar_sfree[tile]);
        const uint32_t b_pready = smem_u32(&bar_pready[tile]), b_pvdone = smem_u32(&bar_pvdone[tile]);
#pragma unroll
        for (int j = 0; j < 2 * C::kMma; ++j)                  // the query scales, once
          tmem_cp_sf(sfq + 4 * j, desc_sf(q_addr + C::kOffQsf + j * 512));
        auto issue_qk = [&](int j, int stg, int ph) {
          px_wait(smem_u32(&bar_full[stg]), ph, &abort_flag, 3);
          if (j > 0) px_wait(b_sfree, (j - 1) & 1, &abort_flag, 4);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // cp.async data -> tensor-core reads
          tc_fence_after();
          const uint32_t st = smem_u32(stage0 + stg * C::kStageBytes);
          const uint64_t k_desc = desc_kmajor(st, kSbo, kLayout);
          const uint32_t sfk = tm + C::kColSfk + (j & 1) * 4 * C::kMma;
#pragma unroll
          for (int i = 0; i < C::kMma; ++i) tmem_cp_sf(sfk + 4 * i, desc_sf(st + C::kStgKsf + i * 512));
#pragma unroll
          for (int i = 0; i < C::kMma; ++i)
            mma_fp4<false>(tm + C::kColS, qb_desc + uint64_t(2 * i), k_desc + uint64_t(2 * i), idesc_qk, sfq + 4 * i, sfk + 4 * i,
                           i > 0 ? 1u : 0u);
#pragma unroll
          for (int i = 0; i < C::kMma; ++i)
            mma_fp4<false>(tm + C::kColS, qr_desc + uint64_t(2 * i), k_desc + uint64_t(2 * i), idesc_qk, sfq + 4 * (C::kMma + i),
                           sfk + 4 * i, 1u);
          mma_commit(b_sfull);
          mma_commit(smem_u32(&bar_empty[stg]));               // the K codes of the stage have been read
        };
        // B = V: N-major, 128-byte swizzle: 64-d blocks 8 KB apart (leading offset), 8-token groups 1 KB apart
        const uint64_t v_desc = desc_full(smem_u32(smem + C::kOffV), C::kStep * 128, 1024, 2);
        if (steps > 0) issue_qk(0, 0, 0);
        for (int j = 0, stg = 1, ph = 0; j < steps; ++j) {
          if (j + 1 < steps) issue_qk(j + 1, stg, ph);
          if (++stg == S) stg = 0, ph ^= 1;
          const int vb = j & 1;
          px_wait(smem_u32(&bar_vready[vb]), (j >> 1) & 1, &abort_flag, 8);
          px_wait(b_pready, j & 1, &abort_flag, 9);
          tc_fence_after();
#pragma unroll
          for (int k16 = 0; k16 < C::kStep / 16; ++k16)
            mma_f16_ts(tm + C::kColO, tm + C::kColP + 8 * k16, v_desc + uint64_t((vb * C::kVBytes + k16 * 2048) >> 4), idesc_pv,
                       (j > 0 || k16 > 0) ? 1u : 0u);
          mma_commit(b_pvdone);
          mma_commit(smem_u32(&bar_vfree[vb]));
        }
        if (steps > 0) px_wait(b_pvdone, (steps - 1) & 1, &abort_flag, 13);   // nothing of this tile is in flight any more
      }
      __syncwarp();
    } else if (warp >= C::kFirstProd) {
      // ============================================================ copies: warp pw, tokens 32 pw .. 32 pw + 31 of a step
      const int pw = warp - C::kFirstProd;
      constexpr int kCpr = C::kRowBytes / 16, kRowsPerIt = 32 / kCpr, kIters = 32 / kRowsPerIt;
      const int r_lane = lane / kCpr, chn = lane % kCpr;
      auto lookup = [&](int j) -> int {                        // lanes 0 and 1: the pages of the warp's two groups of 16 tokens
        const int t0 = (s_begin + j) * C::kStep + 32 * pw + lane * 16;
        if (lane >= 2 || j >= steps || t0 >= p.prefix_len) return 0;
        return __ldg(p.prefix_table + (p.page_shift >= 0 ? t0 >> p.page_shift : t0 / p.page_size));
      };
      int page_next = lookup(0);
      for (int j = 0, stg = 0, ph = 0; j < steps; ++j, stg = (stg + 1 == S ? 0 : stg + 1), ph ^= (stg == 0)) {
        const int tok0 = (s_begin + j) * C::kStep + 32 * pw;
        const int nrows = min(max(((p.prefix_len - tok0) + 15) & ~15, 0), 32);
        int64_t page = page_next;
        page_next = lookup(j + 1);
        page = page < 0 ? 0 : (page >= p.num_pages ? p.num_pages - 1 : page);
        const int t0 = tok0 + lane * 16;
        const int in_page = p.page_shift >= 0 ? (t0 & (p.page_size - 1)) : t0 % p.page_size;
        const int in_row = hkv * p.page_size + in_page;
        const int pg0 = __shfl_sync(0xffffffffu, int(page), 0), pg1 = __shfl_sync(0xffffffffu, int(page), 1);
        const int in0 = __shfl_sync(0xffffffffu, in_row, 0), in1 = __shfl_sync(0xffffffffu, in_row, 1);
        const int64_t code0 = pg0 * p.code_page_stride + int64_t(in0) * C::kRowBytes;
        const int64_t code1 = pg1 * p.code_page_stride + int64_t(in1) * C::kRowBytes;
        const int64_t sf0 = pg0 * p.sf_page_stride + int64_t(in0) * C::kSfPerRow;
        const int64_t sf1 = pg1 * p.sf_page_stride + int64_t(in1) * C::kSfPerRow;
        if (j >= S) px_wait(smem_u32(&bar_empty[stg]), ph ^ 1, &abort_flag, 4);
        __syncwarp();
        const uint32_t st = smem_u32(stage0 + stg * C::kStageBytes);
#pragma unroll
        for (int it = 0; it < kIters; ++it) {
          const int r = it * kRowsPerIt + r_lane;
          if (it * kRowsPerIt < nrows) {
            const int64_t src = ((it * kRowsPerIt) >> 4 ? code1 : code0) + (r & 15) * C::kRowBytes + chn * 16;
            const uint32_t dst = st + swz_off<D>(32 * pw + r, chn * 16);
            cp_async16(dst, p.k_data + src);
            cp_async16(dst + C::kStgV, p.v_data + src);
          }
        }
        if (lane < nrows) {                                    // block scales of token 32 pw + lane
          const int64_t src = (lane < 16 ? sf0 : sf1) + (lane & 15) * C::kSfPerRow;
          const uint32_t kdst = st + C::kStgKsf + lane * 16 + pw * 4;      // [64-column group][32 rows][4 quarters][4 bytes]
#pragma unroll
          for (int i = 0; i < C::kMma; ++i)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(kdst + 512 * i), "l"(p.k_sf + src + 4 * i) : "memory");
          const uint32_t vdst = st + C::kStgVsf + (32 * pw + lane) * C::kSfPerRow;
          if constexpr (D == 128) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(vdst), "l"(p.v_sf + src) : "memory");
          else cp_async16(vdst, p.v_sf + src);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&bar_full[stg])) : "memory");
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && abort_flag != 0 && p.status) atomicExch(p.status, 1 + int(blockIdx.y) + (abort_flag << 16));
  if (warp == C::kFirstIssue) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::kTmemCols) : "memory");
  }
}

template <int D, int NT>
int launch_prefix_tiles(const AttnParams& p, int prefix_splits, cudaStream_t st) {
  using C = PxCfg<D, NT>;
  static bool attr_done[64] = {};
  int dev = 0;
  RI_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) dev = 0;
  if (!attr_done[dev]) {
    RI_CUDA(cudaFuncSetAttribute(resattn_prefix_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes));
    RI_CUDA(cudaFuncSetAttribute(resattn_prefix_kernel<D, NT>, cudaFuncAttributePreferredSharedMemoryCarveout, 100));
    attr_done[dev] = true;
  }
  const int rows_per_cta = NT * C::kRows;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(prefix_splits, p.hkv * ((p.batch * p.group + rows_per_cta - 1) / rows_per_cta));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, resattn_prefix_kernel<D, NT>, p), "shared-prefix attention launch");
}

template <int D>
int launch_prefix(const AttnParams& p, int prefix_splits, cudaStream_t st) {
  if constexpr (D == 128) {
    if (p.batch * p.group > 128) return launch_prefix_tiles<128, 2>(p, prefix_splits, st);
  }
  return launch_prefix_tiles<D, 1>(p, prefix_splits, st);
}
