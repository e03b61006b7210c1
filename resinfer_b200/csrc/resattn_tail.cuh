// ResAttn decode for a batch that shares a prefix: the sequences' own tokens, and the merge.  Included by resattn.cu behind
// resattn_prefix.cuh, inside namespace ri::<anon>::tcattn.
//
// A CTA of four warps takes one (sequence, KV head) and a piece of the tokens from the prefix's end on.  Each warp walks
// over every fourth group of 16 tokens by itself -- no barriers, no operand tiles in shared memory; the codes go from a
// per-warp ring of cp.async copies to registers, are expanded there to FP16 (code x block scale, exact) and multiplied
// with mma.sync:
//
//   S^T[16 tokens x 8 heads] = K . Qbase^T + K . Qres^T     K as the A operand: a thread holds 32 (head_dim 256: 64)
//                                                           consecutive values of two tokens; Q is permuted to match
//   O^T[D x 8 heads]        += V^T . P^T                    V^T as the A operand: a thread holds a scale block of four tokens;
//                                                           P^T comes from S^T's registers by a transposed 8 x 8 move
//
// The query is NVFP4 + NVFP4 residue, both parts exact in FP16; P is rounded to FP16 (11 bits, the operand's), all sums are
// FP32, a maximum is raised when a score exceeds it by more than 2^8.
//
// Eight rows and a few hundred tokens give the tensor cores' large tiles nothing to do: what counts is how soon a CTA
// reads memory and how many run.  What bounds it: instructions, 430 a group of 16 tokens and KV head, 140 of them the
// expansion -- 340 MB of own tokens (256 sequences of up to 2048, 8 heads) 113 us = 3.0 TB/s at 59 % of the issue slots; and
// 3 us before a CTA's first product and 2 behind its last -- 85 MB (64 sequences) 45 us, 24 MB (32 of up to 1024) 20.5 us.
// The decode kernel's form (21 warps, tensor memory) in this place took 54 us for 75 MB; eight warps a CTA were slower
// (340 MB: 136 us), more CTAs an SM spilled.
//
// Merge: the CTA adds its warps' partials (o, l, m) and, after waiting for the launch in front (griddepcontrol.wait), the
// partials of the prefix's pieces; with several pieces per sequence the last one to finish does it (tickets).
template <int D>
struct TlCfg {
  static constexpr int kWarps = 4, kThreads = 128, kStages = 4;
  static constexpr int kRowBytes = D / 2, kSfPerRow = D / 16;
  static constexpr int kVPitch = kRowBytes + 16;               // V rows: even tokens would share their banks
  static constexpr int kOffV = 16 * kRowBytes, kOffKsf = kOffV + 16 * kVPitch, kOffVsf = kOffKsf + 16 * kSfPerRow;
  static constexpr int kStageBytes = kOffVsf + 16 * kSfPerRow;
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  // the warps' partials, in the rings' place: [8 heads][D / 16 blocks][16], pitches for which the sixteen 8-byte accesses of
  // half a warp (four blocks, every other head) share a bank at most in pairs
  static constexpr int kOBlock = 20, kOHead = D / 16 * kOBlock + 4;
  static constexpr int kOBytes = kWarps * 8 * kOHead * 4;
  // query [2][8 heads][4 quarters][D / 4] FP16: a pitch for which the accesses of half a warp (four heads, four quarters) do not
  // share a bank.  Without the two pitches a CTA spent 1 us (head_dim 256: 2 us) on conflicts
  static constexpr int kOffQ = kRingBytes > kOBytes ? kRingBytes : kOBytes;
  static constexpr int kQQuarter = D / 4 + 4, kQHead = 4 * kQQuarter;
  static constexpr int kSmemBytes = kOffQ + 2 * 8 * kQHead * 2;
  static constexpr int kKSteps = D / 16, kMTiles = D / 16, kBlk = D / 128;
};

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// 8 codes -> 4 pairs of FP16, times s2
__device__ __forceinline__ void expand8(uint32_t codes, __half2 s2, uint32_t (&out)[4]) {
  uint32_t h0, h1, h2, h3;
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h0), "=r"(h1), "=r"(h2), "=r"(h3) : "r"(codes));
  out[0] = h2_bits(__hmul2(bits_h2(h0), s2));
  out[1] = h2_bits(__hmul2(bits_h2(h1), s2));
  out[2] = h2_bits(__hmul2(bits_h2(h2), s2));
  out[3] = h2_bits(__hmul2(bits_h2(h3), s2));
}
// the same for codes that cvt_e2m1x8 has just packed, each byte taken out by a shift.  Where the bytes that it packs (mov.b32 w,
// {b0, b1, b2, b3}) reach expand8's unpacking (mov.b32 {b0, b1, b2, b3}, w) in a straight line, CUDA 12.9's compiler joins the
// two and the codes come out wrong: expand8 is for codes from memory only
__device__ __forceinline__ void expand8_packed(uint32_t codes, __half2 s2, uint32_t (&out)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = h2_bits(__hmul2(e2m1x2_to_half2((codes >> (8 * i)) & 0xFFu), s2));
}
// two E4M3 bytes (low half of v) -> FP16 pairs (s0, s0), (s1, s1)
__device__ __forceinline__ void expand_scales(uint32_t v, uint32_t& s0, uint32_t& s1) {
  uint32_t h;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(h) : "r"(v));
  s0 = __byte_perm(h, 0, 0x1010);
  s1 = __byte_perm(h, 0, 0x3232);
}

template <int D>
__global__ void __launch_bounds__(TlCfg<D>::kThreads, D == 128 ? 4 : 2) resattn_tail_kernel(const __grid_constant__ AttnParams p) {
  using C = TlCfg<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float warp_m[C::kWarps][8], warp_l[C::kWarps][8];
  __shared__ float head_m[8], head_l[8], head_r[8];
  __shared__ int last_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hkv = blockIdx.x, b = blockIdx.y, split = blockIdx.z;   // pieces at the sequences' ends, often short, come last
  const int G = p.group;
  // Its inputs were complete when the launch in front released this one: that launch waits for everything before it, and only
  // then releases.  So only the merge waits for it here.  What this CTA reads before its own wait comes from the L2, where the
  // writes of finished launches are (ld.global.cg, cp.async.cg): no line that an SM's L1 holds from before stands in for them.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int begin = p.kv_begin / 16 + split * p.groups_per_split;       // groups of 16 tokens, at their absolute places
  // loads that wait for nothing: the pages of the warp's first groups (if the row has them), a block of the query, the length
  const int32_t* bt = p.block_tables + int64_t(b) * p.bt_stride;
  auto page_at = [&](int group) -> int {
    const int t0 = group * 16;
    return t0 < p.max_tokens ? __ldcg(bt + (p.page_shift >= 0 ? t0 >> p.page_shift : t0 / p.page_size)) : 0;
  };
  int pages[C::kStages];                                               // of the groups whose copies come first, and of the one behind them
#pragma unroll
  for (int k = 0; k < C::kStages; ++k) pages[k] = page_at(begin + warp + k * C::kWarps);
  uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
  const int qg = threadIdx.x / C::kSfPerRow, qblk = threadIdx.x % C::kSfPerRow;   // at most eight heads x kSfPerRow blocks: one per thread
  static_assert(8 * C::kSfPerRow <= C::kThreads, "one block per thread");
  if (qg < G) {
    const uint4* src = reinterpret_cast<const uint4*>(p.q + (int64_t(b) * p.hq + hkv * G + qg) * D + qblk * 16);
    x0 = __ldcg(src);
    x1 = __ldcg(src + 1);
  }
  const int L = min(max(__ldcg(p.seq_lens + b), 0), p.max_tokens);
  // the last piece goes to the sequence's end: one longer than the caller's bound costs time, not tokens
  const int end = L > p.kv_begin ? (split == p.splits - 1 ? max(begin, (L + 15) / 16) : min(begin + p.groups_per_split, (L + 15) / 16)) : begin;
  const int i8 = lane >> 2, q4 = lane & 3;
  float o[C::kMTiles][4];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};              // heads 2 q4, 2 q4 + 1
#pragma unroll
  for (int t = 0; t < C::kMTiles; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;

  if (begin < end) {                                                   // the whole CTA
    // ---------------------------------------------------------------- copies of the warp's first groups
    uint8_t* ring = smem + warp * (C::kStages * C::kStageBytes);
    const int n = begin + warp < end ? (end - begin - warp + C::kWarps - 1) / C::kWarps : 0;   // groups of this warp
    const uint8_t* const k_src = p.k_data + lane * 16;
    const uint8_t* const v_src = p.v_data + lane * 16;
    // lanes 0 .. kSfPerRow - 1 copy K's scales of a group, the next kSfPerRow V's
    const uint8_t* const sf_src = (lane < C::kSfPerRow ? p.k_sf : p.v_sf) + (lane % C::kSfPerRow) * 16;
    const uint32_t dst0 = smem_u32(ring) + lane * 16;
    const uint32_t v_dst0 = smem_u32(ring) + C::kOffV + (lane / (C::kRowBytes / 16)) * C::kVPitch + (lane % (C::kRowBytes / 16)) * 16;
    constexpr int kVStep = 32 / (C::kRowBytes / 16) * C::kVPitch;     // rows that 32 lanes cover
    const uint32_t sf_dst0 = smem_u32(ring) + C::kOffKsf + lane * 16;  // V's scales follow K's
    const int page_row0 = hkv * p.page_size, last_page = int(p.num_pages) - 1;
    const int code_stride = int(p.code_page_stride), sf_stride = int(p.sf_page_stride);   // below 2 GiB: checked on the host
    auto fetch = [&](int k, int page) {
      if (k < n) {
        const int group = begin + warp + k * C::kWarps, t0 = group * 16;
        page = min(max(page, 0), last_page);
        const int row = page_row0 + (p.page_shift >= 0 ? (t0 & (p.page_size - 1)) : t0 % p.page_size);
        const int64_t code = int64_t(page) * code_stride + row * C::kRowBytes, sf = int64_t(page) * sf_stride + row * C::kSfPerRow;
        const uint32_t st = (k % C::kStages) * C::kStageBytes;
#pragma unroll
        for (int c = 0; c < C::kRowBytes / 32; ++c) {                  // 16 rows of kRowBytes / 16 chunks
          cp_async16(dst0 + st + c * 512, k_src + code + c * 512);
          cp_async16(v_dst0 + st + c * kVStep, v_src + code + c * 512);
        }
        if (2 * C::kSfPerRow == 32 || lane < 2 * C::kSfPerRow) cp_async16(sf_dst0 + st, sf_src + sf);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int k = 0; k < C::kStages - 1; ++k) fetch(k, pages[k]);
    int page_next = pages[C::kStages - 1];
    // ---------------------------------------------------------------- query: NVFP4 and its residue, expanded to FP16
    __half* qs = reinterpret_cast<__half*>(smem + C::kOffQ);
    if (threadIdx.x < 8 * C::kSfPerRow) {                              // heads beyond the group: zeros, as loaded
      const uint32_t u[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
      float v[16];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[2 * k] = __uint_as_float(u[k] << 16);
        v[2 * k + 1] = __uint_as_float(u[k] & 0xFFFF0000u);
      }
      const BlockQ bq = quant_query16(v);
      uint32_t s0, s1;
      expand_scales(uint32_t(bq.sf) | uint32_t(bq.sf_res) << 8, s0, s1);
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const uint2 codes = part ? bq.res : bq.base;
        const __half2 s2 = bits_h2(part ? s1 : s0);
        uint32_t lo[4], hi[4];
        expand8_packed(codes.x, s2, lo);
        expand8_packed(codes.y, s2, hi);
        uint2* dst = reinterpret_cast<uint2*>(qs + (part * 8 + qg) * C::kQHead + qblk / (D / 64) * C::kQQuarter + qblk % (D / 64) * 16);
        dst[0] = make_uint2(lo[0], lo[1]);
        dst[1] = make_uint2(lo[2], lo[3]);
        dst[2] = make_uint2(hi[0], hi[1]);
        dst[3] = make_uint2(hi[2], hi[3]);
      }
    }
    __syncthreads();
    // B operands: head i8, k positions 2 q4, 2 q4 + 1 / + 8, + 9 of step ks = values q4 * (D / 4) + 4 ks + 0, 1 / 2, 3
    uint32_t qb[C::kKSteps][2], qr[C::kKSteps][2];
#pragma unroll
    for (int ks = 0; ks < C::kKSteps; ++ks) {
      const uint2 vb = *reinterpret_cast<const uint2*>(qs + i8 * C::kQHead + q4 * C::kQQuarter + 4 * ks);
      const uint2 vr = *reinterpret_cast<const uint2*>(qs + (8 + i8) * C::kQHead + q4 * C::kQQuarter + 4 * ks);
      qb[ks][0] = vb.x; qb[ks][1] = vb.y;
      qr[ks][0] = vr.x; qr[ks][1] = vr.y;
    }
    for (int k = 0; k < n; ++k) {
      fetch(k + C::kStages - 1, page_next);
      if (k + C::kStages < n) page_next = page_at(begin + warp + (k + C::kStages) * C::kWarps);
      asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
      __syncwarp();
      const uint8_t* st = ring + (k % C::kStages) * C::kStageBytes;
      const int t0 = (begin + warp + k * C::kWarps) * 16;
      // ---- scores of tokens t0 + i8 and t0 + i8 + 8
      float sa[4][4] = {};                                             // four chains: base and residue, even and odd steps
#pragma unroll
      for (int h = 0; h < C::kBlk; ++h) {                              // 32 values of the quarter at a time
        uint32_t ka[2][16];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int row = i8 + 8 * u;
          const uint4 w = *reinterpret_cast<const uint4*>(st + row * C::kRowBytes + q4 * (D / 8) + 16 * h);
          const uint32_t sf = *reinterpret_cast<const uint16_t*>(st + C::kOffKsf + row * C::kSfPerRow + q4 * (D / 64) + 2 * h);
          uint32_t s0, s1;
          expand_scales(sf, s0, s1);
          uint32_t e[4];
          expand8(w.x, bits_h2(s0), e); ka[u][0] = e[0]; ka[u][1] = e[1]; ka[u][2] = e[2]; ka[u][3] = e[3];
          expand8(w.y, bits_h2(s0), e); ka[u][4] = e[0]; ka[u][5] = e[1]; ka[u][6] = e[2]; ka[u][7] = e[3];
          expand8(w.z, bits_h2(s1), e); ka[u][8] = e[0]; ka[u][9] = e[1]; ka[u][10] = e[2]; ka[u][11] = e[3];
          expand8(w.w, bits_h2(s1), e); ka[u][12] = e[0]; ka[u][13] = e[1]; ka[u][14] = e[2]; ka[u][15] = e[3];
        }
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          mma_16816(sa[ks & 1], ka[0][2 * ks], ka[1][2 * ks], ka[0][2 * ks + 1], ka[1][2 * ks + 1], qb[8 * h + ks][0], qb[8 * h + ks][1]);
          mma_16816(sa[2 + (ks & 1)], ka[0][2 * ks], ka[1][2 * ks], ka[0][2 * ks + 1], ka[1][2 * ks + 1], qr[8 * h + ks][0], qr[8 * h + ks][1]);
        }
      }
      float s[4];
      const bool partial = t0 < p.kv_begin || t0 + 16 > L;             // some of the tokens are another's, or nobody's
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int tok = t0 + i8 + 8 * (u >> 1);
        s[u] = partial && (tok < p.kv_begin || tok >= L) ? -INFINITY : ((sa[0][u] + sa[1][u]) + (sa[2][u] + sa[3][u])) * p.score_scale_log2;
      }
      if (__any_sync(0xffffffffu, fmaxf(s[0], s[2]) > m[0] + kLazyThreshold || fmaxf(s[1], s[3]) > m[1] + kLazyThreshold)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {                                  // this thread's two heads
          float mx = fmaxf(s[h], s[2 + h]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          const float nw = fmaxf(m[h], mx), f = m[h] == -INFINITY ? 0.f : fast_exp2(m[h] - nw);
          m[h] = nw;
          l[h] *= f;
#pragma unroll
          for (int t = 0; t < C::kMTiles; ++t) {
            o[t][h] *= f;
            o[t][2 + h] *= f;
          }
        }
      }
      float e[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        e[u] = fast_exp2(s[u] - (m[u & 1] == -INFINITY ? 0.f : m[u & 1]));
        l[u & 1] += e[u];
      }
      const uint32_t p0 = transpose8x8(h2_bits(__floats2half2_rn(e[0], e[1])));   // head i8, tokens 2 q4, 2 q4 + 1
      const uint32_t p1 = transpose8x8(h2_bits(__floats2half2_rn(e[2], e[3])));   // ... + 8, + 9
      // ---- O^T: scale block i8 (and i8 + 8) of tokens 2 q4, 2 q4 + 1, 2 q4 + 8, 2 q4 + 9
#pragma unroll
      for (int h = 0; h < C::kBlk; ++h) {
        const int blk = i8 + 8 * h;
        uint32_t sp[2];                                                // (scale of token 2 q4, of 2 q4 + 1), (+ 8, + 9)
        uint2 codes[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int row = 2 * q4 + 8 * u;
          uint32_t f0 = st[C::kOffVsf + row * C::kSfPerRow + blk], f1 = st[C::kOffVsf + (row + 1) * C::kSfPerRow + blk];
          if (partial) {                                               // whatever lies there: 0 x P = 0
            if (t0 + row < p.kv_begin || t0 + row >= L) f0 = 0;
            if (t0 + row + 1 < p.kv_begin || t0 + row + 1 >= L) f1 = 0;
          }
          asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(sp[u]) : "r"(f0 | f1 << 8));
          codes[2 * u] = *reinterpret_cast<const uint2*>(st + C::kOffV + row * C::kVPitch + blk * 8);
          codes[2 * u + 1] = *reinterpret_cast<const uint2*>(st + C::kOffV + (row + 1) * C::kVPitch + blk * 8);
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {                                  // eight values of the block at a time
          uint32_t ev[2][4], od[2][4];                                 // pairs of tokens: even values, odd values
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            // the two tokens' codes side by side in a byte, so that one conversion gives the operand's pair
            const uint32_t c0 = w ? codes[2 * u].y : codes[2 * u].x, c1 = w ? codes[2 * u + 1].y : codes[2 * u + 1].x;
            expand8((c0 & 0x0F0F0F0Fu) | ((c1 << 4) & 0xF0F0F0F0u), bits_h2(sp[u]), ev[u]);
            expand8(((c0 >> 4) & 0x0F0F0F0Fu) | (c1 & 0xF0F0F0F0u), bits_h2(sp[u]), od[u]);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c)                                  // values 8 w + 2 c, + 1 of the block
            mma_16816(o[8 * h + 4 * w + c], ev[0][c], od[0][c], ev[1][c], od[1][c], p0, p1);
        }
      }
      __syncwarp();                                                    // the stage may be refilled
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], x);
      if (n > 0 && m[h] == -INFINITY) m[h] = __int_as_float(0x7fffffff);   // a group has at least one token: see max_nan
    }
    __syncthreads();                                                   // every ring has been read
    float* ow = reinterpret_cast<float*>(smem) + warp * 8 * C::kOHead;
#pragma unroll
    for (int t = 0; t < C::kMTiles; ++t) {
      const int d = C::kOBlock * (i8 + 8 * (t / 8)) + 2 * (t % 8);
      *reinterpret_cast<float2*>(ow + (2 * q4) * C::kOHead + d) = make_float2(o[t][0], o[t][2]);
      *reinterpret_cast<float2*>(ow + (2 * q4 + 1) * C::kOHead + d) = make_float2(o[t][1], o[t][3]);
    }
  }
  if (lane < 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      warp_m[warp][2 * lane + h] = m[h];
      warp_l[warp][2 * lane + h] = l[h];
    }
  }
  __syncthreads();
  // ---------------------------------------------------------------- the CTA's partial: weights 2^(m_w - m) of its warps
  if (threadIdx.x < 8) {
    float mm = -INFINITY, ll = 0.f;
    for (int w = 0; w < C::kWarps; ++w) mm = max_nan(mm, warp_m[w][threadIdx.x]);
    for (int w = 0; w < C::kWarps; ++w) {
      const float f = warp_m[w][threadIdx.x] == -INFINITY ? 0.f : fast_exp2(warp_m[w][threadIdx.x] - mm);
      warp_m[w][threadIdx.x] = f;
      ll += f * warp_l[w][threadIdx.x];
    }
    head_m[threadIdx.x] = mm;
    head_l[threadIdx.x] = ll;
  }
  __syncthreads();
  constexpr int kPer = 8 * D / 4 / C::kThreads;                        // groups of four columns of a thread (for eight heads)
  float4 acc[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int c4 = threadIdx.x + k * C::kThreads, g = c4 / (D / 4), c = c4 % (D / 4);
    acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (g < G && begin < end) {
      const float* src = reinterpret_cast<const float*>(smem) + g * C::kOHead + c / 4 * C::kOBlock + c % 4 * 4;
#pragma unroll
      for (int w = 0; w < C::kWarps; ++w) {
        const float f = warp_m[w][g];
        const float4 v = *reinterpret_cast<const float4*>(src + w * 8 * C::kOHead);
        acc[k].x += f * v.x; acc[k].y += f * v.y; acc[k].z += f * v.z; acc[k].w += f * v.w;
      }
    }
  }
  const int64_t rows = int64_t(p.batch) * p.hq, row0 = int64_t(b) * p.hq + hkv * G;   // slot s of head g: s * rows + row0 + g
  int first = p.splits;                                                // partials to add: slots first .. splits + prefix_splits - 1
  if (p.splits > 1) {
    first = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int c4 = threadIdx.x + k * C::kThreads, g = c4 / (D / 4);
      if (g < G && begin < end) reinterpret_cast<float4*>(p.o_part + (split * rows + row0) * D)[c4] = acc[k];   // nobody reads an empty one's
      acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (threadIdx.x < G) {
      p.l_part[split * rows + row0 + threadIdx.x] = head_l[threadIdx.x];
      p.m_part[split * rows + row0 + threadIdx.x] = head_m[threadIdx.x];
    }
    __threadfence();
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");                   // the prefix's partials, the cleared tickets
  if (p.splits > 1) {
    if (threadIdx.x == 0) {
      last_flag = atomicAdd(p.split_counter + b * p.hkv + hkv, 1) == p.splits - 1;
      __threadfence();
    }
    __syncthreads();
    if (!last_flag) return;
    if (threadIdx.x < 8) {                                             // the CTA's own partial is among the slots now
      head_m[threadIdx.x] = -INFINITY;
      head_l[threadIdx.x] = 0.f;
    }
    __syncthreads();
  }
  // ---------------------------------------------------------------- merge: sixteen threads per head find the weights
  const int total = p.splits + p.prefix_splits - first;
  float* w_sh = reinterpret_cast<float*>(smem + C::kOBytes);           // [total][8] maxima, then weights; [total][8] row sums
  float* l_sh = w_sh + total * 8;
  constexpr int kBatch = 8;                                            // partials whose loads are in flight together
  float4 v[kPer][kBatch];
  const float4* src0 = reinterpret_cast<const float4*>(p.o_part + (first * rows + row0) * D) + threadIdx.x;
  auto load_batch = [&](int s0) {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (s0 + j < total && threadIdx.x + k * C::kThreads < G * (D / 4))
          v[k][j] = __ldcg(src0 + k * C::kThreads + (s0 + j) * rows * (D / 4));
  };
  load_batch(0);                                                       // before their weights are known
  {
    const int g = threadIdx.x >> 4, x16 = threadIdx.x & 15;
    float mm = head_m[g];
    for (int s = x16; s < total && g < G; s += 16) {
      const float ms = __ldcg(p.m_part + (first + s) * rows + row0 + g), ls = __ldcg(p.l_part + (first + s) * rows + row0 + g);
      w_sh[s * 8 + g] = ms;
      l_sh[s * 8 + g] = ls;
      mm = max_nan(mm, ms);
    }
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) mm = max_nan(mm, __shfl_xor_sync(0xffffffffu, mm, x));
    float ll = 0.f;
    for (int s = x16; s < total && g < G; s += 16) {                   // this thread's own entries
      const float ms = w_sh[s * 8 + g], w = ms == -INFINITY ? 0.f : fast_exp2(ms - mm);
      w_sh[s * 8 + g] = w;
      if (w != 0.f) ll += w * l_sh[s * 8 + g];
    }
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, x);
    __syncwarp();
    if (x16 == 0) {
      const float f = head_m[g] == -INFINITY ? 0.f : fast_exp2(head_m[g] - mm);
      ll += f * head_l[g];
      head_m[g] = f;                                                   // the weight of what the CTA holds in registers
      head_r[g] = ll > 0.f ? p.out_scale / ll : 0.f;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int c4 = threadIdx.x + k * C::kThreads, g = min(c4 / (D / 4), 7);
    const float f = head_m[g];
    acc[k].x *= f; acc[k].y *= f; acc[k].z *= f; acc[k].w *= f;
  }
  for (int s0 = 0; s0 < total; s0 += kBatch) {                         // in order
    if (s0 > 0) load_batch(s0);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int c4 = threadIdx.x + k * C::kThreads, g = c4 / (D / 4);
      float w[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) w[j] = s0 + j < total && g < G ? w_sh[(s0 + j) * 8 + g] : 0.f;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {                               // no branches: 32 of them in a row took 1 us a batch
        const bool some = w[j] != 0.f;                                 // empty partials hold no data
        acc[k].x += w[j] * (some ? v[k][j].x : 0.f);
        acc[k].y += w[j] * (some ? v[k][j].y : 0.f);
        acc[k].z += w[j] * (some ? v[k][j].z : 0.f);
        acc[k].w += w[j] * (some ? v[k][j].w : 0.f);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int c4 = threadIdx.x + k * C::kThreads, g = c4 / (D / 4);
    if (g >= G) continue;
    float4 a = acc[k];
    const float r = head_r[g];
    a.x *= r; a.y *= r; a.z *= r; a.w *= r;
    const int64_t oi = row0 * D + 4 * c4;
    if (p.out_f32) {
      *reinterpret_cast<float4*>(static_cast<float*>(p.out) + oi) = a;
    } else {
      __nv_bfloat162 lo = __floats2bfloat162_rn(a.x, a.y), hi = __floats2bfloat162_rn(a.z, a.w);
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + oi) =
          make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
    }
  }
}

// the second launch of a shared-prefix decode (or, without a prefix launch in front, the whole decode)
template <int D>
int launch_tail(const AttnParams& p, cudaStream_t st) {
  using C = TlCfg<D>;
  static bool attr_done[64] = {};
  int dev = 0;
  RI_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) dev = 0;
  const int weights = (p.splits + p.prefix_splits) * 8 * 4 * 2;
  constexpr int kMost = C::kOBytes + 512 * 64 > C::kSmemBytes ? C::kOBytes + 512 * 64 : C::kSmemBytes;
  if (!attr_done[dev]) {
    RI_CUDA(cudaFuncSetAttribute(resattn_tail_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
    RI_CUDA(cudaFuncSetAttribute(resattn_tail_kernel<D>, cudaFuncAttributePreferredSharedMemoryCarveout, 100));
    attr_done[dev] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.hkv, p.batch, p.splits);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kOBytes + weights > C::kSmemBytes ? C::kOBytes + weights : C::kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  if (p.prefix_splits > 0) {      // released by the prefix launch; without one, the kernel has no wait in front of its inputs
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
  }
  return cuda_status(cudaLaunchKernelEx(&cfg, resattn_tail_kernel<D>, p), "shared-prefix decode launch");
}
