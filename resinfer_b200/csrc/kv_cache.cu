// Paged NVFP4 KV cache: quantising K / V rows into it, and reading them back.
//
// A pool keeps, for K and for V, codes [pages, Hkv, page_size, D/2] and E4M3 block scales
// [pages, Hkv, page_size, D/16]; pages may lie further apart than their rows (an engine's interleaved cache).
// A block of 16 values with largest magnitude a and global scale g is held as
//     s = e4m3((1/g) (a / 6)),   code_i = e2m1(x_i ((1/g) / s)),   value_i = code_i s g      (0 where s = 0)
// -- the arithmetic of this library's NVFP4 quantisers operation by operation (nvfp4_scale, quant_plain16), so a
// cache written here has the bytes that nvfp4::scaled_fp4_quant_mext_r1 gives for the same rows.
//
// Both kernels stream: a thread owns one 16-value block of K and the same block of V (two independent 32-byte
// loads or stores in flight), consecutive threads own consecutive blocks of a token's [Hkv, D] row, so the dense
// side is fully coalesced and the cache side is touched in whole 64-byte (head_dim 128) code rows.  Bound by
// memory; nothing is staged.  Measured at 8 KV heads of 128, bytes that have to move over time, of a 6.55 TB/s copy:
// 131072 tokens written 112 us = 6.15 TB/s (0.94), read from a block table 110 us = 6.27 TB/s (0.96); 256 tokens 1.9 and
// 2.4 us, what a launch costs.
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "resinfer_b200.h"

namespace ri {
namespace {

struct PoolRef {
  uint8_t* k_data; uint8_t* k_sf;
  uint8_t* v_data; uint8_t* v_sf;
  int64_t num_slots;                       // pages * page_size
  int64_t code_page_stride, sf_page_stride;
  int page_size, page_shift;               // page_shift: log2(page_size) when it is a power of two, else -1
  int hkv, blocks;                         // KV heads, 16-value blocks per row (D / 16)
};

// Where tokens live: a list of slots, or the sequences of a batch laid end to end.
struct TokenRef {
  const void* slots; int slots64;
  const int32_t* block_tables; int64_t bt_stride, bt_cols;
  const int32_t* cu_seqlens; int batch;
  int64_t num_tokens;
};

// byte offsets of block `blk` of head `head` in slot `slot`
__device__ __forceinline__ void slot_offsets(const PoolRef& p, int64_t slot, int head, int blk, int64_t& code, int64_t& sf) {
  int64_t page;
  int off;
  if (p.page_shift >= 0) {
    page = slot >> p.page_shift;
    off = int(slot) & (p.page_size - 1);
  } else {
    page = slot / p.page_size;
    off = int(slot - page * p.page_size);
  }
  const int64_t row = int64_t(head) * p.page_size + off;
  code = page * p.code_page_stride + (row * p.blocks + blk) * 8;
  sf = page * p.sf_page_stride + row * p.blocks + blk;
}

__device__ __forceinline__ int64_t load_slot(const TokenRef& t, int64_t tok) {
  return t.slots64 ? __ldg(static_cast<const int64_t*>(t.slots) + tok)
                   : int64_t(__ldg(static_cast<const int32_t*>(t.slots) + tok));
}

// 16 values from an address that need not be aligned beyond the element
template <typename T>
__device__ __forceinline__ void load16_any(const T* p, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = float(p[i]);
}

struct DenseIn {
  const void* k; const void* v;
  int64_t k_token, k_head, v_token, v_head;   // strides in elements
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) kv_write_kernel(const DenseIn in, const TokenRef t, const PoolRef p,
                                                       float k_gs_inv, float v_gs_inv) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");   // inputs may come from a kernel still running
  const int unit = blockIdx.y * blockDim.x + threadIdx.x;
  const int64_t tok = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  if (unit >= p.hkv * p.blocks || tok >= t.num_tokens) return;
  const int head = unit / p.blocks, blk = unit - head * p.blocks;
  const T* ks = static_cast<const T*>(in.k) + tok * in.k_token + head * in.k_head + blk * 16;
  const T* vs = static_cast<const T*>(in.v) + tok * in.v_token + head * in.v_head + blk * 16;
  const int64_t slot = load_slot(t, tok);
  float kx[16], vx[16];
  if constexpr (VEC) {                                 // loaded before the slot is looked at: one memory latency, not two
    load16(ks, kx);
    load16(vs, vx);
  } else {
    load16_any(ks, kx);
    load16_any(vs, vx);
  }
  if (slot < 0 || slot >= p.num_slots) return;         // padding
  int64_t code, sf;
  slot_offsets(p, slot, head, blk, code, sf);
  auto store = [&](const float (&x)[16], float gs, uint8_t* codes, uint8_t* scales) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i]));
    uint8_t byte;
    const float mult = nvfp4_scale(amax, gs, &byte);
    *reinterpret_cast<uint2*>(codes + code) = quant_plain16(x, mult);
    scales[sf] = byte;
  };
  store(kx, k_gs_inv, p.k_data, p.k_sf);
  store(vx, v_gs_inv, p.v_data, p.v_sf);
}

// two values of an output row as one 32-bit word (16-bit types)
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}

__device__ __forceinline__ void store32(void* dst, const uint32_t (&w)[8]) {   // 32 bytes to a 16-byte aligned address
  if ((reinterpret_cast<uintptr_t>(dst) & 31) == 0) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
  } else {
    static_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    static_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// one held block -> 16 values of the output row.  code * s is exact in FP32 (6 significant bits), the product with
// the global scale is rounded once to FP32 and once to the output type.
template <typename T>
__device__ __forceinline__ void store_held16(T* dst, uint2 codes, uint8_t sf_byte, float gs) {
  float x[16];
  float lo[8], hi[8];
  e2m1x8_to_float(codes.x, lo);
  e2m1x8_to_float(codes.y, hi);
  const float s = decode_e4m3(sf_byte);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = (lo[i] * s) * gs;
    x[8 + i] = (hi[i] * s) * gs;
  }
  uint32_t w[8];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(x[8 * h + i]);
      store32(dst + 8 * h, w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
    store32(dst, w);
  }
}

// NT tokens per thread, blockDim.y apart: their table look-ups and their loads are in flight together.
template <typename T, bool BATCH, int NT>
__global__ void __launch_bounds__(256) kv_read_kernel(T* __restrict__ k_out, T* __restrict__ v_out, const TokenRef t,
                                                      const PoolRef p, float k_gs, float v_gs, int zero_tail) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int unit = blockIdx.y * blockDim.x + threadIdx.x;
  if (unit >= p.hkv * p.blocks) return;
  const int head = unit / p.blocks, blk = unit - head * p.blocks;
  const int64_t tok0 = int64_t(blockIdx.x) * (blockDim.y * NT) + threadIdx.y;
  int64_t slot[NT];
  bool write[NT];
  int seq = 0;                                                        // sequence of this thread's last token
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t tok = tok0 + j * int(blockDim.y);
    write[j] = tok < t.num_tokens;
    slot[j] = -1;
    if (!write[j]) continue;
    if constexpr (BATCH) {
      // the sequence of `tok`: the next one's start is beyond it.  Usually the last token's; else searched
      if (j == 0 || tok >= __ldg(t.cu_seqlens + seq + 1)) {
        int hi = t.batch;
        while (hi - seq > 1) {
          const int mid = (seq + hi) >> 1;
          if (__ldg(t.cu_seqlens + mid) <= tok) seq = mid;
          else hi = mid;
        }
      }
      const int64_t pos = tok - __ldg(t.cu_seqlens + seq);
      if (pos >= 0 && tok < __ldg(t.cu_seqlens + seq + 1)) {
        const int64_t col = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
        if (col < t.bt_cols) {
          const int64_t page = __ldg(t.block_tables + seq * t.bt_stride + col);
          slot[j] = page * p.page_size + (pos - col * p.page_size);   // negative for an unused table entry
        }
      } else if (tok >= __ldg(t.cu_seqlens + t.batch) && !zero_tail) {
        write[j] = false;                                             // rows behind the last sequence stay as they are
      }
    } else {
      slot[j] = load_slot(t, tok);
    }
  }
  uint2 kc[NT], vc[NT];
  uint8_t ksf[NT], vsf[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    kc[j] = vc[j] = make_uint2(0, 0);                                 // no slot: code 0 times scale 0
    ksf[j] = vsf[j] = 0;
    if (slot[j] >= 0 && slot[j] < p.num_slots) {
      int64_t code, sf;
      slot_offsets(p, slot[j], head, blk, code, sf);
      kc[j] = __ldg(reinterpret_cast<const uint2*>(p.k_data + code));
      vc[j] = __ldg(reinterpret_cast<const uint2*>(p.v_data + code));
      ksf[j] = __ldg(p.k_sf + sf);
      vsf[j] = __ldg(p.v_sf + sf);
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    if (!write[j]) continue;
    const int64_t dst = ((tok0 + j * int(blockDim.y)) * (p.hkv * p.blocks) + unit) * 16;
    store_held16(k_out + dst, kc[j], ksf[j], k_gs);
    store_held16(v_out + dst, vc[j], vsf[j], v_gs);
  }
}

int check_pool(PoolRef* p, const uint8_t* k_data, const uint8_t* k_sf, const uint8_t* v_data, const uint8_t* v_sf,
               int64_t num_pages, int64_t code_page_stride, int64_t sf_page_stride, int num_kv_heads, int head_dim,
               int page_size) {
  RI_CHECK_ARG(num_kv_heads > 0 && num_kv_heads <= 65536 && head_dim >= 16 && head_dim <= 65536 && head_dim % 16 == 0,
               "a paged NVFP4 cache has head_dim a multiple of 16 and at least one KV head, got %d heads of %d",
               num_kv_heads, head_dim);
  RI_CHECK_ARG(int64_t(num_kv_heads) * (head_dim / 16) <= (1 << 20), "%d KV heads of %d are too wide a row", num_kv_heads, head_dim);
  RI_CHECK_ARG(page_size >= 16 && page_size % 16 == 0, "page size must be a multiple of 16, got %d", page_size);
  RI_CHECK_ARG(num_pages > 0 && k_data && k_sf && v_data && v_sf, "empty page pool");
  const int64_t page_rows = int64_t(num_kv_heads) * page_size;
  if (code_page_stride == 0) code_page_stride = page_rows * (head_dim / 2);
  if (sf_page_stride == 0) sf_page_stride = page_rows * (head_dim / 16);
  RI_CHECK_ARG(code_page_stride >= page_rows * (head_dim / 2) && sf_page_stride >= page_rows * (head_dim / 16) &&
                   code_page_stride % 16 == 0 && sf_page_stride % 16 == 0,
               "page strides (%lld, %lld bytes) must be multiples of 16 and hold a page's %lld rows",
               (long long)code_page_stride, (long long)sf_page_stride, (long long)page_rows);
  RI_CHECK_ARG(((reinterpret_cast<uintptr_t>(k_data) | reinterpret_cast<uintptr_t>(v_data) |
                 reinterpret_cast<uintptr_t>(k_sf) | reinterpret_cast<uintptr_t>(v_sf)) & 15) == 0,
               "the KV pool must be 16-byte aligned");
  p->k_data = const_cast<uint8_t*>(k_data); p->k_sf = const_cast<uint8_t*>(k_sf);
  p->v_data = const_cast<uint8_t*>(v_data); p->v_sf = const_cast<uint8_t*>(v_sf);
  p->num_slots = num_pages * page_size;
  p->code_page_stride = code_page_stride; p->sf_page_stride = sf_page_stride;
  p->page_size = page_size;
  p->page_shift = -1;
  for (int s = 4; s < 31; ++s)
    if ((1 << s) == page_size) p->page_shift = s;
  p->hkv = num_kv_heads; p->blocks = head_dim / 16;
  return RI_OK;
}

int check_scale(float g, const char* name) {
  RI_CHECK_ARG(isfinite(g) && g > 0.f && isfinite(1.0f / g), "%s must be a positive finite number with a finite reciprocal, got %g", name, double(g));
  return RI_OK;
}

// threads of a CTA: x over a token's blocks, y over tokens
void geometry(int64_t tokens, int units, int per_thread, cudaLaunchConfig_t* cfg) {
  const int tx = units < 256 ? units : 256;
  const int ty = 256 / tx;
  const int64_t per_cta = int64_t(ty) * per_thread;
  cfg->blockDim = dim3(tx, ty);
  cfg->gridDim = dim3((unsigned)((tokens + per_cta - 1) / per_cta), (unsigned)((units + tx - 1) / tx));
}

}  // namespace
}  // namespace ri

using namespace ri;

extern "C" int ri_kv_write_nvfp4(const void* k, const void* v, int dtype, int64_t k_token_stride, int64_t k_head_stride,
                                 int64_t v_token_stride, int64_t v_head_stride, const void* slots, int slot_bits,
                                 int64_t num_tokens, uint8_t* k_data, uint8_t* k_sf, uint8_t* v_data, uint8_t* v_sf,
                                 int64_t num_pages, int64_t code_page_stride, int64_t sf_page_stride, int num_kv_heads,
                                 int head_dim, int page_size, float k_global_scale, float v_global_scale, void* stream) {
  RI_CHECK_ARG(dtype == RI_DTYPE_BF16 || dtype == RI_DTYPE_FP16, "K and V must be bf16 or fp16");
  RI_CHECK_ARG(slot_bits == 32 || slot_bits == 64, "slots must be 32- or 64-bit integers");
  RI_CHECK_ARG(num_tokens >= 0 && num_tokens < (int64_t(1) << 31), "bad token count %lld", (long long)num_tokens);
  PoolRef p{};
  int s = check_pool(&p, k_data, k_sf, v_data, v_sf, num_pages, code_page_stride, sf_page_stride, num_kv_heads, head_dim, page_size);
  if (s) return s;
  if ((s = check_scale(k_global_scale, "k_global_scale")) || (s = check_scale(v_global_scale, "v_global_scale"))) return s;
  if (num_tokens == 0) return RI_OK;
  RI_CHECK_ARG(k && v && slots, "K, V and the slots must not be null");
  RI_CHECK_ARG(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 1) == 0 &&
                   (reinterpret_cast<uintptr_t>(slots) & (slot_bits / 8 - 1)) == 0, "misaligned K, V or slots");
  DeviceInfo di;
  if ((s = device_info(&di))) return s;
  const DenseIn in{k, v, k_token_stride, k_head_stride, v_token_stride, v_head_stride};
  TokenRef t{};
  t.slots = slots; t.slots64 = slot_bits == 64; t.num_tokens = num_tokens;
  // rows at 16-byte boundaries in 32-byte loads; others value by value: 16384 tokens take 36.4 us that way against 12.7
  const bool vec = (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0) &&
                   ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) == 0;
  cudaLaunchConfig_t cfg{};
  geometry(num_tokens, num_kv_heads * (head_dim / 16), 1, &cfg);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const float kg = 1.0f / k_global_scale, vg = 1.0f / v_global_scale;
  auto go = [&](auto kernel) { return cuda_status(cudaLaunchKernelEx(&cfg, kernel, in, t, p, kg, vg), "KV cache write launch"); };
  if (dtype == RI_DTYPE_BF16) return vec ? go(kv_write_kernel<__nv_bfloat16, true>) : go(kv_write_kernel<__nv_bfloat16, false>);
  return vec ? go(kv_write_kernel<__half, true>) : go(kv_write_kernel<__half, false>);
}

extern "C" int ri_kv_read_nvfp4(const uint8_t* k_data, const uint8_t* k_sf, const uint8_t* v_data, const uint8_t* v_sf,
                                int64_t num_pages, int64_t code_page_stride, int64_t sf_page_stride, int num_kv_heads,
                                int head_dim, int page_size, const void* slots, int slot_bits, const int32_t* block_tables,
                                int64_t bt_stride, int64_t bt_cols, const int32_t* cu_seqlens, int batch,
                                int64_t num_tokens, float k_global_scale, float v_global_scale, void* k_out, void* v_out,
                                int out_dtype, int zero_tail, void* stream) {
  RI_CHECK_ARG(out_dtype == RI_DTYPE_BF16 || out_dtype == RI_DTYPE_FP16 || out_dtype == RI_DTYPE_F32, "output must be bf16, fp16 or fp32");
  RI_CHECK_ARG(num_tokens >= 0 && num_tokens < (int64_t(1) << 31), "bad token count %lld", (long long)num_tokens);
  PoolRef p{};
  int s = check_pool(&p, k_data, k_sf, v_data, v_sf, num_pages, code_page_stride, sf_page_stride, num_kv_heads, head_dim, page_size);
  if (s) return s;
  if ((s = check_scale(k_global_scale, "k_global_scale")) || (s = check_scale(v_global_scale, "v_global_scale"))) return s;
  const bool by_batch = slots == nullptr && block_tables != nullptr;
  if (by_batch) {
    RI_CHECK_ARG(cu_seqlens != nullptr && batch >= 1 && bt_cols >= 1 && bt_stride >= 0, "a batch needs block tables and cumulative lengths");
  } else {
    RI_CHECK_ARG(slot_bits == 32 || slot_bits == 64, "slots must be 32- or 64-bit integers");
    RI_CHECK_ARG(num_tokens == 0 || (slots && (reinterpret_cast<uintptr_t>(slots) & (slot_bits / 8 - 1)) == 0), "slots must be given and aligned");
  }
  if (num_tokens == 0) return RI_OK;
  RI_CHECK_ARG(k_out && v_out && ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) == 0,
               "outputs must be 16-byte aligned");
  DeviceInfo di;
  if ((s = device_info(&di))) return s;
  TokenRef t{};
  t.slots = slots; t.slots64 = slot_bits == 64; t.num_tokens = num_tokens;
  t.block_tables = block_tables; t.bt_stride = bt_stride; t.bt_cols = bt_cols; t.cu_seqlens = cu_seqlens; t.batch = batch;
  cudaLaunchConfig_t cfg{};
  const int units = num_kv_heads * (head_dim / 16);
  // Four tokens a thread where that leaves several waves of CTAs; one below.  us for one / four at 8 heads of 128: from slots
  // 2048 tokens 3.6 / 5.2, 65536 57.2 / 55.1, 131072 111.0 / 106.6; from a block table 24576 tokens 23.5 / 24.2, 65536
  // 57.7 / 57.6, 131072 112.7 / 109.8; 40001 tokens in 48 sequences, 4 heads of 256, 41.7 / 39.9.
  const bool wide = num_tokens * units >= int64_t(di.sm_count) * 2048 * 8;
  geometry(num_tokens, units, wide ? 4 : 1, &cfg);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  auto go = [&](auto* type) {
    using T = std::remove_pointer_t<decltype(type)>;
    T* ko = static_cast<T*>(k_out);
    T* vo = static_cast<T*>(v_out);
    auto launch = [&](auto kernel) {
      return cuda_status(cudaLaunchKernelEx(&cfg, kernel, ko, vo, t, p, k_global_scale, v_global_scale, zero_tail), "KV cache read launch");
    };
    if (by_batch) return wide ? launch(kv_read_kernel<T, true, 4>) : launch(kv_read_kernel<T, true, 1>);
    return wide ? launch(kv_read_kernel<T, false, 4>) : launch(kv_read_kernel<T, false, 1>);
  };
  if (out_dtype == RI_DTYPE_BF16) return go(static_cast<__nv_bfloat16*>(nullptr));
  if (out_dtype == RI_DTYPE_FP16) return go(static_cast<__half*>(nullptr));
  return go(static_cast<float*>(nullptr));
}
