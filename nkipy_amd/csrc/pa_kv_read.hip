// Reading a paged KV cache back: the first seq_lens[b] tokens of every sequence, gathered through its block table and
// dequantised, as dense bf16 rows: token t of sequence b becomes row cu[b] + t of k_out / v_out [total, Hkv, D], the
// form in which packed prompt attention takes its keys and values.  np.take of the pool by the table
// (nkipy/src/nkipy/core/tensor.py:575-640) with the cast that the pool's type asks for:
//   int8   code x scale of its (token, kv head)         fp8 (e4m3fn)   code x scale of its (block, kv head)
//   bf16   the bits as they are
// each product in float32, rounded once.
//
// Pure streaming, HBM bound: a byte in, two bytes out (four with bf16).  270 K tokens of 8 heads of 128, int8: 316-329 us,
// 5.1-5.3 TB/s (a copy of 2 GiB reaches 4.9); 2 K tokens 5.5 us.  A workgroup takes 16 tokens of one sequence; a
// token's heads are adjacent in the pool and in the output, so consecutive lanes walk whole rows.  The sequence of a
// workgroup is found by bisection (packed_find); rows of the output that no token falls on are left as they are.
#include "pa_common.h"

namespace pa {
namespace {

constexpr int WG = 256, TOK_SHIFT = 4, UNR = 4;

template <int KV>      // pool type: PA_BF16, PA_FP8_E4M3FN, PA_INT8
__global__ __launch_bounds__(WG) void kv_read_kernel(KvReadParams p) {
  constexpr int EB = KV == PA_BF16 ? 2 : 1;
  int tile;
  const int b = packed_find(as_packed(p.cu), p.B, p.total, TOK_SHIFT, blockIdx.x, &tile);
  const int first = packed_row(as_packed(p.cu), b, p.total);
  const int n = min(min(p.seq_lens[b], p.max_blocks * p.block_size), packed_row(as_packed(p.cu), b + 1, p.total) - first);
  const int t0 = tile << TOK_SHIFT;
  if (tile < 0 || t0 >= n) return;
  const bool is_v = blockIdx.y != 0;
  const char* pool = (const char*)(is_v ? p.v_cache : p.k_cache);
  const float* scales = is_v ? p.v_scale : p.k_scale;
  uint16_t* out = (uint16_t*)(is_v ? p.v_out : p.k_out);
  const int cpr = p.Hkv * p.D / 8, cph = p.D / 8;           // 8-element chunks per token, per head
  const int live = min(n - t0, 1 << TOK_SHIFT) * cpr;
  for (int i0 = threadIdx.x; i0 < live; i0 += UNR * WG) {
    uint4 raw[UNR];
    float sc[UNR];
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const int i = min(i0 + u * WG, live - 1);              // (past the end: the last chunk again, not stored)
      const int tok = i / cpr, c = i - tok * cpr;
      const int pos = t0 + tok;
      const int jb = p.block_shift >= 0 ? pos >> p.block_shift : pos / p.block_size;
      const int in_blk = pos - jb * p.block_size;
      int blk = p.block_tables[(long)b * p.max_blocks + jb];
      const bool ok = blk >= 0 && blk < p.num_blocks;        // a bad table entry reads nothing: zeros
      blk = ok ? blk : 0;
      const char* src = pool + (((long)blk * p.block_size + in_blk) * cpr + c) * (8 * EB);
      if (EB == 2) raw[u] = *(const uint4*)src;
      else {
        const uint2 w = *(const uint2*)src;
        raw[u] = make_uint4(w.x, w.y, 0, 0);
      }
      sc[u] = 1.f;
      if (KV == PA_INT8) sc[u] = scales[((long)blk * p.Hkv + c / cph) * p.block_size + in_blk];
      if (KV == PA_FP8_E4M3FN) sc[u] = scales[(long)blk * p.Hkv + c / cph];
      if (!ok) { raw[u] = make_uint4(0, 0, 0, 0); sc[u] = 0.f; }
    }
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const int i = i0 + u * WG;
      if (i >= live) break;
      uint4 o = raw[u];
      if (KV != PA_BF16) {
        float f[8];
        if (KV == PA_INT8) {
          const uint32_t w[2] = {raw[u].x, raw[u].y};
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = (float)(int)(int8_t)(w[j >> 2] >> (8 * (j & 3)));
        } else {
          fp8x4_to_float(raw[u].x, f);
          fp8x4_to_float(raw[u].y, f + 4);
        }
        o = make_uint4(pack_bf16x2(f[0] * sc[u], f[1] * sc[u]), pack_bf16x2(f[2] * sc[u], f[3] * sc[u]),
                       pack_bf16x2(f[4] * sc[u], f[5] * sc[u]), pack_bf16x2(f[6] * sc[u], f[7] * sc[u]));
      }
      const int tok = i / cpr, c = i - tok * cpr;
      *(uint4*)(out + ((long)(first + t0 + tok) * cpr + c) * 8) = o;
    }
  }
}

}  // namespace

hipError_t launch_kv_read(const KvReadParams& p, hipStream_t s) {
  const dim3 grid((p.total >> TOK_SHIFT) + p.B, 2);
  switch (p.kv_dtype) {
    case PA_BF16: hipLaunchKernelGGL(kv_read_kernel<PA_BF16>, grid, dim3(WG), 0, s, p); break;
    case PA_FP8_E4M3FN: hipLaunchKernelGGL(kv_read_kernel<PA_FP8_E4M3FN>, grid, dim3(WG), 0, s, p); break;
    case PA_INT8: hipLaunchKernelGGL(kv_read_kernel<PA_INT8>, grid, dim3(WG), 0, s, p); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace pa
