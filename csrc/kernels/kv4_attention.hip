// Attention over the 4-bit paged KV cache (layout and format: kv4.h), plain: one wave per query row and head, 64 keys at a time,
// a key per lane for the scores and two dims per lane for the output, 32-bit arithmetic and running softmax.
#include "hipserve/kv4.h"

namespace hipserve {

template <int D>
__global__ __launch_bounds__(256) void kv4_attention_kernel(Kv4Attn a, const int* __restrict__ cu_q, int seqs,
                                                            const int* __restrict__ ctx_lens,
                                                            const int* __restrict__ tiles, int rows,
                                                            unsigned short* __restrict__ out16) {
  __shared__ float qs[4][D];
  __shared__ float ps[4][64];
  __shared__ int pages[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int h = blockIdx.y, kh = h / (a.nq / a.cache.nkv);
  int seq, pos, row, ctx;
  if (tiles != nullptr) {  // a row of a tile of 128 rows of a sequence
    seq = tiles[2 * (blockIdx.x / 32)];
    if (seq < 0 || seq >= seqs) return;
    const int r = tiles[2 * (blockIdx.x / 32) + 1] + blockIdx.x % 32 * 4 + wave;
    const int qlen = cu_q[seq + 1] - cu_q[seq];
    if (r < 0 || r >= qlen) return;
    ctx = ctx_lens[seq];
    pos = ctx - qlen + r;
    row = cu_q[seq] + r;
    if (row < 0 || row >= rows) return;
  } else {
    seq = row = blockIdx.x * 4 + wave;
    if (seq >= rows) return;
    ctx = ctx_lens[seq];
    pos = ctx - 1;
  }
  const int bs = a.cache.block_size;
  const int limit = min(pos + 1, a.bt_width * bs);
  const unsigned short* q = static_cast<const unsigned short*>(a.q) + row * a.q_stride + (long)h * D;
  for (int d = lane; d < D; d += 64) qs[wave][d] = bf16_to_f32(q[d]);
  const long head_bytes = kv4_head_bytes(bs, D);
  const int code_bytes = kv4_code_bytes(bs, D);
  const int* bt = a.block_tables + (long)seq * a.bt_stride;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int j0 = 0; j0 < limit; j0 += 64) {
    const int j = j0 + lane;
    const int page = j < limit ? kv4_page(bt[j / bs], a.cache.blocks) : -1;
    const bool sees = page >= 0 && kv4_sees(j, pos, a.window, a.sinks);
    float sc = -INFINITY;
    if (sees) {
      const unsigned char* kp = static_cast<const unsigned char*>(a.cache.k) + ((long)page * a.cache.nkv + kh) * head_bytes;
      const int off = j % bs;
      float dot = 0.f;
      for (int g = 0; g < D / 32; ++g) {
        const int byte = kp[code_bytes + g * bs + kv4_key_scale_at(off)];
        const float s = byte == kKv4Nan ? NAN : kv4_scale(byte);
        float part = 0.f;
        for (int w = 0; w < 4; ++w) {
          const unsigned c = *reinterpret_cast<const unsigned*>(kp + off * (D / 2) + g * 16 + w * 4);
          const unsigned v[4] = {kv4_widen2<0>(c, 1.f), kv4_widen2<1>(c, 1.f), kv4_widen2<2>(c, 1.f), kv4_widen2<3>(c, 1.f)};
          for (int e = 0; e < 4; ++e) {
            part += bf16_to_f32(v[e] & 0xffff) * qs[wave][g * 32 + w * 8 + 2 * e];
            part += bf16_to_f32(v[e] >> 16) * qs[wave][g * 32 + w * 8 + 2 * e + 1];
          }
        }
        dot += part * s;
      }
      sc = dot * a.scale * kLog2E;
    }
    const float m_new = fmaxf(m, wave_max(sc));
    if (m_new == -INFINITY && !__any(sc != sc)) continue;  // nothing seen so far
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float p = sees ? exp2f(sc - base) : 0.f;
    const float alpha = exp2f(m - base);
    m = m_new;
    l = l * alpha + wave_sum(p);
    ps[wave][lane] = p;
    pages[wave][lane] = page;
    o0 *= alpha;
    o1 *= alpha;
    if (lane < D / 2) {
      for (int e = 0; e < 64; ++e) {
        const int page_e = pages[wave][e];
        if (page_e < 0 || !kv4_sees(j0 + e, pos, a.window, a.sinks)) continue;
        const unsigned char* vp = static_cast<const unsigned char*>(a.cache.v) + ((long)page_e * a.cache.nkv + kh) * head_bytes;
        const int off = (j0 + e) % bs;
        const int byte = vp[code_bytes + (lane >> 4) * bs + off];
        const float s = byte == kKv4Nan ? NAN : kv4_scale(byte);
        const unsigned v = kv4_widen2<0>(vp[lane * bs + off], 1.f);
        o0 += ps[wave][e] * (bf16_to_f32(v & 0xffff) * s);
        o1 += ps[wave][e] * (bf16_to_f32(v >> 16) * s);
      }
    }
  }
  if (lane < D / 2) {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: zeros
    unsigned short* out = static_cast<unsigned short*>(a.out) + row * a.out_stride + (long)h * D;
    const unsigned pair = pack_bf16x2(o0 * inv, o1 * inv);
    *reinterpret_cast<unsigned*>(out + 2 * lane) = pair;
    if (out16 != nullptr) {
      store_o16(out16, (long)row * a.out_stride, h * D + 2 * lane, (unsigned short)pair);
      store_o16(out16, (long)row * a.out_stride, h * D + 2 * lane + 1, (unsigned short)(pair >> 16));
    }
  }
}

static void kv4_attention(const Kv4Attn& a, const int* cu_q, int seqs, const int* ctx, const int* tiles, int blocks,
                          int rows, void* out16, hipStream_t s) {
  const dim3 grid(blocks, a.nq);
  auto* o16 = static_cast<unsigned short*>(out16);
  if (a.cache.D == 128) kv4_attention_kernel<128><<<grid, 256, 0, s>>>(a, cu_q, seqs, ctx, tiles, rows, o16);
  else if (a.cache.D == 96) kv4_attention_kernel<96><<<grid, 256, 0, s>>>(a, cu_q, seqs, ctx, tiles, rows, o16);
  else kv4_attention_kernel<64><<<grid, 256, 0, s>>>(a, cu_q, seqs, ctx, tiles, rows, o16);
}

void launch_kv4_prefill(const Kv4Attn& a, const int* cu_q, int seqs, const int* ctx_lens, int rows, const int* tiles,
                        int ntiles, hipStream_t s) {
  if (ntiles > 0) kv4_attention(a, cu_q, seqs, ctx_lens, tiles, ntiles * 32, rows, nullptr, s);
}

}  // namespace hipserve
