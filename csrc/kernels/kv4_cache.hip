// Writers and reader of the 4-bit paged KV cache (layout and format: kv4.h).
//
// kv4_write: the rotary embedding of a step's queries and keys and the step's keys and values quantised into their slots. The
// arithmetic up to the quantisation is rope_cache's and splitk_rope_cache's, rounding for rounding (bf16 after the sum, the bias, the
// norm and the rotation), so the cache holds the 4-bit rounding of what a bf16 cache would hold and the queries are the same bits.
// A workgroup takes kTok tokens of one kv head and its queries: rotated keys and the values go through LDS as bf16, four lanes
// then hold a group of 32 dims (the two halves of a rotated head need not be whole groups: heads of 96).
#include "hipserve/kv4.h"

namespace hipserve {

struct Kv4In {
  const float* ws;  // split-K partials [S, T, N], or null: the rows of qkv
  long slice;       // T * N
  int S, N;
  const unsigned short* bias;
  const float* qw;
  const float* kw;
  float eps;
};

// 8 values of column col of a row: of the partials (summed, rounded to bf16, the bias added and rounded again), or the row itself
template <bool kParts>
HS_DEVICE void kv4_in8(float (&x)[8], const Kv4In& in, const unsigned short* __restrict__ row, int t, int col) {
  if constexpr (kParts) {
    sum8_bf16(x, in.ws + (long)t * in.N + col, in.slice, in.S);
    if (in.bias != nullptr) add_bias8(x, in.bias + col);
  } else {
    const u16x8 v = *reinterpret_cast<const u16x8*>(row + col);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = bf16_to_f32(v[j]);
  }
}

template <int kMode, bool kParts, int kTok, int kThreads>
__global__ __launch_bounds__(kThreads) void kv4_write_kernel(unsigned short* __restrict__ qkv, long qkv_stride, Kv4In in,
                                                             const long* __restrict__ positions, long max_pos,
                                                             const long* __restrict__ slots,
                                                             const float* __restrict__ cos_sin,
                                                             unsigned char* __restrict__ k_cache,
                                                             unsigned char* __restrict__ v_cache, long nslots, int T,
                                                             int nq, int nkv, int D, int bs) {
  __shared__ __attribute__((aligned(16))) unsigned short kv[2][kTok][128];
  const int t0 = blockIdx.x * kTok, nt = min(kTok, T - t0);
  const int kh = blockIdx.y;
  const int h0 = nq * kh / nkv, nh = nq * (kh + 1) / nkv - h0;  // this kv head's queries
  const int half = D / 2;
  const int chunks = kMode == 0 ? half / 8 : D / 8;
  // queries and the key: 8 + 8 values of the two halves of a head (rotate-half), or 8 neighbouring ones
  for (int it = threadIdx.x; it < nt * (nh + 1) * chunks; it += kThreads) {
    const int c = it % chunks, hl = it / chunks % (nh + 1), tt = it / chunks / (nh + 1);
    const int t = t0 + tt;
    const bool is_k = hl == nh;
    const int col = is_k ? (nq + kh) * D : (h0 + hl) * D;
    unsigned short* row = qkv + t * qkv_stride;
    const float* cs = cos_sin + min(max(positions[t], 0L), max_pos - 1) * D;
    unsigned short* dst = is_k ? kv[0][tt] : row + col;
    if constexpr (kMode == 0) {
      float x[8], y[8];
      kv4_in8<kParts>(x, in, row, t, col + c * 8);
      kv4_in8<kParts>(y, in, row, t, col + half + c * 8);
      if (kParts && in.qw != nullptr) {  // a head's lanes are neighbours (chunks is a power of two), as in splitk_rope_cache
        float ss = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
#pragma unroll
        for (int j = 0; j < 8; ++j) s2 += y[j] * y[j];
        ss += s2;
        for (int o = chunks / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
        const float inv = rsqrtf(ss / D + in.eps);
        const float* nw = is_k ? in.kw : in.qw;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = bf16_to_f32(f32_to_bf16(x[j] * inv * nw[c * 8 + j]));
          y[j] = bf16_to_f32(f32_to_bf16(y[j] * inv * nw[half + c * 8 + j]));
        }
      }
      u16x8 va, vb;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float ra, rb;
        rope_rot(x[j], y[j], cs[c * 8 + j], cs[half + c * 8 + j], ra, rb);
        va[j] = f32_to_bf16(ra);
        vb[j] = f32_to_bf16(rb);
      }
      *reinterpret_cast<u16x8*>(dst + c * 8) = va;
      *reinterpret_cast<u16x8*>(dst + half + c * 8) = vb;
    } else {
      float x[8];
      kv4_in8<kParts>(x, in, row, t, col + c * 8);
      u16x8 v;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        float ra, rb;
        rope_rot(x[2 * p], x[2 * p + 1], cs[c * 4 + p], cs[half + c * 4 + p], ra, rb);
        v[2 * p] = f32_to_bf16(ra);
        v[2 * p + 1] = f32_to_bf16(rb);
      }
      *reinterpret_cast<u16x8*>(dst + c * 8) = v;
    }
  }
  for (int it = threadIdx.x; it < nt * (D / 8); it += kThreads) {
    const int c = it % (D / 8), tt = it / (D / 8);
    float x[8];
    kv4_in8<kParts>(x, in, qkv + (t0 + tt) * qkv_stride, t0 + tt, (nq + nkv + kh) * D + c * 8);
    u16x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = f32_to_bf16(x[j]);
    *reinterpret_cast<u16x8*>(&kv[1][tt][c * 8]) = v;
  }
  __syncthreads();
  // four neighbouring lanes hold a group; D / 8 is a multiple of four
  const long head_bytes = kv4_head_bytes(bs, D);
  const int code_bytes = kv4_code_bytes(bs, D);
  for (int it = threadIdx.x; it < nt * (D / 8) * 2; it += kThreads) {
    const int c = it % (D / 8), which = it / (D / 8) & 1, tt = it / (D / 8) / 2;
    const long slot = slots[t0 + tt];
    const u16x8 v = *reinterpret_cast<const u16x8*>(&kv[which][tt][c * 8]);
    unsigned m = kv4_amax8(v);
    m = max(m, (unsigned)__shfl_xor((int)m, 1, 64));
    m = max(m, (unsigned)__shfl_xor((int)m, 2, 64));
    if (slot < 0 || slot >= nslots) continue;
    const int byte = kv4_scale_byte(m);
    const unsigned codes = kv4_quantise8(v, byte);
    const int off = (int)(slot % bs);
    const long base = (slot / bs * nkv + kh) * head_bytes;
    if (which == 0) {
      *reinterpret_cast<unsigned*>(k_cache + base + off * (D / 2) + c * 4) = codes;
      if ((c & 3) == 0) k_cache[base + code_bytes + (c >> 2) * bs + kv4_key_scale_at(off)] = (unsigned char)byte;
    } else {
#pragma unroll
      for (int p = 0; p < 4; ++p) v_cache[base + (c * 4 + p) * bs + off] = (unsigned char)(codes >> (8 * p));
      if ((c & 3) == 0) v_cache[base + code_bytes + (c >> 2) * bs + off] = (unsigned char)byte;
    }
  }
}

void launch_kv4_write(void* qkv, long qkv_stride, const float* ws, int S, const void* bias, const float* qw,
                      const float* kw, float eps, const long* positions, const long* slots, const float* cos_sin,
                      long max_pos, const Kv4Cache& c, int T, int nq, int mode, hipStream_t s) {
  if (T <= 0) return;
  const int N = (nq + 2 * c.nkv) * c.D;
  const Kv4In in{ws, (long)T * N, S, N, static_cast<const unsigned short*>(bias), qw, kw, eps};
  auto* q = static_cast<unsigned short*>(qkv);
  auto* kc = static_cast<unsigned char*>(c.k);
  auto* vc = static_cast<unsigned char*>(c.v);
  const long nslots = c.blocks * c.block_size;
#define HS_KV4_WRITE(mode_, parts, tok, threads)                                                                      \
  kv4_write_kernel<mode_, parts, tok, threads><<<dim3(cdiv(T, tok), c.nkv), threads, 0, s>>>(                         \
      q, qkv_stride, in, positions, max_pos, slots, cos_sin, kc, vc, nslots, T, nq, c.nkv, c.D, c.block_size)
  if (ws != nullptr) {
    if (mode == 0) HS_KV4_WRITE(0, true, 1, 64);
    else HS_KV4_WRITE(1, true, 1, 64);
  } else {
    if (mode == 0) HS_KV4_WRITE(0, false, 1, 64);
    else HS_KV4_WRITE(1, false, 1, 64);
  }
#undef HS_KV4_WRITE
}

// Rows of slots as bf16: a thread takes 8 dims of a token's key or value.
__global__ __launch_bounds__(256) void kv4_read_kernel(unsigned short* __restrict__ k_out, long k_stride,
                                                       unsigned short* __restrict__ v_out, long v_stride,
                                                       const unsigned char* __restrict__ k_cache,
                                                       const unsigned char* __restrict__ v_cache,
                                                       const long* __restrict__ slots, long nslots, int T, int nkv,
                                                       int D, int bs) {
  const int items = nkv * (D / 8);
  const long it = (long)blockIdx.x * 256 + threadIdx.x;
  const long t = it / (2 * items);
  if (t >= T) return;
  const int e = (int)(it - t * 2 * items), which = e / items, kh = e % items / (D / 8), c = e % (D / 8);
  const long slot = slots[t];
  u32x4 out{0, 0, 0, 0};
  if (slot >= 0 && slot < nslots) {
    const int off = (int)(slot % bs);
    const unsigned char* p = (which == 0 ? k_cache : v_cache) + (slot / bs * nkv + kh) * (long)kv4_head_bytes(bs, D);
    unsigned w = 0;
    if (which == 0) {
      w = *reinterpret_cast<const unsigned*>(p + off * (D / 2) + c * 4);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) w |= (unsigned)p[(c * 4 + j) * bs + off] << (8 * j);
    }
    const int byte = p[kv4_code_bytes(bs, D) + (c >> 2) * bs + (which == 0 ? kv4_key_scale_at(off) : off)];
    const float s = kv4_scale(byte);
    out = byte == kKv4Nan ? u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u}
                          : u32x4{kv4_widen2<0>(w, s), kv4_widen2<1>(w, s), kv4_widen2<2>(w, s), kv4_widen2<3>(w, s)};
  }
  *reinterpret_cast<u32x4*>((which == 0 ? k_out + t * k_stride : v_out + t * v_stride) + kh * D + c * 8) = out;
}

void launch_kv4_read(void* k_out, long k_stride, void* v_out, long v_stride, const Kv4Cache& c, const long* slots, int T,
                     hipStream_t s) {
  if (T <= 0) return;
  const long items = (long)T * 2 * c.nkv * (c.D / 8);
  kv4_read_kernel<<<dim3((items + 255) / 256), 256, 0, s>>>(
      static_cast<unsigned short*>(k_out), k_stride, static_cast<unsigned short*>(v_out), v_stride,
      static_cast<const unsigned char*>(c.k), static_cast<const unsigned char*>(c.v), slots, c.blocks * c.block_size, T,
      c.nkv, c.D, c.block_size);
}

}  // namespace hipserve
