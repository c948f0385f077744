// Decode attention over the 4-bit paged KV cache (layout and format: kv4.h): one query per sequence, the queries of a kv head
// together, the visible context cut over workgroups ("partitions") and merged by a second kernel.
//
//   out[h] = sum_j softmax_j(scale q[h] . k_j) v_j   over the visible j: the last `window` ones and the first `sinks` (all without a window)
//
// What bounds it is the cache's bytes (17 D / 32 per token, head and K or V), so nothing is unpacked that need not be:
//  * scores: K codes go from memory into v_mfma_scale_f32_16x16x128_f8f6f4 as they are, rows = 16 tokens, their scale bytes as its
//    block scales. The other operand is q in two e4m3 numbers: a bf16 value has 8 significant bits, e4m3 has 4, and what the first
//    leaves is one e4m3 number again, so q is exact (values below 2^-14 of the row's largest within 2^-21 of it) where one number alone
//    would lose half of its bits. One power of two per row keeps both in range and goes into the softmax's scale.
//  * P . V: a byte of V is one token's two dims; v_cvt_scalef32_pk_bf16_fp4 applies the token's scale as it widens, two
//    v_perm per pair of tokens sort the two dims. Scales ride in the exponent, so a shift makes one of a byte.
//  * tokens of a 64-key chunk sit so that the lanes that get their scores are the lanes that feed their P: no exchange.
//  * softmax in base 2, 32 bits; P is rounded to bf16 (2^-8 relative a probability, what the bf16 product takes), its
//    sum is not. The running maximum moves only when a score is over 2^8 above it, so most chunks exchange nothing.
//  * the next chunk's loads are issued before the current chunk's products, from two register sets.
// Hidden keys: the score is -inf whatever the key holds, and the value's scale is replaced, as 0 * NaN is not 0.
#include "hipserve/kv4.h"

namespace hipserve {

constexpr int kKv4Chunk = 64;

// the visible keys of a row as chunks of 64: the chunks of the first `sinks` keys, then those from the window's first key on
struct Kv4Chunks {
  int lo, sink, first, count;  // first key of the window, chunks of sinks, first chunk of the window, chunks in all
  HS_DEVICE Kv4Chunks(int ctx, int window, int sinks) {
    lo = window > 0 ? max(0, ctx - window) : 0;
    first = lo / kKv4Chunk;
    sink = min((min(sinks, lo) + kKv4Chunk - 1) / kKv4Chunk, first);
    count = ctx > 0 ? sink + (ctx + kKv4Chunk - 1) / kKv4Chunk - first : 0;
  }
  HS_DEVICE int token(int v) const { return (v < sink ? v : v - sink + first) * kKv4Chunk; }
};

// 16 values as e4m3 numbers hi + lo / 16
HS_DEVICE void kv4_split16(const float (&x)[16], u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    int h = 0, l = 0;
    h = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w], x[4 * w + 1], h, false);
    h = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w + 2], x[4 * w + 3], h, true);
    const float r0 = x[4 * w] - __builtin_amdgcn_cvt_f32_fp8(h, 0), r1 = x[4 * w + 1] - __builtin_amdgcn_cvt_f32_fp8(h, 1);
    const float r2 = x[4 * w + 2] - __builtin_amdgcn_cvt_f32_fp8(h, 2), r3 = x[4 * w + 3] - __builtin_amdgcn_cvt_f32_fp8(h, 3);
    l = __builtin_amdgcn_cvt_pk_fp8_f32(r0 * 16.f, r1 * 16.f, l, false);
    l = __builtin_amdgcn_cvt_pk_fp8_f32(r2 * 16.f, r3 * 16.f, l, true);
    hi[w] = (unsigned)h;
    lo[w] = (unsigned)l;
  }
}

HS_DEVICE i32x8 kv4_pad(const u32x4 a, const u32x4 b) {
  return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

template <int kByte>  // 16 tokens x 128 dims of FP4 under byte kByte of ks, times q's two parts
HS_DEVICE f32x4 kv4_scores(const u32x4 k, unsigned ks, const i32x8 hi, const i32x8 lo) {
  const i32x8 a = kv4_pad(k, u32x4{0, 0, 0, 0});
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, lo, s, 4, 0, kByte, (int)ks, 0, 123);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, hi, s, 4, 0, kByte, (int)ks, 0, 127);
}

// bytes of a word whose bit in `keep` (bit i: byte i) is set, 127 (scale 1) for the others
HS_DEVICE unsigned kv4_keep_scales(unsigned w, unsigned keep) {
  const unsigned m = (((keep & 15u) * 0x00204081u) & 0x01010101u) * 255u;
  return (w & m) | (0x7f7f7f7fu & ~m);
}

template <int D, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2, 8))) void kv4_decode_kernel(Kv4Attn a, const int* __restrict__ ctx_lens,
                                                            float* __restrict__ tmp_out, float* __restrict__ tmp_ml,
                                                            int part_chunks, int max_parts,
                                                            unsigned short* __restrict__ out16) {
  constexpr int NG = D / 32;             // scale groups of a head
  constexpr int NK = D == 64 ? 2 : 4;    // K loads a chunk: at 64 dims the upper lanes of a product take other tokens
  const int part = blockIdx.x, kh = blockIdx.y, b = blockIdx.z;
  const int nq = a.nq, nkv = a.cache.nkv, bs = a.cache.block_size, G = nq / nkv;
  const int ctx = min(ctx_lens[b], a.bt_width * bs);
  const Kv4Chunks chunks(ctx, a.window, a.sinks);
  const int c0 = part * part_chunks, c1 = min(c0 + part_chunks, chunks.count);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned short* out = static_cast<unsigned short*>(a.out) + (long)b * a.out_stride + (long)kh * G * D;
  if (c0 >= c1) {
    if (part == 0)  // a row without keys
      for (int i = tid; i < G * D; i += 64 * W) {
        out[i] = 0;
        if (out16 != nullptr) store_o16(out16, (long)b * a.out_stride, kh * G * D + i, 0);
      }
    return;
  }
  const int col = lane & 15, grp = lane >> 4;

  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* olds = reinterpret_cast<float*>(smem);              // [W][G][D]
  float* red = olds + W * G * D;                             // [W][G][2]
  int* pages = reinterpret_cast<int*>(red + W * G * 2);      // 4 a chunk: a run of 16 tokens lies in one page
  const int* bt = a.block_tables + (long)b * a.bt_stride;
  const int bsh = __builtin_ctz(bs), bmask = bs - 1;
  for (int i = tid; i < (c1 - c0) * 4; i += 64 * W) {
    const int tok = chunks.token(c0 + (i >> 2)) + 16 * (i & 3);
    pages[i] = tok < ctx ? kv4_page(bt[tok >> bsh], a.cache.blocks) : -1;
  }
  __syncthreads();

  // ---- loads of a chunk
  const long head_bytes = kv4_head_bytes(bs, D), page_bytes = head_bytes * nkv;
  const int code_bytes = kv4_code_bytes(bs, D);
  const unsigned char* kbase = static_cast<const unsigned char*>(a.cache.k) + kh * head_bytes;
  const unsigned char* vbase = static_cast<const unsigned char*>(a.cache.v) + kh * head_bytes;
  // keys: lane (m, g) loads the 32 dims g of tokens 16 (m >> 2) + 4 t + (m & 3) (64 dims: group g & 1, t = 2 u + (g >> 1))
  const int kgrp = D == 64 ? (grp & 1) : min(grp, NG - 1);
  const int krow = (col & 3) + (D == 64 ? 4 * (grp >> 1) : 0);
  struct Chunk {
    u32x4 k[NK], v[NG], vs[NG];
    unsigned ks;
    int page;  // of this lane's 16 tokens
  };
  auto load = [&](int c, Chunk& ch) {
    c = min(c, c1 - 1);
    const int tok = chunks.token(c);
    const int kp = pages[(c - c0) * 4 + (col >> 2)], vp = pages[(c - c0) * 4 + grp];
    const int ko = (tok + 16 * (col >> 2)) & bmask, vo = (tok + 16 * grp) & bmask;
    const unsigned char* k = kbase + (long)max(kp, 0) * page_bytes;
    const unsigned char* kc = k + (ko + krow) * (D / 2) + 16 * kgrp;
#pragma unroll
    for (int u = 0; u < NK; ++u)
      ch.k[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kc + u * (16 / NK) * (D / 2)));
    ch.ks = *reinterpret_cast<const unsigned*>(k + code_bytes + kgrp * bs + ko + 4 * (col & 3));
    const unsigned char* v = vbase + (long)max(vp, 0) * page_bytes;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      ch.v[n] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(v + (16 * n + col) * bs + vo));
      ch.vs[n] = *reinterpret_cast<const u32x4*>(v + code_bytes + n * bs + vo);
    }
    ch.page = vp;
  };

  // ---- q: head `col`, dims 16 grp .. and 64 + 16 grp .. of the product's k
  i32x8 qhi[D == 64 ? 2 : 1], qlo[D == 64 ? 2 : 1];
  float sl;
  {
    const unsigned short* qp = static_cast<const unsigned short*>(a.q) + (long)b * a.q_stride + (long)(kh * G + col) * D;
    constexpr int NH = D == 64 ? 1 : 2;
    u16x8 raw[NH][2];
    unsigned am = 0;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d0 = 64 * h + 16 * grp + 8 * e;
        raw[h][e] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
        if (col < G && d0 < D) raw[h][e] = *reinterpret_cast<const u16x8*>(qp + d0);
        am = max(am, kv4_amax8(raw[h][e]));
      }
    am = max(am, (unsigned)__shfl_xor((int)am, 16, 64));
    am = max(am, (unsigned)__shfl_xor((int)am, 32, 64));
    const int eb = min(max((int)(am >> 7), 8), 254);  // the largest value comes to [128, 256)
    float up = __uint_as_float((unsigned)(261 - eb) << 23);
    if (a.scale < 0.f) up = -up;  // the multiplier below is not negative: the largest product has the largest score
    // never 0: a hidden key's -inf has to stay one
    sl = am >= 0x7f80u ? NAN : fmaxf(fabsf(a.scale) * kLog2E * __uint_as_float((unsigned)(eb - 7) << 23), 1.17549435e-38f);
    u32x4 hi[NH], lo[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      float x[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = am >= 0x7f80u ? 0.f : bf16_to_f32(raw[h][j >> 3][j & 7]) * up;
      kv4_split16(x, hi[h], lo[h]);
    }
    const u32x4 z{0, 0, 0, 0};
    if constexpr (D == 64) {
      qhi[0] = kv4_pad(hi[0], z);
      qhi[1] = kv4_pad(z, hi[0]);
      qlo[0] = kv4_pad(lo[0], z);
      qlo[1] = kv4_pad(z, lo[0]);
    } else {
      qhi[0] = kv4_pad(hi[0], hi[1]);
      qlo[0] = kv4_pad(lo[0], lo[1]);
    }
  }

  f32x4 o[NG][2];  // rows: heads 4 grp + r, columns: dims 32 n + 2 col (+ 1)
#pragma unroll
  for (int n = 0; n < NG; ++n) o[n][0] = o[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -1e30f, l_run = 0.f;  // of head `col`; the sum over this lane's tokens alone

  auto compute = [&](int c, const Chunk& ch) {
    const int tok = chunks.token(c);
    // ---- scores of tokens tok + 16 grp + 4 t + r for head `col`
    f32x4 st[4];
    if constexpr (D == 64) {
      const unsigned sh = ch.ks >> (8 * (grp >> 1));  // bytes 0 and 2: this lane's tokens of the two loads
      const unsigned s0 = grp < 2 ? sh : 0x7f7f7f7fu, s1 = grp < 2 ? 0x7f7f7f7fu : sh;
      st[0] = kv4_scores<0>(ch.k[0], s0, qhi[0], qlo[0]);
      st[1] = kv4_scores<0>(ch.k[0], s1, qhi[1], qlo[1]);
      st[2] = kv4_scores<2>(ch.k[1], s0, qhi[0], qlo[0]);
      st[3] = kv4_scores<2>(ch.k[1], s1, qhi[1], qlo[1]);
    } else {
      const unsigned ks = D == 96 && grp == 3 ? 0x7f7f7f7fu : ch.ks;
      st[0] = kv4_scores<0>(ch.k[0], ks, qhi[0], qlo[0]);
      st[1] = kv4_scores<1>(ch.k[1], ks, qhi[0], qlo[0]);
      st[2] = kv4_scores<2>(ch.k[2], ks, qhi[0], qlo[0]);
      st[3] = kv4_scores<3>(ch.k[3], ks, qhi[0], qlo[0]);
    }
    unsigned vis = 0xffffu;  // which of this lane's 16 tokens are visible
    const bool whole = tok + kKv4Chunk <= ctx && (tok >= chunks.lo || tok + kKv4Chunk <= a.sinks);
    const bool edge = !whole || __any(ch.page < 0);
    if (edge) {
      vis = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = tok + 16 * grp + i;
        if (ch.page >= 0 && j < ctx && (j >= chunks.lo || j < a.sinks)) vis |= 1u << i;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (!(vis >> i & 1)) st[i >> 2][i & 3] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, st[i >> 2][i & 3]);
    mx *= sl;  // a row of zeros has sl > 0 too; of NaN it stays NaN and fmaxf drops it
    if (__any(mx > m_run + 8.f)) {
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float m_new = fmaxf(m_run, mx);
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float a_r = __shfl(alpha, 4 * grp + r, 64);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          o[n][0][r] *= a_r;
          o[n][1][r] *= a_r;
        }
      }
    }
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
    bf16x8 p[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i >> 2][i & 3], sl, -m_run));
      ps[i & 3] += x;
      p[i >> 3][i & 7] = static_cast<__bf16>(x);
    }
    l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
    // ---- O += P . V
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      u32x4 even[2], odd[2];
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // tokens 4 q .. 4 q + 3 of the lane's 16
        const unsigned w = ch.v[n][q];
        unsigned s = ch.vs[n][q];
        if (edge) s = kv4_keep_scales(s, vis >> (4 * q));
        const unsigned x0 = kv4_widen2<0>(w, __uint_as_float(s << 23)), x1 = kv4_widen2<1>(w, __uint_as_float(s << 15));
        const unsigned x2 = kv4_widen2<2>(w, __uint_as_float(s << 7)), x3 = kv4_widen2<3>(w, __uint_as_float(s >> 1));
        even[q >> 1][2 * (q & 1)] = __builtin_amdgcn_perm(x1, x0, 0x05040100u);
        odd[q >> 1][2 * (q & 1)] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
        even[q >> 1][2 * (q & 1) + 1] = __builtin_amdgcn_perm(x3, x2, 0x05040100u);
        odd[q >> 1][2 * (q & 1) + 1] = __builtin_amdgcn_perm(x3, x2, 0x07060302u);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        o[n][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p[s], __builtin_bit_cast(bf16x8, even[s]), o[n][0], 0, 0, 0);
        o[n][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p[s], __builtin_bit_cast(bf16x8, odd[s]), o[n][1], 0, 0, 0);
      }
    }
  };

  Chunk A, B;
  int c = c0 + wave;
  if (c < c1) {
    load(c, A);
    for (; c + W < c1; c += 2 * W) {
      load(c + W, B);
      __builtin_amdgcn_sched_barrier(0);
      compute(c, A);
      load(c + 2 * W, A);
      __builtin_amdgcn_sched_barrier(0);
      compute(c + W, B);
    }
    if (c < c1) compute(c, A);
  }

  // ---- the waves' results
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  if (lane < G) {
    red[(wave * G + lane) * 2] = m_run;
    red[(wave * G + lane) * 2 + 1] = l_run;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (4 * grp + r < G) {
      float2* dst = reinterpret_cast<float2*>(olds + (wave * G + 4 * grp + r) * D);
#pragma unroll
      for (int n = 0; n < NG; ++n) dst[16 * n + col] = float2{o[n][0][r], o[n][1][r]};
    }
  __syncthreads();
  const bool one = chunks.count <= part_chunks;
  for (int i = tid; i < G * D; i += 64 * W) {
    const int h = i / D, d = i % D;
    float M = -1e30f;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, red[(w * G + h) * 2]);
    float L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = __builtin_amdgcn_exp2f(red[(w * G + h) * 2] - M);
      L += red[(w * G + h) * 2 + 1] * f;
      acc += olds[(w * G + h) * D + d] * f;
    }
    const float y = L == 0.f ? 0.f : acc / L;
    if (one) {
      const unsigned short ob = f32_to_bf16(y);
      out[i] = ob;
      if (out16 != nullptr) store_o16(out16, (long)b * a.out_stride, kh * G * D + i, ob);
    } else {
      const long base = ((long)b * nq + kh * G + h) * max_parts + part;
      tmp_out[base * D + d] = y;
      if (d == 0) {
        tmp_ml[base * 2] = M;
        tmp_ml[base * 2 + 1] = L;
      }
    }
  }
}

// Merges a row's partitions: a workgroup per (head, sequence), lane groups of D lanes take every kGroups-th partition, four at a time.
template <int D>
__global__ __launch_bounds__(384) void kv4_decode_merge_kernel(Kv4Attn a, const int* __restrict__ ctx_lens,
                                                               const float* __restrict__ tmp_out,
                                                               const float* __restrict__ tmp_ml, int part_chunks,
                                                               int max_parts, unsigned short* __restrict__ out16) {
  constexpr int kGroups = 384 / D;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, d = tid % D, grp = tid / D;
  const Kv4Chunks chunks(min(ctx_lens[b], a.bt_width * a.cache.block_size), a.window, a.sinks);
  if (chunks.count <= part_chunks) return;
  const int np = (chunks.count + part_chunks - 1) / part_chunks;
  const long base = ((long)b * a.nq + h) * max_parts;
  float M = -1e30f;
  for (int p = tid & 63; p < np; p += 64) M = fmaxf(M, tmp_ml[(base + p) * 2]);
  M = wave_max(M);
  float L[4] = {0.f, 0.f, 0.f, 0.f}, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int p = grp; p < np; p += 4 * kGroups)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long q = base + min(p + u * kGroups, np - 1);
      const float w = __builtin_amdgcn_exp2f(tmp_ml[q * 2] - M) * tmp_ml[q * 2 + 1], x = tmp_out[q * D + d];
      if (p + u * kGroups < np) {
        L[u] += w;
        acc[u] += w * x;
      }
    }
  __shared__ float sums[2][kGroups][D];
  sums[0][grp][d] = (L[0] + L[1]) + (L[2] + L[3]);
  sums[1][grp][d] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
  __syncthreads();
  if (grp == 0) {
    float l = 0.f, y = 0.f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      l += sums[0][g][d];
      y += sums[1][g][d];
    }
    const unsigned short ob = f32_to_bf16(l == 0.f ? 0.f : y / l);
    static_cast<unsigned short*>(a.out)[(long)b * a.out_stride + (long)h * D + d] = ob;
    if (out16 != nullptr) store_o16(out16, (long)b * a.out_stride, h * D + d, ob);
  }
}

template <int D>
static void kv4_decode(const Kv4Attn& a, const int* ctx, float* tmp_out, float* tmp_ml, int B, int part_size, int max_parts,
                       unsigned short* out16, hipStream_t s) {
  const int G = a.nq / a.cache.nkv, chunks = part_size / kKv4Chunk;
  const dim3 grid(max_parts, a.cache.nkv, B);
  auto smem = [&](int w) { return (size_t)w * G * (D + 2) * sizeof(float) + (size_t)chunks * 4 * sizeof(int); };
  kv4_decode_kernel<D, 4><<<grid, 256, smem(4), s>>>(a, ctx, tmp_out, tmp_ml, chunks, max_parts, out16);
  if (max_parts > 1)
    kv4_decode_merge_kernel<D><<<dim3(a.nq, B), 384, 0, s>>>(a, ctx, tmp_out, tmp_ml, chunks, max_parts, out16);
}

void launch_kv4_decode(const Kv4Attn& a, const int* context_lens, float* tmp_out, float* tmp_ml, int B, int part_size,
                       int max_parts, void* out16, hipStream_t s) {
  if (B <= 0) return;
  auto* o16 = static_cast<unsigned short*>(out16);
  if (a.cache.D == 128) kv4_decode<128>(a, context_lens, tmp_out, tmp_ml, B, part_size, max_parts, o16, s);
  else if (a.cache.D == 96) kv4_decode<96>(a, context_lens, tmp_out, tmp_ml, B, part_size, max_parts, o16, s);
  else kv4_decode<64>(a, context_lens, tmp_out, tmp_ml, B, part_size, max_parts, o16, s);
}

}  // namespace hipserve
