// Decode attention over the 4-bit paged KV cache (layout and format: kv4.h): one query per sequence, the queries of a kv head
// together, the visible context cut over workgroups ("partitions") and merged by a second kernel.
//
//   out[h] = sum_j softmax_j(scale q[h] . k_j) v_j   over the visible j: the last `window` ones and the first `sinks` (all without a window)
//
// What bounds it is the cache's bytes (17 D / 32 per token, head and K or V), so nothing is unpacked that need not be:
//  * scores: K codes go from memory into v_mfma_scale_f32_16x16x128_f8f6f4 as they are, rows = 16 tokens, their scale bytes as its
//    block scales. The other operand is q in two e4m3 numbers: a bf16 value has 8 significant bits, e4m3 has 4, and what the first
//    leaves is one e4m3 number again, so q is exact (values below 2^-13 of the largest of their 32 dims within 2^-21 of it) where one number
//    alone would lose half of its bits. A power of two per 32 dims, the keys' groups, keeps both in range: the scale bytes of that operand.
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

// Which chunks a workgroup takes. All sequences' chunks are cut into runs of one length, so that ragged batches fill the chip evenly:
// about kKv4Slots workgroups over the kv heads, what the chip holds at once (two a compute unit). A second round of workgroups costs 6 - 9 us
// (the chain of lengths, block table and first keys before a wave has work: 64 sequences of 8192 in 512 / 1024 / 2048 workgroups
// 104 / 113 / 124 us). Every wave works this out for itself from all lengths.
constexpr int kKv4Slots = 512;
constexpr int kKv4Waves = 4;  // of a workgroup: 2 and 8 take 1.02 - 1.2 times as long

// sum or maximum (of numbers >= 0) over a wave, and sums up to and with every lane, on the DPP crossbar
template <int kCtrl, int kRows>
HS_DEVICE int kv4_dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, kCtrl, kRows, 0xf, false); }
HS_DEVICE int kv4_scan(int v) {
  v += kv4_dpp<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
  v += kv4_dpp<0x112, 0xf>(v);
  v += kv4_dpp<0x114, 0xf>(v);
  v += kv4_dpp<0x118, 0xf>(v);
  v += kv4_dpp<0x142, 0xa>(v);  // row_bcast:15 -> rows 1, 3
  v += kv4_dpp<0x143, 0xc>(v);  // row_bcast:31 -> rows 2, 3
  return v;
}
HS_DEVICE int kv4_wave_sum(int v) { return __builtin_amdgcn_readlane(kv4_scan(v), 63); }
HS_DEVICE int kv4_wave_max(int v) {
  v = max(v, kv4_dpp<0x111, 0xf>(v));
  v = max(v, kv4_dpp<0x112, 0xf>(v));
  v = max(v, kv4_dpp<0x114, 0xf>(v));
  v = max(v, kv4_dpp<0x118, 0xf>(v));
  v = max(v, kv4_dpp<0x142, 0xa>(v));
  v = max(v, kv4_dpp<0x143, 0xc>(v));
  return __builtin_amdgcn_readlane(v, 63);
}

struct Kv4Run {
  int chunks;        // of a run
  int b, part, ctx;  // the workgroup's sequence (B: it has none), its partition, the sequence's length
};

HS_DEVICE int kv4_length(const int* __restrict__ ctx_lens, int B, int b, int cap) { return b < B ? min(ctx_lens[b], cap) : 0; }

// `own` >= 0: of that sequence; else of workgroup w among the runs of all sequences, where one without keys has one run
HS_DEVICE Kv4Run kv4_run(const int* __restrict__ ctx_lens, int B, int cap, int window, int sinks, int nkv, int max_parts,
                         int own, int w) {
  const int lane = threadIdx.x & 63;
  const int len0 = kv4_length(ctx_lens, B, lane, cap);
  int total = Kv4Chunks(len0, window, sinks).count, most = total;
  for (int b = 64 + lane; b < B; b += 64) {
    const int n = Kv4Chunks(kv4_length(ctx_lens, B, b, cap), window, sinks).count;
    total += n;
    most = max(most, n);
  }
  total = kv4_wave_sum(total);
  most = kv4_wave_max(most);
  // a sequence's last run is half a run short on average. The quotient in 32-bit floats, and one more: never below the true one by
  // what the grid does not cover
  const int slots = max(kKv4Slots - B * nkv / 2, kKv4Slots / 2);
  int run = max((int)((float)total * (float)nkv / (float)slots) + 1, (most + max_parts - 1) / max_parts);
  run = (run + kKv4Waves - 1) / kKv4Waves * kKv4Waves;
  if (own >= 0) return {run, own, 0, kv4_length(ctx_lens, B, own, cap)};
  int before = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    const int len = b0 == 0 ? len0 : kv4_length(ctx_lens, B, b0 + lane, cap);
    const int n = b0 + lane < B ? max((Kv4Chunks(len, window, sinks).count + run - 1) / run, 1) : 0;
    const int upto = before + kv4_scan(n);
    const unsigned long after = __ballot(upto > w);
    if (after) {
      const int l = __builtin_ctzl(after);
      return {run, b0 + l, w - __builtin_amdgcn_readlane(upto - n, l), __builtin_amdgcn_readlane(len, l)};
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return {run, B, 0, 0};
}

HS_DEVICE i32x8 kv4_pad(const u32x4 a, const u32x4 b) {
  return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

template <int kByte>  // 16 tokens x 128 dims of FP4 under byte kByte of ks, times q's two parts under bytes 0 and 1 of qs
HS_DEVICE f32x4 kv4_scores(const u32x4 k, unsigned ks, const i32x8 hi, const i32x8 lo, int qs) {
  const i32x8 a = kv4_pad(k, u32x4{0, 0, 0, 0});
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, lo, s, 4, 0, kByte, (int)ks, 1, qs);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, hi, s, 4, 0, kByte, (int)ks, 0, qs);
}

// bytes of a word whose bit in `keep` (bit i: byte i) is set, 127 (scale 1) for the others
HS_DEVICE unsigned kv4_keep_scales(unsigned w, unsigned keep) {
  const unsigned m = (((keep & 15u) * 0x00204081u) & 0x01010101u) * 255u;
  return (w & m) | (0x7f7f7f7fu & ~m);
}

template <int D>
__global__ __launch_bounds__(64 * kKv4Waves) __attribute__((amdgpu_waves_per_eu(2, 8))) void kv4_decode_kernel(Kv4Attn a, const int* __restrict__ ctx_lens,
                                                            float* __restrict__ tmp_out, float* __restrict__ tmp_ml,
                                                            int B, int max_parts, unsigned short* __restrict__ out16) {
  constexpr int NG = D / 32;             // scale groups of a head
  constexpr int W = kKv4Waves;
  constexpr int NK = D == 64 ? 2 : 4;    // K loads a chunk: at 64 dims the upper lanes of a product take other tokens
  const int kh = blockIdx.y;
  const int nq = a.nq, nkv = a.cache.nkv, bs = a.cache.block_size, G = nq / nkv;
  const int cap = a.bt_width * bs;
  Kv4Run run{INT32_MAX / kKv4Chunk, (int)blockIdx.x, 0, 0};
  if (max_parts > 1) run = kv4_run(ctx_lens, B, cap, a.window, a.sinks, nkv, max_parts, -1, blockIdx.x);
  else run.ctx = min(ctx_lens[run.b], cap);
  if (run.b >= B) return;
  const int b = run.b, part = run.part, part_chunks = run.chunks, ctx = run.ctx;
  const Kv4Chunks chunks(ctx, a.window, a.sinks);
  const int c0 = part * part_chunks, c1 = min(c0 + part_chunks, chunks.count);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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
  const int* bt = a.block_tables + (long)b * a.bt_stride;
  const int bsh = __builtin_ctz(bs), bmask = bs - 1;

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
  // a run of 16 tokens lies in one page: the pages of a lane's keys and values. They are asked for a chunk before its loads, and
  // before the loads of the chunk between, so that the wait for them is for nothing younger
  struct Pages {
    int k, v;
  };
  auto pages = [&](int c) {
    const int tok = chunks.token(min(c, c1 - 1));
    return Pages{bt[min(tok + 16 * (col >> 2), ctx - 1) >> bsh], bt[min(tok + 16 * grp, ctx - 1) >> bsh]};
  };
  auto load = [&](int c, const Pages& pg, Chunk& ch) {
    const int tok = chunks.token(min(c, c1 - 1));
    const int kp = kv4_page(pg.k, a.cache.blocks), vp = kv4_page(pg.v, a.cache.blocks);
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

  // ---- q: head `col`, dims 16 grp .. and 64 + 16 grp .. of the product's k; on its way before the first chunk
  constexpr int NH = D == 64 ? 1 : 2;
  u16x8 raw[NH][2];
  {
    const unsigned short* qp = static_cast<const unsigned short*>(a.q) + (long)b * a.q_stride + (long)(kh * G + col) * D;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d0 = 64 * h + 16 * grp + 8 * e;
        raw[h][e] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
        if (col < G && d0 < D) raw[h][e] = *reinterpret_cast<const u16x8*>(qp + d0);
      }
  }
  Chunk A, B_;
  Pages pg;
  const int c = c0 + wave;
  if (c < c1) {
    pg = pages(c);
    const Pages next = pages(c + W);
    load(c, pg, A);
    pg = next;
  }
  i32x8 qhi[D == 64 ? 2 : 1], qlo[D == 64 ? 2 : 1];
  int qs;  // of the dims that this lane's 32 of the product's k are: 32 (grp & 1) .. of 64 dims, 32 grp .. of more
  const float sl = kv4_score_scale(a.scale);
  {
    int own[NH];  // of dims 64 h + 32 (grp >> 1) .., which lanes of two grp hold
    u32x4 hi[NH], lo[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      unsigned am = max(kv4_amax8(raw[h][0]), kv4_amax8(raw[h][1]));
      am = max(am, (unsigned)__shfl_xor((int)am, 16, 64));
      own[h] = kv4_query_scales(am);
      const float down = kv4_scale(own[h] & 255), down16 = kv4_scale(own[h] >> 8 & 255);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        u32x2 x, y;
        kv4_split8(raw[h][e], down, down16, x, y);
        hi[h][2 * e] = x[0];
        hi[h][2 * e + 1] = x[1];
        lo[h][2 * e] = y[0];
        lo[h][2 * e + 1] = y[1];
      }
    }
    const int from = col + 32 * (grp & 1);
    qs = __shfl(own[0], from, 64);
    if constexpr (NH == 2) {
      const int second = __shfl(own[1], from, 64);
      if (grp >= 2) qs = second;
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
  float m_run = kKv4Least, l_run = 0.f;      // of head `col`; the sum over this lane's tokens alone
  bool far = false;                          // of some head of the wave

  auto compute = [&](int c, Chunk& ch) {
    const int tok = chunks.token(c);
    // ---- scores of tokens tok + 16 grp + 4 t + r for head `col`
    f32x4 st[4];
    if constexpr (D == 64) {
      const unsigned sh = ch.ks >> (8 * (grp >> 1));  // bytes 0 and 2: this lane's tokens of the two loads
      const unsigned s0 = grp < 2 ? sh : 0x7f7f7f7fu, s1 = grp < 2 ? 0x7f7f7f7fu : sh;
      st[0] = kv4_scores<0>(ch.k[0], s0, qhi[0], qlo[0], qs);
      st[1] = kv4_scores<0>(ch.k[0], s1, qhi[1], qlo[1], qs);
      st[2] = kv4_scores<2>(ch.k[1], s0, qhi[0], qlo[0], qs);
      st[3] = kv4_scores<2>(ch.k[1], s1, qhi[1], qlo[1], qs);
    } else {
      const unsigned ks = D == 96 && grp == 3 ? 0x7f7f7f7fu : ch.ks;
      st[0] = kv4_scores<0>(ch.k[0], ks, qhi[0], qlo[0], qs);
      st[1] = kv4_scores<1>(ch.k[1], ks, qhi[0], qlo[0], qs);
      st[2] = kv4_scores<2>(ch.k[2], ks, qhi[0], qlo[0], qs);
      st[3] = kv4_scores<3>(ch.k[3], ks, qhi[0], qlo[0], qs);
    }
    const bool whole = tok + kKv4Chunk <= ctx && (tok >= chunks.lo || tok + kKv4Chunk <= a.sinks);
    if (!whole || __any(ch.page < 0)) {
      // which of this lane's 16 tokens are visible, as bits: below ctx, and in the window or among the sinks
      const int j0 = tok + 16 * grp;
      auto below = [](int n) { return n <= 0 ? 0u : n >= 16 ? 0xffffu : (1u << n) - 1u; };
      const unsigned vis = ch.page < 0 ? 0u : below(ctx - j0) & (~below(chunks.lo - j0) | below(a.sinks - j0));
#pragma unroll
      for (int i = 0; i < 16; ++i) st[i >> 2][i & 3] = vis >> i & 1 ? st[i >> 2][i & 3] : -INFINITY;
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) ch.vs[n][q] = kv4_keep_scales(ch.vs[n][q], vis >> (4 * q));
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
      far = __any(kv4_far(m_run));
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
    float by = sl;
    if (far) {
#pragma unroll
      for (int i = 0; i < 16; ++i) st[i >> 2][i & 3] *= sl;
      by = 1.f;
    }
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
    bf16x8 p[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i >> 2][i & 3], by, -m_run));
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
        const unsigned s = ch.vs[n][q];
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

  if (c < c1) {
    int i = c;
    for (; i + W < c1; i += 2 * W) {
      Pages next = pages(i + 2 * W);
      load(i + W, pg, B_);
      pg = next;
      __builtin_amdgcn_sched_barrier(0);
      compute(i, A);
      next = pages(i + 3 * W);
      load(i + 2 * W, pg, A);
      pg = next;
      __builtin_amdgcn_sched_barrier(0);
      compute(i + W, B_);
    }
    if (i < c1) compute(i, A);
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
    float M = kKv4Least;
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

// Merges a row's partitions: a workgroup per (head, sequence), D / 4 lanes of four dims a partition, four partitions of a lane at a
// time. Few waves, as rows of one partition have nothing to merge: 2048 workgroups of 16 waves that only found that out took 9 us.
template <int D>
__global__ __launch_bounds__(256) void kv4_decode_merge_kernel(Kv4Attn a, const int* __restrict__ ctx_lens,
                                                               const float* __restrict__ tmp_out,
                                                               const float* __restrict__ tmp_ml, int B, int max_parts,
                                                               unsigned short* __restrict__ out16) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, d4 = tid % kLanes, grp = tid / kLanes;
  const Kv4Run run = kv4_run(ctx_lens, B, a.bt_width * a.cache.block_size, a.window, a.sinks, a.cache.nkv, max_parts, b, 0);
  const int count = Kv4Chunks(run.ctx, a.window, a.sinks).count;
  if (count <= run.chunks) return;
  const int np = (count + run.chunks - 1) / run.chunks;
  const long base = ((long)b * a.nq + h) * max_parts;
  float M = kKv4Least;
  for (int p = tid & 63; p < np; p += 64) M = fmaxf(M, tmp_ml[(base + p) * 2]);
  M = wave_max(M);
  float L[4] = {0.f, 0.f, 0.f, 0.f};
  f32x4 acc[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (grp < kGroups)
    for (int p = grp; p < np; p += 4 * kGroups)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const long q = base + min(p + u * kGroups, np - 1);
        const float w = __builtin_amdgcn_exp2f(tmp_ml[q * 2] - M) * tmp_ml[q * 2 + 1];
        const f32x4 x = *reinterpret_cast<const f32x4*>(tmp_out + q * D + 4 * d4);
        if (p + u * kGroups < np) {
          L[u] += w;
          acc[u] += w * x;
        }
      }
  __shared__ f32x4 sums[kGroups][kLanes];
  __shared__ float ls[kGroups];
  if (grp < kGroups) {
    sums[grp][d4] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
    if (d4 == 0) ls[grp] = (L[0] + L[1]) + (L[2] + L[3]);
  }
  __syncthreads();
  if (tid < D) {
    float l = 0.f, y = 0.f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      l += ls[g];
      y += sums[g][tid >> 2][tid & 3];
    }
    const unsigned short ob = f32_to_bf16(l == 0.f ? 0.f : y / l);
    static_cast<unsigned short*>(a.out)[(long)b * a.out_stride + (long)h * D + tid] = ob;
    if (out16 != nullptr) store_o16(out16, (long)b * a.out_stride, h * D + tid, ob);
  }
}

template <int D>
static void kv4_decode(const Kv4Attn& a, const int* ctx, float* tmp_out, float* tmp_ml, int B, int max_parts,
                       unsigned short* out16, hipStream_t s) {
  const int nkv = a.cache.nkv, G = a.nq / nkv;
  // one partition: a workgroup per sequence and kv head; else the runs of kv4_run, at most so many and one more a sequence
  const dim3 grid(max_parts > 1 ? cdiv(kKv4Slots, nkv) + B : B, nkv);
  const size_t smem = (size_t)kKv4Waves * G * (D + 2) * sizeof(float);
  kv4_decode_kernel<D><<<grid, 64 * kKv4Waves, smem, s>>>(a, ctx, tmp_out, tmp_ml, B, max_parts, out16);
  if (max_parts > 1) kv4_decode_merge_kernel<D><<<dim3(a.nq, B), 256, 0, s>>>(a, ctx, tmp_out, tmp_ml, B, max_parts, out16);
}

void launch_kv4_decode(const Kv4Attn& a, const int* context_lens, float* tmp_out, float* tmp_ml, int B, int max_parts,
                       void* out16, hipStream_t s) {
  if (B <= 0) return;
  auto* o16 = static_cast<unsigned short*>(out16);
  if (a.cache.D == 128) kv4_decode<128>(a, context_lens, tmp_out, tmp_ml, B, max_parts, o16, s);
  else if (a.cache.D == 96) kv4_decode<96>(a, context_lens, tmp_out, tmp_ml, B, max_parts, o16, s);
  else kv4_decode<64>(a, context_lens, tmp_out, tmp_ml, B, max_parts, o16, s);
}

}  // namespace hipserve
