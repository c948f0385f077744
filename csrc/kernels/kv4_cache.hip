// Writers and reader of the 4-bit paged KV cache (layout and format: kv4.h).
//
// kv4_write: the rotary embedding of a step's queries and keys and the step's keys and values quantised into their slots. The
// arithmetic up to the quantisation is rope_cache's and splitk_rope_cache's, rounding for rounding (bf16 after the sum, the bias, the
// norm and the rotation), so the cache holds the 4-bit rounding of what a bf16 cache would hold and the queries are the same bits.
// A workgroup takes tokens of one kv head and its queries: rotated keys and the values go through LDS as bf16, four lanes
// then hold a group of 32 dims (the two halves of a rotated head need not be whole groups: heads of 96).
//
// Bound by bytes for a prompt step and by the chain of loads for a decode step, hence two kernels: a token a workgroup, one
// pass of loads for queries, key and value together; and runs of 16 tokens of a page, whose values leave as 16-byte stores (a
// byte is one token's two dims, so single tokens store bytes). Workgroups of a row's heads follow each other: rows of several heads are
// neighbouring bytes (91560 rows read 91.0 us with the heads far apart, 89.7 so; the prompt step's write 1.8 us).
#include "hipserve/kv4.h"

namespace hipserve {

// Rows times kv heads from which runs of a page are taken together, 13 a compute unit: below, a token a workgroup is a shorter chain of loads.
// Token / runs, us: 32 / 8 heads 64 rows 3.5 / 4.8, 384 rows 5.0 / 5.2, 512 rows 6.1 / 5.4, 8192 rows 40 / 37; 32 / 32 heads 64 rows 4.2 / 4.4,
// 128 rows 5.6 / 4.6, 8192 rows 119 / 69; 8 / 2 heads 1024 rows 4.2 / 5.1, 2048 rows 5.7 / 5.3.
constexpr long kKv4RowsFrom = 13 * 256;

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

// rotate-half: 8 + 8 values of the two halves of a head by the cosines and sines co, si
HS_DEVICE void kv4_rotate16(const float (&x)[8], const float (&y)[8], const float (&co)[8], const float (&si)[8], u16x8& a,
                            u16x8& b) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float ra, rb;
    rope_rot(x[j], y[j], co[j], si[j], ra, rb);
    a[j] = f32_to_bf16(ra);
    b[j] = f32_to_bf16(rb);
  }
}
// neighbouring dims: 4 pairs
HS_DEVICE u16x8 kv4_rotate8(const float (&x)[8], const float* co, const float* si) {
  u16x8 v;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    float ra, rb;
    rope_rot(x[2 * p], x[2 * p + 1], co[p], si[p], ra, rb);
    v[2 * p] = f32_to_bf16(ra);
    v[2 * p + 1] = f32_to_bf16(rb);
  }
  return v;
}

// largest magnitude's bits of a group: over a quad of lanes with 8 of its dims each
HS_DEVICE unsigned kv4_quad_amax(const u16x8 v) {
  unsigned m = kv4_amax8(v);
  m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, false));  // quad_perm [1, 0, 3, 2]
  return max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, false));  // [2, 3, 0, 1]
}

// 8 dims c of a token's key (values: kV) to its slot, byte by byte where a byte is a token's
template <bool kV>
HS_DEVICE void kv4_put8(unsigned char* __restrict__ cache, long base, int off, int c, unsigned codes, int byte, int bs, int D) {
  unsigned char* p = cache + base;
  if (!kV) {
    *reinterpret_cast<unsigned*>(p + off * (D / 2) + c * 4) = codes;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) p[(c * 4 + j) * bs + off] = (unsigned char)(codes >> (8 * j));
  }
  if ((c & 3) == 0) p[kv4_code_bytes(bs, D) + (c >> 2) * bs + (kV ? off : kv4_key_scale_at(off))] = (unsigned char)byte;
}

// One token and kv head a workgroup. Every thread loads two runs of 8: of the halves of a query or the key, or a run of the value.
template <int kMode, bool kParts, int D>
__global__ __launch_bounds__(256) void kv4_write_token_kernel(unsigned short* __restrict__ qkv, long qkv_stride, Kv4In in,
                                                              const long* __restrict__ positions, long max_pos,
                                                              const long* __restrict__ slots,
                                                              const float* __restrict__ cos_sin,
                                                              unsigned char* __restrict__ k_cache,
                                                              unsigned char* __restrict__ v_cache, long nslots, int nq,
                                                              int nkv, int bs) {
  constexpr int half = D / 2, CH = kMode == 0 ? half / 8 : D / 8;
  __shared__ __attribute__((aligned(16))) unsigned short kv[2][D];
  const int t = blockIdx.x / nkv, kh = blockIdx.x % nkv;
  const int h0 = nq * kh / nkv, nh = nq * (kh + 1) / nkv - h0;  // this kv head's queries
  const long slot = slots[t];
  unsigned short* row = qkv + t * qkv_stride;
  const float* cs = cos_sin + min(max(positions[t], 0L), max_pos - 1) * D;
  const int qk = (nh + 1) * CH;
  for (int it = threadIdx.x; it < qk + D / 8; it += blockDim.x) {
    const bool is_v = it >= qk;
    const int hl = it / CH, c = is_v ? it - qk : it % CH;
    const bool is_k = hl == nh;
    const int col = is_v ? (nq + nkv + kh) * D : is_k ? (nq + kh) * D : (h0 + hl) * D;
    float x[8], y[8], co[8], si[8];
    const int i0 = is_v ? 0 : kMode == 0 ? c * 8 : c * 4;
#pragma unroll
    for (int j = 0; j < (kMode == 0 ? 8 : 4); ++j) {
      co[j] = cs[i0 + j];
      si[j] = cs[half + i0 + j];
    }
    kv4_in8<kParts>(x, in, row, t, col + c * 8);
    if (kMode == 0) kv4_in8<kParts>(y, in, row, t, is_v ? col + c * 8 : col + half + c * 8);
    u16x8 va, vb;
    if (is_v) {
#pragma unroll
      for (int j = 0; j < 8; ++j) va[j] = f32_to_bf16(x[j]);
      *reinterpret_cast<u16x8*>(&kv[1][c * 8]) = va;
      continue;
    }
    unsigned short* dst = is_k ? kv[0] : row + col;
    if constexpr (kMode == 0) {
      if (kParts && in.qw != nullptr) {  // a head's lanes are neighbours (CH is a power of two), as in splitk_rope_cache
        float ss = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
#pragma unroll
        for (int j = 0; j < 8; ++j) s2 += y[j] * y[j];
        ss += s2;
        for (int o = CH / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
        const float inv = rsqrtf(ss / D + in.eps);
        const float* nw = is_k ? in.kw : in.qw;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = bf16_to_f32(f32_to_bf16(x[j] * inv * nw[c * 8 + j]));
          y[j] = bf16_to_f32(f32_to_bf16(y[j] * inv * nw[half + c * 8 + j]));
        }
      }
      kv4_rotate16(x, y, co, si, va, vb);
      *reinterpret_cast<u16x8*>(dst + c * 8) = va;
      *reinterpret_cast<u16x8*>(dst + half + c * 8) = vb;
    } else {
      *reinterpret_cast<u16x8*>(dst + c * 8) = kv4_rotate8(x, co, si);
    }
  }
  __syncthreads();
  if (slot < 0 || slot >= nslots) return;
  const int it = threadIdx.x;  // D / 8 lanes for the key, as many for the value; a group is a quad
  if (it < 2 * (D / 8)) {
    const int which = it / (D / 8), c = it % (D / 8);
    const u16x8 v = *reinterpret_cast<const u16x8*>(&kv[which][c * 8]);
    const int byte = kv4_scale_byte(kv4_quad_amax(v));
    const unsigned codes = kv4_quantise8(v, byte);
    const int off = (int)(slot % bs);
    const long base = (slot / bs * nkv + kh) * (long)kv4_head_bytes(bs, D);
    if (which == 0) kv4_put8<false>(k_cache, base, off, c, codes, byte, bs, D);
    else kv4_put8<true>(v_cache, base, off, c, codes, byte, bs, D);
  }
}

// Rows in the order of a step, in runs: a run is rows of neighbouring slots within 16 slots of a page. The workgroup of rows t0 ..
// t0 + 15 takes the runs that begin there, rows first .. end - 1 (at most 31), so that the rows of a prompt are taken page by page
// wherever it begins in the step. Every wave works this out for itself.
struct Kv4Rows {
  int first, end;
  long slot;   // of the first row
  bool whole;  // one run of 16 rows: all of a page's 16 slots
};
HS_DEVICE Kv4Rows kv4_rows(const long* __restrict__ slots, long nslots, int t0, int T) {
  const int lane = threadIdx.x & 63, t = t0 + lane;
  const long s = t < T ? slots[t] : -1, before = t > 0 && t < T ? slots[t - 1] : -2;
  const bool begins = t >= T || t == 0 || s < 0 || (s & 15) == 0 || s != before + 1;
  const unsigned mask = (unsigned)__ballot(begins);
  Kv4Rows r{0, 0, -1, false};
  if ((mask & 0xffffu) == 0) return r;
  const int f = __builtin_ctz(mask), e = 16 + __builtin_ctz(mask >> 16);
  r.first = t0 + f;
  r.end = min(t0 + e, T);
  r.slot = __builtin_bit_cast(long, ((unsigned long)(unsigned)__builtin_amdgcn_readlane((int)(s >> 32), f) << 32) |
                                        (unsigned)__builtin_amdgcn_readlane((int)s, f));
  r.whole = r.end - r.first == 16 && ((mask >> f) & 0xffffu) == 1u && r.slot >= 0 && (r.slot & 15) == 0 && r.slot <= nslots - 16;
  return r;
}

// A prompt step: 16 lanes a token; the chunk's cosines and sines stay in registers over the heads.
template <int kMode, int D>
__global__ __launch_bounds__(256) void kv4_write_rows_kernel(unsigned short* __restrict__ qkv, long qkv_stride,
                                                             const long* __restrict__ positions, long max_pos,
                                                             const long* __restrict__ slots,
                                                             const float* __restrict__ cos_sin,
                                                             unsigned char* __restrict__ k_cache,
                                                             unsigned char* __restrict__ v_cache, long nslots, int T, int nq,
                                                             int nkv, int bs) {
  constexpr int half = D / 2, CH = kMode == 0 ? half / 8 : D / 8, HP = 16 / CH;  // lanes a head; heads at a time
  constexpr int NG = D / 32, C8 = D / 8;
  constexpr int PAD = 8;  // a token's row of LDS: 16 lanes of different tokens on different banks
  __shared__ __attribute__((aligned(16))) unsigned short ks[16][D + PAD];
  __shared__ __attribute__((aligned(16))) unsigned char vcode[D / 2][16];
  __shared__ __attribute__((aligned(16))) unsigned char scale[2][NG][16];
  const Kv4Rows rows = kv4_rows(slots, nslots, blockIdx.x / nkv * 16, T);
  const int kh = blockIdx.x % nkv;
  const int h0 = nq * kh / nkv, nh = nq * (kh + 1) / nkv - h0;  // this kv head's queries, then its key
  const int tt = threadIdx.x >> 4, l = threadIdx.x & 15, c = l % CH;
  const long head_bytes = kv4_head_bytes(bs, D);
  const int code_bytes = kv4_code_bytes(bs, D);
  for (int r0 = rows.first; r0 < rows.end; r0 += 16) {
    const int t = r0 + tt;
    const bool live = t < rows.end;
    unsigned short* row = qkv + (long)min(t, T - 1) * qkv_stride;
    u16x8 v8{0, 0, 0, 0, 0, 0, 0, 0};
    if (live && l < C8) v8 = *reinterpret_cast<const u16x8*>(row + (nq + nkv + kh) * D + l * 8);
    if (live && l < HP * CH) {
      const float* cs = cos_sin + min(max(positions[t], 0L), max_pos - 1) * D;
      constexpr int NC = kMode == 0 ? 8 : 4;
      float co[8], si[8];
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        co[j] = cs[c * NC + j];
        si[j] = cs[half + c * NC + j];
      }
      // heads l / CH, + HP, ...: three at a time, their loads first
      for (int g0 = l / CH; g0 <= nh; g0 += 3 * HP) {
        u16x8 a[3], b[3];
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          const int hl = min(g0 + q * HP, nh), col = hl == nh ? (nq + kh) * D : (h0 + hl) * D;
          a[q] = *reinterpret_cast<const u16x8*>(row + col + c * 8);
          if (kMode == 0) b[q] = *reinterpret_cast<const u16x8*>(row + col + half + c * 8);
        }
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          const int hl = g0 + q * HP;
          if (hl > nh) continue;
          unsigned short* dst = hl == nh ? ks[tt] : row + (h0 + hl) * D;
          float x[8], y[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = bf16_to_f32(a[q][j]);
          if constexpr (kMode == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = bf16_to_f32(b[q][j]);
            u16x8 va, vb;
            kv4_rotate16(x, y, co, si, va, vb);
            *reinterpret_cast<u16x8*>(dst + c * 8) = va;
            *reinterpret_cast<u16x8*>(dst + half + c * 8) = vb;
          } else {
            *reinterpret_cast<u16x8*>(dst + c * 8) = kv4_rotate8(x, co, si);
          }
        }
      }
    }
    __syncthreads();
    const long slot = rows.whole ? rows.slot + tt : live ? slots[t] : -1;
    const bool keep = slot >= 0 && slot < nslots;
    const int off = keep ? (int)(slot % bs) : 0;
    const long base = keep ? (slot / bs * nkv + kh) * head_bytes : 0;
    if (l < C8) {  // a group is a quad of lanes
      const u16x8 k8 = *reinterpret_cast<const u16x8*>(&ks[tt][l * 8]);
      const int kb = kv4_scale_byte(kv4_quad_amax(k8)), vb = kv4_scale_byte(kv4_quad_amax(v8));
      const unsigned kc = kv4_quantise8(k8, kb), vc = kv4_quantise8(v8, vb);
      if (rows.whole) {
        *reinterpret_cast<unsigned*>(k_cache + base + off * (D / 2) + l * 4) = kc;
#pragma unroll
        for (int j = 0; j < 4; ++j) vcode[l * 4 + j][tt] = (unsigned char)(vc >> (8 * j));
        if ((l & 3) == 0) {
          scale[0][l >> 2][kv4_key_scale_at(tt)] = (unsigned char)kb;
          scale[1][l >> 2][tt] = (unsigned char)vb;
        }
      } else if (keep) {
        kv4_put8<false>(k_cache, base, off, l, kc, kb, bs, D);
        kv4_put8<true>(v_cache, base, off, l, vc, vb, bs, D);
      }
    }
    __syncthreads();
    if (rows.whole) {  // 16 tokens of a pair of dims, or 16 tokens' scales, a thread
      const int o = (int)(rows.slot % bs), i = threadIdx.x;
      const long at = (rows.slot / bs * nkv + kh) * head_bytes;
      if (i < D / 2) *reinterpret_cast<u32x4*>(v_cache + at + i * bs + o) = *reinterpret_cast<const u32x4*>(vcode[i]);
      else if (i < D / 2 + NG)
        *reinterpret_cast<u32x4*>(v_cache + at + code_bytes + (i - D / 2) * bs + o) = *reinterpret_cast<const u32x4*>(scale[1][i - D / 2]);
      else if (i < D / 2 + 2 * NG)
        *reinterpret_cast<u32x4*>(k_cache + at + code_bytes + (i - D / 2 - NG) * bs + o) =
            *reinterpret_cast<const u32x4*>(scale[0][i - D / 2 - NG]);
    }
  }
}

template <int D>
static void kv4_write(unsigned short* q, long qkv_stride, const Kv4In& in, const long* positions, long max_pos, const long* slots,
                      const float* cos_sin, const Kv4Cache& c, int T, int nq, int mode, hipStream_t s) {
  auto* kc = static_cast<unsigned char*>(c.k);
  auto* vc = static_cast<unsigned char*>(c.v);
  const long nslots = c.blocks * c.block_size;
  if (in.ws == nullptr && (long)T * c.nkv >= kKv4RowsFrom) {
#define HS_KV4_WRITE(mode_)                                                                                              \
  kv4_write_rows_kernel<mode_, D><<<cdiv(T, 16) * c.nkv, 256, 0, s>>>(q, qkv_stride, positions, max_pos, slots, cos_sin, kc, \
                                                                           vc, nslots, T, nq, c.nkv, c.block_size)
    if (mode == 0) HS_KV4_WRITE(0);
    else HS_KV4_WRITE(1);
#undef HS_KV4_WRITE
    return;
  }
  // a pass of 8 values a thread, whole waves
  const int items = (cdiv(nq, c.nkv) + 1) * (mode == 0 ? D / 16 : D / 8) + D / 8;
  const int threads = min(256, cdiv(items, 64) * 64);
#define HS_KV4_WRITE(mode_, parts)                                                                                        \
  kv4_write_token_kernel<mode_, parts, D><<<T * c.nkv, threads, 0, s>>>(q, qkv_stride, in, positions, max_pos, slots, cos_sin, \
                                                                             kc, vc, nslots, nq, c.nkv, c.block_size)
  if (in.ws != nullptr) {
    if (mode == 0) HS_KV4_WRITE(0, true);
    else HS_KV4_WRITE(1, true);
  } else {
    if (mode == 0) HS_KV4_WRITE(0, false);
    else HS_KV4_WRITE(1, false);
  }
#undef HS_KV4_WRITE
}

void launch_kv4_write(void* qkv, long qkv_stride, const float* ws, int S, const void* bias, const float* qw,
                      const float* kw, float eps, const long* positions, const long* slots, const float* cos_sin,
                      long max_pos, const Kv4Cache& c, int T, int nq, int mode, hipStream_t s) {
  if (T <= 0) return;
  const int N = (nq + 2 * c.nkv) * c.D;
  const Kv4In in{ws, (long)T * N, S, N, static_cast<const unsigned short*>(bias), qw, kw, eps};
  auto* q = static_cast<unsigned short*>(qkv);
  if (c.D == 128) kv4_write<128>(q, qkv_stride, in, positions, max_pos, slots, cos_sin, c, T, nq, mode, s);
  else if (c.D == 96) kv4_write<96>(q, qkv_stride, in, positions, max_pos, slots, cos_sin, c, T, nq, mode, s);
  else kv4_write<64>(q, qkv_stride, in, positions, max_pos, slots, cos_sin, c, T, nq, mode, s);
}

// 8 codes under a scale byte, as bf16
HS_DEVICE u32x4 kv4_widen8(unsigned w, int byte) {
  if (byte == kKv4Nan) return u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
  const float s = kv4_scale(byte);
  return u32x4{kv4_widen2<0>(w, s), kv4_widen2<1>(w, s), kv4_widen2<2>(w, s), kv4_widen2<3>(w, s)};
}

// Rows of slots as bf16: runs of 16 as the writer takes them, 16 lanes a token, 8 dims a lane, of kHeads heads. Bound by the bytes of
// the rows where enough loads are under way: four heads a workgroup ask for theirs together. A whole run's value codes come as 16 tokens
// of a pair of dims and turn in LDS.
template <int D, int kHeads>
__global__ __launch_bounds__(256) void kv4_read_kernel(unsigned short* __restrict__ k_out, long k_stride,
                                                       unsigned short* __restrict__ v_out, long v_stride,
                                                       const unsigned char* __restrict__ k_cache,
                                                       const unsigned char* __restrict__ v_cache,
                                                       const long* __restrict__ slots, long nslots, int T, int nkv, int bs) {
  constexpr int C8 = D / 8, ROW = D / 2 + 4;
  __shared__ __attribute__((aligned(16))) unsigned char vcode[kHeads][16][ROW];
  const int parts = cdiv(nkv, kHeads);
  const Kv4Rows rows = kv4_rows(slots, nslots, blockIdx.x / parts * 16, T);
  const int kh0 = blockIdx.x % parts * kHeads, heads = min(kHeads, nkv - kh0);
  const int tt = threadIdx.x >> 4, l = threadIdx.x & 15;
  const long head_bytes = kv4_head_bytes(bs, D);
  const int code_bytes = kv4_code_bytes(bs, D);
  for (int r0 = rows.first; r0 < rows.end; r0 += 16) {
    const int t = r0 + tt;
    const long slot = rows.whole ? rows.slot + tt : t < rows.end ? slots[t] : -1;
    const bool keep = slot >= 0 && slot < nslots;
    const int off = keep ? (int)(slot % bs) : 0;
    const long base = keep ? (slot / bs * nkv + kh0) * head_bytes : 0;
    if (rows.whole) {
      const int u = threadIdx.x / (D / 2), i = threadIdx.x % (D / 2);
      if (u < heads) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(v_cache + (rows.slot / bs * nkv + kh0 + u) * head_bytes + i * bs + rows.slot % bs);
#pragma unroll
        for (int j = 0; j < 16; ++j) vcode[u][j][i] = (unsigned char)(w[j >> 2] >> (8 * (j & 3)));
      }
    }
    const bool mine = t < rows.end && l < C8;
    unsigned kc[kHeads], vc[kHeads];
    int kb[kHeads], vb[kHeads];
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      kc[u] = vc[u] = 0;
      kb[u] = vb[u] = 127;  // a slot outside of the cache: zeros
      if (!mine || !keep || u >= heads) continue;
      const unsigned char *kp = k_cache + base + u * head_bytes, *vp = v_cache + base + u * head_bytes;
      kc[u] = *reinterpret_cast<const unsigned*>(kp + off * (D / 2) + l * 4);
      kb[u] = kp[code_bytes + (l >> 2) * bs + kv4_key_scale_at(off)];
      vb[u] = vp[code_bytes + (l >> 2) * bs + off];
      if (!rows.whole)
#pragma unroll
        for (int j = 0; j < 4; ++j) vc[u] |= (unsigned)vp[(l * 4 + j) * bs + off] << (8 * j);
    }
    if (rows.whole) __syncthreads();
    if (!mine) continue;
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      if (u >= heads) break;
      if (rows.whole) vc[u] = *reinterpret_cast<const unsigned*>(&vcode[u][tt][l * 4]);
      const long at = (long)(kh0 + u) * D + l * 8;
      __builtin_nontemporal_store(kv4_widen8(kc[u], kb[u]), reinterpret_cast<u32x4*>(k_out + t * k_stride + at));
      __builtin_nontemporal_store(kv4_widen8(vc[u], vb[u]), reinterpret_cast<u32x4*>(v_out + t * v_stride + at));
    }
  }
}

void launch_kv4_read(void* k_out, long k_stride, void* v_out, long v_stride, const Kv4Cache& c, const long* slots, int T,
                     hipStream_t s) {
  if (T <= 0) return;
#define HS_KV4_READ(d, heads)                                                                                             \
  kv4_read_kernel<d, heads><<<cdiv(T, 16) * cdiv(c.nkv, heads), 256, 0, s>>>(                                            \
      static_cast<unsigned short*>(k_out), k_stride, static_cast<unsigned short*>(v_out), v_stride,                       \
      static_cast<const unsigned char*>(c.k), static_cast<const unsigned char*>(c.v), slots, c.blocks * c.block_size, T,   \
      c.nkv, c.block_size)
  if (c.D == 128) HS_KV4_READ(128, 4);
  else if (c.D == 96) HS_KV4_READ(96, 4);
  else HS_KV4_READ(64, 4);
#undef HS_KV4_READ
}

}  // namespace hipserve
