// Causal attention of prompt portions over the 4-bit paged KV cache (layout and format: kv4.h), with a sliding window and first tokens
// that stay visible beside it. Keys of the step itself come from the cache like the older ones: kv4_write has run before.
//
// Bound by the matrix cores and by what stands beside their products, so a tile is unpacked once for all its readers:
//  * workgroup = up to 8 query heads of one kv head x blocks of 32 rows, a wave each; 64 keys a tile, two LDS buffers, one barrier
//    a tile, the loads of the next two tiles in registers.
//  * S^T = K . Q^T on v_mfma_scale_f32_32x32x64_f8f6f4: K's codes lie in LDS as they are (a quarter of bf16's LDS reads), their
//    scale bytes are the product's; q as two e4m3 numbers (see kv4_decode.hip), exact for a bf16 q, at bf16's rate.
//  * V is widened to bf16 on its way into LDS, transposed as it lies in the cache: a thread takes 8 tokens of two dims, v_cvt applies the
//    scales, v_perm sorts the dims.
//  * keys sit in K's LDS rows with bits 2 and 3 exchanged: a lane's scores are then 8 neighbouring keys a step of the second product,
//    O^T = V^T . P^T, and P is its operand without an exchange.
//  * softmax in base 2, 32 bits; P is rounded to bf16, its sum is not; O is rescaled when a score is over 2^8 above the maximum.
// Hidden keys have score -inf whatever they hold. A value's NaN (scale byte 255) must reach the rows that see it alone, and 0 * NaN is
// not 0: it is staged as a finite number and put into the accumulators of the rows that see it, in a branch that no other tile takes.
#include "hipserve/kv4.h"

namespace hipserve {

constexpr int kKv4Tile = 64;

HS_DEVICE float kv4_max32(float v) {  // over lanes l and l ^ 32
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
HS_DEVICE float kv4_sum32(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}

// whether a byte of w is 255
HS_DEVICE bool kv4_any_nan(unsigned w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & w & 0x80808080u) != 0; }
HS_DEVICE unsigned kv4_no_nan(unsigned w) {  // 255 -> 127
  return w ^ ((((w & 0x7f7f7f7fu) + 0x01010101u) & w & 0x80808080u));
}

template <int D, int HG, int NWV>
__global__ __launch_bounds__(64 * NWV) __attribute__((amdgpu_waves_per_eu(2, 8))) void kv4_prefill_kernel(Kv4Attn a, const int* __restrict__ cu_q, int seqs,
                                                               const int* __restrict__ ctx_lens, int rows,
                                                               const int* __restrict__ tiles) {
  constexpr int NG = D / 32, KS = (D + 63) / 64;   // scale groups; steps of the first product
  constexpr int RB = NWV / HG, QR = 32 * RB, SUB = 128 / QR;
  constexpr int NT = 64 * NWV;
  constexpr int KLD = D == 64 ? 48 : 80;           // bytes of K's LDS rows, an odd multiple of 16: 16 lanes' reads on 16 bank groups
  constexpr int VLD = kKv4Tile + 8;
  constexpr int NKI = kKv4Tile * D / 16, NVI = kKv4Tile / 8 * (D / 2);  // 8-byte pieces of K; 8 tokens x 2 dims of V
  constexpr int NKP = (NKI + NT - 1) / NT, NVP = (NVI + NT - 1) / NT;
  __shared__ __attribute__((aligned(16))) unsigned char kl[2][kKv4Tile * KLD];
  __shared__ __attribute__((aligned(16))) unsigned short vl[2][D * VLD];
  __shared__ unsigned ksc[2][kKv4Tile];                                      // a key's scale bytes, in LDS row order
  __shared__ __attribute__((aligned(8))) unsigned char vsc[2][NG][kKv4Tile];  // values' scale bytes
  __shared__ __attribute__((aligned(4))) unsigned char nopage[2][4];                                     // runs of 16 tokens without a page
  __shared__ int nans;                                                       // a value's scale byte of 255 has come by

  // dispatch order: kv-head groups fastest, then the host's tiles, the later rows of a tile first
  const int L = blockIdx.x + gridDim.x * blockIdx.y, gy = gridDim.y;
  const int gyi = L % gy, rest = L / gy;
  const int t = rest / SUB, sub = SUB - 1 - (rest - t * SUB);
  const int seq = tiles[2 * t], r0 = tiles[2 * t + 1] + sub * QR;
  if (seq < 0 || seq >= seqs) return;
  const int q0 = cu_q[seq], qlen = cu_q[seq + 1] - q0;
  if (r0 < 0 || r0 >= qlen || q0 < 0 || q0 + qlen > rows) return;  // the whole workgroup, before any barrier
  const int nkv = a.cache.nkv, bs = a.cache.block_size, G = a.nq / nkv;
  const int ctx = ctx_lens[seq], cap = a.bt_width * bs;
  const int kh = gyi / (G / HG);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = gyi * HG + wave % HG;
  const int qi = lane & 31, half = lane >> 5;
  const int wrow0 = r0 + wave / HG * 32;
  const bool wactive = wrow0 < qlen;
  const int row = min(wrow0 + qi, qlen - 1);
  const int pos = ctx - qlen + row;                                    // this lane's row
  const int wmin = ctx - qlen + wrow0, wmax = ctx - qlen + min(wrow0 + 31, qlen - 1);  // the wave's
  const int window = a.window, sinks = a.sinks;
  // tiles of the workgroup: those of the first `sinks` keys, then from its first row's window on
  const int last = min(ctx - qlen + min(r0 + QR - 1, qlen - 1), cap - 1);  // the last key that some row sees
  const int lo = window > 0 ? max(0, ctx - qlen + r0 - window + 1) : 0;
  const int first = lo / kKv4Tile, nst = min((min(sinks, lo) + kKv4Tile - 1) / kKv4Tile, first);
  const int nkt = last < 0 ? 0 : max(0, nst + last / kKv4Tile + 1 - first);
  auto tile_key = [&](int v) { return (v < nst ? v : v - nst + first) * kKv4Tile; };
  const int* bt = a.block_tables + (long)seq * a.bt_stride;
  const int bsh = __builtin_ctz(bs), bmask = bs - 1;

  // ---- staging. Pages are asked for a tile before the loads that need them.
  const long head_bytes = kv4_head_bytes(bs, D), page_bytes = head_bytes * nkv;
  const int code_bytes = kv4_code_bytes(bs, D);
  const unsigned char* kbase = static_cast<const unsigned char*>(a.cache.k) + kh * head_bytes;
  const unsigned char* vbase = static_cast<const unsigned char*>(a.cache.v) + kh * head_bytes;
  struct Pages {
    int k[NKP], v[NVP], s;
  };
  struct Stage {
    u32x2 k[NKP], v[NVP], vs[NVP];
    unsigned ks;
    int vpage[NVP];
  };
  auto pages = [&](int v, Pages& pg) {
    const int key = tile_key(min(v, nkt - 1));
#pragma unroll
    for (int i = 0; i < NKP; ++i) pg.k[i] = bt[min(key + (tid + NT * i) / (D / 16) % kKv4Tile, last) >> bsh];
#pragma unroll
    for (int i = 0; i < NVP; ++i) pg.v[i] = bt[min(key + 16 * ((tid + NT * i) / D % 4), last) >> bsh];
    pg.s = bt[min(key + lane, last) >> bsh];
  };
  auto load = [&](int v, const Pages& pg, Stage& st) {
    const int key = tile_key(min(v, nkt - 1));
#pragma unroll
    for (int i = 0; i < NKP; ++i) {
      const int it = tid + NT * i, kk = it / (D / 16) % kKv4Tile, piece = it % (D / 16);
      st.k[i] = *reinterpret_cast<const u32x2*>(kbase + (long)max(kv4_page(pg.k[i], a.cache.blocks), 0) * page_bytes +
                                                ((key + kk) & bmask) * (D / 2) + 8 * piece);
    }
#pragma unroll
    for (int i = 0; i < NVP; ++i) {
      const int it = tid + NT * i, run = it / D % 4, p = it % D >> 1, h8 = it & 1;
      const int page = kv4_page(pg.v[i], a.cache.blocks), off = ((key + 16 * run) & bmask) + 8 * h8;
      const unsigned char* vp = vbase + (long)max(page, 0) * page_bytes;
      st.v[i] = *reinterpret_cast<const u32x2*>(vp + p * bs + off);
      st.vs[i] = *reinterpret_cast<const u32x2*>(vp + code_bytes + (p >> 4) * bs + off);
      st.vpage[i] = page;
    }
    if (wave == 0) {  // a key's scale bytes, together
      const unsigned char* sp = kbase + (long)max(kv4_page(pg.s, a.cache.blocks), 0) * page_bytes + code_bytes +
                                kv4_key_scale_at((key + lane) & bmask);
      unsigned w = 0;
#pragma unroll
      for (int g = 0; g < 4; ++g) w |= (g < NG ? (unsigned)sp[g * bs] : 127u) << (8 * g);
      st.ks = w;
    }
  };
  auto store = [&](Stage& st, int buf) {
#pragma unroll
    for (int i = 0; i < NKP; ++i) {
      const int it = tid + NT * i, kk = it / (D / 16), piece = it % (D / 16);
      const int krow = (kk & ~12) | ((kk & 4) << 1) | ((kk & 8) >> 1);
      if (NKI % NT == 0 || it < NKI) *reinterpret_cast<u32x2*>(&kl[buf][krow * KLD + 8 * piece]) = st.k[i];
    }
    if (wave == 0) ksc[buf][(lane & ~12) | ((lane & 4) << 1) | ((lane & 8) >> 1)] = st.ks;
#pragma unroll
    for (int i = 0; i < NVP; ++i) {
      const int it = tid + NT * i, run = it / D, p = it % D >> 1, h8 = it & 1;
      if (NVI % NT != 0 && it >= NVI) continue;
      if ((p & 15) == 0) *reinterpret_cast<u32x2*>(&vsc[buf][p >> 4][16 * run + 8 * h8]) = st.vs[i];
      if ((it % D) == 0) nopage[buf][run] = st.vpage[i] < 0;
      if (kv4_any_nan(st.vs[i][0]) || kv4_any_nan(st.vs[i][1])) {
        nans = 1;
        st.vs[i][0] = kv4_no_nan(st.vs[i][0]);
        st.vs[i][1] = kv4_no_nan(st.vs[i][1]);
      }
      u32x4 even, odd;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const unsigned w = st.v[i][q], s = st.vs[i][q];
        const unsigned x0 = kv4_widen2<0>(w, __uint_as_float(s << 23)), x1 = kv4_widen2<1>(w, __uint_as_float(s << 15));
        const unsigned x2 = kv4_widen2<2>(w, __uint_as_float(s << 7)), x3 = kv4_widen2<3>(w, __uint_as_float(s >> 1));
        even[2 * q] = __builtin_amdgcn_perm(x1, x0, 0x05040100u);
        odd[2 * q] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
        even[2 * q + 1] = __builtin_amdgcn_perm(x3, x2, 0x05040100u);
        odd[2 * q + 1] = __builtin_amdgcn_perm(x3, x2, 0x07060302u);
      }
      unsigned short* dst = &vl[buf][2 * p * VLD + 16 * run + 8 * h8];
      *reinterpret_cast<u32x4*>(dst) = even;
      *reinterpret_cast<u32x4*>(dst + VLD) = odd;
    }
  };

  Pages pg;
  Stage sa, sb;
  if (nkt > 0) {
    pages(0, pg);
    Pages next;
    pages(1, next);
    load(0, pg, sa);
    pages(2, pg);
    load(1, next, sb);
  }

  // ---- q of this lane's row: dims 64 s + 16 half .. and 64 s + 32 + 16 half .. of step s
  i32x8 qhi[KS], qlo[KS];
  float sl;
  {
    const unsigned short* qp = static_cast<const unsigned short*>(a.q) + (long)(q0 + row) * a.q_stride + (long)h * D + 16 * half;
    u16x8 raw[KS][4];
    unsigned am = 0;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d0 = 64 * s + 32 * (e >> 1) + 8 * (e & 1);
        raw[s][e] = d0 < D ? *reinterpret_cast<const u16x8*>(qp + d0) : u16x8{0, 0, 0, 0, 0, 0, 0, 0};
        am = max(am, kv4_amax8(raw[s][e]));
      }
    am = max(am, (unsigned)__shfl_xor((int)am, 32, 64));
    const int eb = min(max((int)(am >> 7), 16), 254);  // the largest value comes to [128, 256)
    const float down = __uint_as_float((unsigned)(eb - 7) << 23), down16 = __uint_as_float((unsigned)(eb - 11) << 23);
    // never 0: a hidden key's -inf has to stay one
    sl = am >= 0x7f80u ? NAN : fmaxf(a.scale * kLog2E * down, 1.17549435e-38f);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u32x2 hi, lo2;
        kv4_split8(raw[s][e], down, down16, hi, lo2);
        qhi[s][2 * e] = (int)hi[0];
        qhi[s][2 * e + 1] = (int)hi[1];
        qlo[s][2 * e] = (int)lo2[0];
        qlo[s][2 * e + 1] = (int)lo2[1];
      }
  }

  f32x16 o[NG];
#pragma unroll
  for (int nb = 0; nb < NG; ++nb)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[nb][r] = 0.f;
  float m_run = -1e30f, l_run = 0.f;

  auto compute = [&](int v, int buf) __attribute__((always_inline)) {
    const int key = tile_key(v);
    if (!wactive || key > wmax || (window > 0 && key + kKv4Tile - 1 <= wmin - window && key >= sinks)) return;
    const unsigned gone = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const unsigned*>(nopage[buf]));
    const int bad = __builtin_amdgcn_readfirstlane(nans);
    // ---- scores: rows (keys) of the tile's halves, columns (queries) qi
    f32x16 st[2];
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
      for (int r = 0; r < 16; ++r) st[h2][r] = 0.f;
    unsigned ks[2];
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2) ks[h2] = ksc[buf][32 * h2 + qi] >> (8 * half);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      u32x4 kf[2];
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2)
        kf[h2] = *reinterpret_cast<const u32x4*>(&kl[buf][(32 * h2 + qi) * KLD + 16 * min(2 * s + half, NG - 1)]);
#pragma unroll
      for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {
          const i32x8 ka{(int)kf[h2][0], (int)kf[h2][1], (int)kf[h2][2], (int)kf[h2][3], 0, 0, 0, 0};
          const i32x8 qb = part == 0 ? qlo[s] : qhi[s];
          const int qs = part == 0 ? 123 : 127;
          if (s == 0) st[h2] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(ka, qb, st[h2], 4, 0, 0, (int)ks[h2], 0, qs);
          else st[h2] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(ka, qb, st[h2], 4, 0, 2, (int)ks[h2], 0, qs);
        }
    }
    // ---- hidden keys, in tiles that some row of the wave does not see whole; slot (h2, r): key 32 h2 + 16 (r >> 3) + 8 half + (r & 7)
    const bool whole = key + kKv4Tile - 1 <= min(wmin, cap - 1) &&
                       (window <= 0 || key > wmax - window || key + kKv4Tile <= sinks) && gone == 0;
    if (!whole) {
      const int lim = min(pos, cap - 1) - key - 8 * half;  // offsets above: behind the row
      if (window <= 0) {
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
          for (int r = 0; r < 16; ++r) st[h2][r] = 32 * h2 + 16 * (r >> 3) + (r & 7) > lim ? -INFINITY : st[h2][r];
      } else {
        const int wlo = pos - window - key - 8 * half;  // offsets up to this one: before the window,
        const int slo = sinks - key - 8 * half;         // and hidden unless below this one
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int off = 32 * h2 + 16 * (r >> 3) + (r & 7);
            const bool hidden = (off > lim) | ((off <= wlo) & (off >= slo));
            st[h2][r] = hidden ? -INFINITY : st[h2][r];
          }
      }
      if (gone)
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (gone >> (8 * (2 * h2 + (r >> 3))) & 255u) st[h2][r] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[h2][r]);
    mx *= sl;
    if (__any(mx > m_run + 8.f)) {
      const float m_new = fmaxf(m_run, kv4_max32(mx));
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int nb = 0; nb < NG; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[nb][r] *= alpha;
    }
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2) {
      bf16x8 pb[2];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(st[h2][r], sl, -m_run));
        ps[r & 3] += p;
        pb[r >> 3][r & 7] = static_cast<__bf16>(p);
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const unsigned short* vb = &vl[buf][qi * VLD + 32 * h2 + 16 * s2 + 8 * half];
#pragma unroll
        for (int nb = 0; nb < NG; ++nb) {
          const u16x8 va = *reinterpret_cast<const u16x8*>(vb + 32 * nb * VLD);
          o[nb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, va), pb[s2], o[nb], 0, 0, 0);
        }
      }
    }
    l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
    if (bad) {  // values of NaN among this tile's: into the rows that see them
      unsigned long seen = 0;
      for (int j = 0; j < kKv4Tile; ++j)
        if (key + j < cap && !(gone >> (8 * (j >> 4)) & 255u) && kv4_sees(key + j, pos, window, sinks)) seen |= 1ul << j;
#pragma unroll
      for (int nb = 0; nb < NG; ++nb) {
        const unsigned long lost = __ballot(vsc[buf][nb][lane] == kKv4Nan);
        if (seen & lost)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[nb][r] = NAN;
      }
    }
  };

  if (tid == 0) nans = 0;
  __syncthreads();
  if (nkt > 0) store(sa, 0);
  __syncthreads();
  for (int v = 0; v < nkt; v += 2) {
    // tile v in buffer 0; sb holds tile v + 1; pg the pages of tile v + 2
    Pages next;
    pages(v + 3, next);
    load(v + 2, pg, sa);
    compute(v, 0);
    if (v + 1 < nkt) store(sb, 1);
    __syncthreads();
    if (v + 1 >= nkt) break;
    pages(v + 4, pg);
    load(v + 3, next, sb);
    compute(v + 1, 1);
    if (v + 2 < nkt) store(sa, 0);
    __syncthreads();
  }
  if (!wactive || wrow0 + qi >= qlen) return;
  l_run = kv4_sum32(l_run);
  const float inv = l_run == 0.f ? 0.f : 1.f / l_run;  // a row that sees nothing: zeros
  unsigned short* op = static_cast<unsigned short*>(a.out) + (long)(q0 + row) * a.out_stride + (long)h * D;
#pragma unroll
  for (int nb = 0; nb < NG; ++nb)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      u16x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = f32_to_bf16(o[nb][4 * g + j] * inv);
      *reinterpret_cast<u16x4*>(op + 32 * nb + 8 * g + 4 * half) = w;
    }
}

template <int D, int HG, int NWV>
static void kv4_prefill(const Kv4Attn& a, const int* cu_q, int seqs, const int* ctx, int rows, const int* tiles, int ntiles,
                        hipStream_t s) {
  constexpr int SUB = 128 / (32 * (NWV / HG));
  kv4_prefill_kernel<D, HG, NWV><<<dim3(ntiles * SUB, a.nq / HG), 64 * NWV, 0, s>>>(a, cu_q, seqs, ctx, rows, tiles);
}

// as many query heads a workgroup as divide a kv head's, up to 8 waves
template <int D>
static void kv4_prefill_d(const Kv4Attn& a, const int* cu_q, int seqs, const int* ctx, int rows, const int* tiles, int ntiles,
                          hipStream_t s) {
  const int G = a.nq / a.cache.nkv;
  if (G % 8 == 0) kv4_prefill<D, 8, 8>(a, cu_q, seqs, ctx, rows, tiles, ntiles, s);
  else if (G % 4 == 0) kv4_prefill<D, 4, 8>(a, cu_q, seqs, ctx, rows, tiles, ntiles, s);
  else if (G % 2 == 0) kv4_prefill<D, 2, 8>(a, cu_q, seqs, ctx, rows, tiles, ntiles, s);
  else kv4_prefill<D, 1, 4>(a, cu_q, seqs, ctx, rows, tiles, ntiles, s);
}

void launch_kv4_prefill(const Kv4Attn& a, const int* cu_q, int seqs, const int* ctx_lens, int rows, const int* tiles,
                        int ntiles, hipStream_t s) {
  if (ntiles <= 0) return;
  if (a.cache.D == 128) kv4_prefill_d<128>(a, cu_q, seqs, ctx_lens, rows, tiles, ntiles, s);
  else if (a.cache.D == 96) kv4_prefill_d<96>(a, cu_q, seqs, ctx_lens, rows, tiles, ntiles, s);
  else kv4_prefill_d<64>(a, cu_q, seqs, ctx_lens, rows, tiles, ntiles, s);
}

}  // namespace hipserve
