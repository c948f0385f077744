// Causal attention of prompt portions over the 4-bit paged KV cache (layout and format: kv4.h), with a sliding window and first tokens
// that stay visible beside it. Keys of the step itself come from the cache like the older ones: kv4_write has run before.
//
// Bound by the matrix cores and by what stands beside their products, so a tile is unpacked once for all its readers:
//  * workgroup = up to 8 query heads of one kv head x blocks of 32 rows, a wave each; 64 keys a tile, staged through registers into
//    the tiles of LDS after the ones in use.
//    - 8 waves (two queries per kv head or more): two tiles a barrier, and half of the waves stage the next two before their products,
//      the others after them: of a SIMD's two waves one unpacks while the other multiplies.
//    - 4 waves (one query per kv head): the values of a tile and the scores of the next one together, one tile a barrier, two
//      workgroups a compute unit, as four tiles of LDS would leave room for one.
//    Each at the other's shape is slower: 8 waves by the second 887 against 840 us (4096 rows at 16384, 32 / 8 heads), 4 waves by
//    the first 124 against 111 us (8 x 1024 rows, 32 / 32 heads).
//  * S^T = K . Q^T on v_mfma_scale_f32_32x32x64_f8f6f4: K's codes lie in LDS as they are (a quarter of bf16's LDS reads), their
//    scale bytes are the product's; q as two e4m3 numbers (see kv4_decode.hip), the bits of a bf16 q, at bf16's rate.
//  * V is widened to bf16 on its way into LDS, transposed as it lies in the cache: a thread takes 8 tokens of two dims, v_cvt applies the
//    scales, v_perm sorts the dims.
//  * keys sit in K's LDS rows with bits 2 and 3 exchanged: a lane's scores are then 8 neighbouring keys a step of the second product,
//    O^T = V^T . P^T, and P is its operand without an exchange.
//  * softmax in base 2, 32 bits; P is rounded to bf16, as its product takes it, and its 32-bit sum is that of the rounded P: both come
//    from one dot product instruction, and what the rounding does to the weights it does to their sum. O is rescaled when a
//    score is over 2^8 above the maximum.
//  * rows leave through LDS, a row's dims together: 16-byte stores of 256 neighbouring bytes.
// Hidden keys have score -inf whatever they hold. A value's NaN (scale byte 255) must reach the rows that see it alone, and 0 * NaN is
// not 0: it is staged as a finite number and put into the accumulators of the rows that see it, in a branch that no other tile takes.
//
// 32 / 8 heads of 128 dims: 8192 rows 542 - 589 us (0.93 - 1.01 PFLOP/s), 4096 rows at 16384 846 us (1.14), a window of 4096 there 266 us; the 8-bit
// part of the products is twice the bf16 part's operations, so this is what a bf16 cache's kernel does (530 - 584, 878, 274 us) at 17 / 64 of its bytes.
#include <atomic>

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

HS_DEVICE i32x8 kv4_pad(const u32x4 a) { return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0}; }

// whether a byte of w is 255
HS_DEVICE bool kv4_any_nan(unsigned w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & w & 0x80808080u) != 0; }
HS_DEVICE unsigned kv4_no_nan(unsigned w) {  // 255 -> 127
  return w ^ ((((w & 0x7f7f7f7fu) + 0x01010101u) & w & 0x80808080u));
}

// A tile in LDS. K's rows are an odd multiple of 16 bytes, V^T's of 16 bytes too: 16 lanes' 16-byte reads on 16 bank groups.
template <int D>
struct Kv4Tile {
  static constexpr int KLD = D == 64 ? 48 : 80, VLD = kKv4Tile + 8;
  __attribute__((aligned(16))) unsigned short v[D * VLD];
  __attribute__((aligned(16))) unsigned char k[kKv4Tile * KLD];
  __attribute__((aligned(16))) unsigned char ks[D / 32][kKv4Tile];  // scale bytes, keys in the cache's order of them
  __attribute__((aligned(16))) unsigned char vs[D / 32][kKv4Tile];
  unsigned char nopage[4];                                          // runs of 16 tokens without a page
};

// A workgroup's rows and the tiles they see: those of the first `sinks` keys, then those from its first row's window on.
struct Kv4Block {
  int seq, r0, q0, qlen, ctx;  // sequence, first row in it, its first row of all, its rows and length
  int last, first, nst, nkt;    // last key that some row sees, first tile of the window, tiles of the first keys, tiles in all
};
template <int QR>
HS_DEVICE bool kv4_block(Kv4Block& b, const Kv4Attn& a, const int* __restrict__ cu_q, int seqs, const int* __restrict__ ctx_lens,
                         int rows, const int* __restrict__ tiles, int t, int sub) {
  b.seq = tiles[2 * t];
  b.r0 = tiles[2 * t + 1] + sub * QR;
  if (b.seq < 0 || b.seq >= seqs) return false;
  b.q0 = cu_q[b.seq];
  const int q1 = cu_q[b.seq + 1];
  if (b.q0 < 0 || q1 < b.q0 || q1 > rows) return false;  // before their difference, which others may have beyond 32 bits
  b.qlen = q1 - b.q0;
  if (b.r0 < 0 || b.r0 >= b.qlen) return false;
  b.ctx = max(ctx_lens[b.seq], 0);
  b.last = min(b.ctx - b.qlen + min(b.r0 + QR - 1, b.qlen - 1), a.bt_width * a.cache.block_size - 1);
  const int lo = a.window > 0 ? max(0, b.ctx - b.qlen + b.r0 - a.window + 1) : 0;
  const int end = b.last < 0 ? 0 : b.last / kKv4Tile + 1;  // tiles that the table has keys of: a length may go beyond it
  b.first = lo / kKv4Tile;
  b.nst = min((min(a.sinks, lo) + kKv4Tile - 1) / kKv4Tile, min(b.first, end));
  b.nkt = b.nst + max(0, end - b.first);
  return true;
}

// Few rows over a long context: their tiles are cut into up to `splits` runs, a workgroup each, and merged by a second kernel: 128 rows at
// 8192 keys 230 -> 49 us, one row 171 -> 27. A part costs what some 7 tiles do (its sums are 128 KB a workgroup, written and read), so runs of
// at least 8: with 4 a row of 8192 keys takes 38 us instead of 27, 500 rows of 500 keys 26 instead of 23, and only 64 rows of 1024 less, 23
// instead of 27.
constexpr int kKv4LeastRun = 8;
HS_HOST_DEVICE int kv4_tile_run(int nkt, int splits) { return max((nkt + splits - 1) / splits, kKv4LeastRun); }

// HG: query heads a workgroup; NWV: its waves; UN: tiles a barrier
template <int D, int HG, int NWV, int UN>
__global__ __launch_bounds__(64 * NWV) __attribute__((amdgpu_waves_per_eu(2, 8))) void kv4_prefill_kernel(
    Kv4Attn a, const int* __restrict__ cu_q, int seqs, const int* __restrict__ ctx_lens, int rows,
    const int* __restrict__ tiles, bool apart, float* __restrict__ work) {
  constexpr int NG = D / 32, KS = (D + 63) / 64;   // scale groups; steps of the first product
  constexpr int QR = 32 * NWV / HG, SUB = 128 / QR;
  constexpr int NT = 64 * NWV;
  constexpr int KLD = Kv4Tile<D>::KLD, VLD = Kv4Tile<D>::VLD;
  constexpr int NP = 512 / NT;  // runs of a tile that two waves take
  extern __shared__ __attribute__((aligned(16))) char smem[];
  Kv4Tile<D>* buf = reinterpret_cast<Kv4Tile<D>*>(smem);
  __shared__ int nans;  // a value's scale byte of 255 has come by

  // Dispatch order: kv-head groups fastest, then the host's tiles, the later rows of a tile first. Workgroups go round the chip's XCDs and
  // their shader engines in turn, so those of a tile that have no rows (short sequences) must not all come at the same place of that round:
  // from one tile to the next the order within a tile turns. Where they are many (`apart`), a tile's workgroups come a whole
  // round of tiles apart, those without rows together: 32 sequences of 20 rows at 4000 keys 182 -> 97 us; one sequence of 4096 rows,
  // 150 us, would take 158.
  const int heads = blockIdx.x, t = apart ? blockIdx.y : blockIdx.z;
  const int sub = (SUB - 1 - (apart ? blockIdx.z : blockIdx.y - blockIdx.z * SUB / 4)) & (SUB - 1);
  const int splits = apart ? gridDim.z / SUB : 1, split = apart ? blockIdx.z / SUB : 0;
  Kv4Block blk;
  if (!kv4_block<QR>(blk, a, cu_q, seqs, ctx_lens, rows, tiles, t, sub)) return;  // the whole workgroup, before any barrier
  const int r0 = blk.r0, q0 = blk.q0, qlen = blk.qlen, ctx = blk.ctx, last = blk.last, first = blk.first, nst = blk.nst;
  const int run = splits > 1 ? kv4_tile_run(blk.nkt, splits) : INT32_MAX / 2;
  const int v0 = splits > 1 ? run * split : 0, nkt = min(run, blk.nkt - v0);  // this workgroup's tiles, counted from the first of them
  if (v0 > 0 && nkt <= 0) return;
  const int nkv = a.cache.nkv, bs = a.cache.block_size, G = a.nq / nkv;
  const int cap = a.bt_width * bs;
  const int kh = heads / (G / HG);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = heads * HG + wave % HG;
  const int qi = lane & 31, half = lane >> 5;
  const int wrow0 = r0 + wave / HG * 32;
  const int row = min(wrow0 + qi, qlen - 1);
  const int pos = ctx - qlen + row;                                    // this lane's row
  const int wmin = ctx - qlen + wrow0, wmax = ctx - qlen + min(wrow0 + 31, qlen - 1);  // the wave's
  const int window = a.window, sinks = a.sinks;
  auto tile_key = [&](int i) {
    const int v = i + v0;
    return (v < nst ? v : v - nst + first) * kKv4Tile;
  };
  const int* bt = a.block_tables + (long)blk.seq * a.bt_stride;
  const int bsh = __builtin_ctz(bs), bmask = bs - 1;

  // ---- q of this lane's row, on its way first: dims 64 s + 16 half .. and 64 s + 32 + 16 half .. of step s
  u16x8 raw[KS][4];
  {
    const unsigned short* qp = static_cast<const unsigned short*>(a.q) + (long)(q0 + row) * a.q_stride + (long)h * D + 16 * half;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d0 = 64 * s + 32 * (e >> 1) + 8 * (e & 1);
        raw[s][e] = d0 < D ? *reinterpret_cast<const u16x8*>(qp + d0) : u16x8{0, 0, 0, 0, 0, 0, 0, 0};
      }
  }

  // ---- staging: two waves take a run of 16 tokens, a lane of the first D a key's 16 dims and 8 tokens of two dims. The run's page is
  // the same for a wave, so that addresses are scalars; it is asked for a step before the loads that need it.
  const long head_bytes = kv4_head_bytes(bs, D), page_bytes = head_bytes * nkv;
  const int code_bytes = kv4_code_bytes(bs, D);
  const unsigned char* kbase = static_cast<const unsigned char*>(a.cache.k) + kh * head_bytes;
  const unsigned char* vbase = static_cast<const unsigned char*>(a.cache.v) + kh * head_bytes;
  struct Stage {
    u32x2 k[NP], v[NP], vs[NP];
    u32x4 ks[NP];  // lanes in < NG: the scale bytes of a run's keys
    bool page[NP];
  };
  const int in = tid & 127;
  const int kin = (in / (D / 16)) * (D / 2) + 8 * (in % (D / 16)), vin = (in >> 1) * bs + 8 * (in & 1);
  const int sin = (in >> 5) * bs + 8 * (in & 1), ksin = in * bs;
  auto run_of = [&](int i) { return (wave >> 1) + NT / 128 * i; };
  auto pages = [&](int v, int (&pg)[NP]) {
    const int key = tile_key(min(v, nkt - 1));
#pragma unroll
    for (int i = 0; i < NP; ++i) pg[i] = bt[min(key + 16 * run_of(i), last) >> bsh];
  };
  auto load = [&](int v, const int (&pg)[NP], Stage& s) {
    const int key = tile_key(min(v, nkt - 1));
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int page = kv4_page(pg[i], a.cache.blocks), off = (key + 16 * run_of(i)) & bmask;
      const long at = (long)max(page, 0) * page_bytes;
      const unsigned char *kp = kbase + at, *vp = vbase + at + off;
      s.page[i] = page >= 0;
      if (D == 128 || in < D) {
        s.k[i] = *reinterpret_cast<const u32x2*>(kp + off * (D / 2) + (unsigned)kin);
        s.v[i] = *reinterpret_cast<const u32x2*>(vp + (unsigned)vin);
        s.vs[i] = *reinterpret_cast<const u32x2*>(vp + code_bytes + (unsigned)sin);
      }
      if (in < NG) s.ks[i] = *reinterpret_cast<const u32x4*>(kp + code_bytes + off + (unsigned)ksin);
    }
  };
  // what every thread does, without a branch, and the few that have more
  auto store = [&](Stage& s, Kv4Tile<D>& b) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int run = run_of(i);
      if (D != 128 && in >= D) continue;
      const int kk = 16 * run + in / (D / 16), krow = (kk & ~12) | ((kk & 4) << 1) | ((kk & 8) >> 1);
      *reinterpret_cast<u32x2*>(&b.k[krow * KLD + 8 * (in % (D / 16))]) = s.k[i];
      u32x4 even, odd;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const unsigned w = s.v[i][q], c = kv4_no_nan(s.vs[i][q]);
        const unsigned x0 = kv4_widen2<0>(w, __uint_as_float(c << 23)), x1 = kv4_widen2<1>(w, __uint_as_float(c << 15));
        const unsigned x2 = kv4_widen2<2>(w, __uint_as_float(c << 7)), x3 = kv4_widen2<3>(w, __uint_as_float(c >> 1));
        even[2 * q] = __builtin_amdgcn_perm(x1, x0, 0x05040100u);
        odd[2 * q] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
        even[2 * q + 1] = __builtin_amdgcn_perm(x3, x2, 0x05040100u);
        odd[2 * q + 1] = __builtin_amdgcn_perm(x3, x2, 0x07060302u);
      }
      unsigned short* dst = &b.v[(in & ~1) * VLD + 16 * run + 8 * (in & 1)];
      *reinterpret_cast<u32x4*>(dst) = even;
      *reinterpret_cast<u32x4*>(dst + VLD) = odd;
    }
  };
  auto store_scales = [&](const Stage& s, Kv4Tile<D>& b) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int run = run_of(i);
      if (D != 128 && in >= D) continue;
      if ((in & 30) == 0) {
        *reinterpret_cast<u32x2*>(&b.vs[in >> 5][16 * run + 8 * (in & 1)]) = s.vs[i];
        if (kv4_any_nan(s.vs[i][0]) || kv4_any_nan(s.vs[i][1])) nans = 1;
      }
      if (in < NG) *reinterpret_cast<u32x4*>(&b.ks[in][16 * run]) = s.ks[i];
      if (in == 0) b.nopage[run] = !s.page[i];
    }
  };

  Stage stage[UN];
  int pgs[UN][NP];
  auto ask = [&](int v) {  // the pages of tiles v .. v + UN - 1
#pragma unroll
    for (int u = 0; u < UN; ++u) pages(v + u, pgs[u]);
  };
  auto fetch = [&](int v) {
#pragma unroll
    for (int u = 0; u < UN; ++u) load(v + u, pgs[u], stage[u]);
  };
  if (nkt > 0) {
    ask(0);
    fetch(0);
    ask(UN);
  }

  // ---- q's two parts, a scale per 32 dims (see kv4.h)
  i32x8 qhi[KS], qlo[KS];
  int qs[KS];  // of the dims that this lane's 32 of a step's k are: 64 s + 32 half ..
  const float sl = kv4_score_scale(a.scale);
#pragma unroll
  for (int s = 0; s < KS; ++s) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      unsigned am = max(kv4_amax8(raw[s][2 * g]), kv4_amax8(raw[s][2 * g + 1]));
      am = max(am, (unsigned)__shfl_xor((int)am, 32, 64));
      const int own = kv4_query_scales(am);
      if (g == 0 || half) qs[s] = own;
      const float down = kv4_scale(own & 255), down16 = kv4_scale(own >> 8 & 255);
#pragma unroll
      for (int e = 2 * g; e < 2 * g + 2; ++e) {
        u32x2 hi, lo2;
        kv4_split8(raw[s][e], down, down16, hi, lo2);
        qhi[s][2 * e] = (int)hi[0];
        qhi[s][2 * e + 1] = (int)hi[1];
        qlo[s][2 * e] = (int)lo2[0];
        qlo[s][2 * e + 1] = (int)lo2[1];
      }
    }
  }

  f32x16 o[NG], st[2];
  bf16x8 pb[4];  // P of 16 keys a step
#pragma unroll
  for (int nb = 0; nb < NG; ++nb)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[nb][r] = 0.f;
  float m_run = kKv4Least, l_run = 0.f;
  bool far = false;  // of some row of the wave

  auto sees_some = [&](int v) {  // whether a row of the wave may see a key of tile v
    const int key = tile_key(v);
    return wrow0 < qlen && key <= wmax && (window <= 0 || key + kKv4Tile - 1 > wmin - window || key < sinks);
  };
  // scores: rows (keys) of the tile's halves, columns (queries) qi. Key 16 j + o of a half lies in row 16 j + r with o's bits 2 and 3
  // exchanged, and its scale byte at 16 j + 4 (o % 4) + o / 4
  const int ks_at = (qi & 16) | ((qi & 3) << 2) | ((qi >> 1) & 2) | ((qi >> 3) & 1);
  auto scores = [&](const Kv4Tile<D>& b) __attribute__((always_inline)) {
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
      for (int r = 0; r < 16; ++r) st[h2][r] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int g = min(2 * s + half, NG - 1);
      u32x4 kf[2];
      int ks[2];
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {
        kf[h2] = *reinterpret_cast<const u32x4*>(&b.k[(32 * h2 + qi) * KLD + 16 * g]);
        ks[h2] = b.ks[g][32 * h2 + ks_at];
        if (D == 96 && s == 1 && half) ks[h2] = 127;  // no such dims: q is zero there, whatever the scale of others is
      }
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2)
        st[h2] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kv4_pad(kf[h2]), qlo[s], st[h2], 4, 0, 0, ks[h2], 1, qs[s]);
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2)
        st[h2] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kv4_pad(kf[h2]), qhi[s], st[h2], 4, 0, 0, ks[h2], 0, qs[s]);
    }
  };
  auto softmax = [&](int v, const Kv4Tile<D>& b) __attribute__((always_inline)) {
    const int key = tile_key(v);
    const unsigned gone = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const unsigned*>(b.nopage));
    // hidden keys, in tiles that some row of the wave does not see whole; slot (h2, r): key 32 h2 + 16 (r >> 3) + 8 half + (r & 7)
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
      far = __any(kv4_far(m_run));
      l_run *= alpha;
#pragma unroll
      for (int nb = 0; nb < NG; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[nb][r] *= alpha;
    }
    float by = sl;
    if (far) {
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[h2][r] *= sl;
      by = 1.f;
    }
    // the sum is that of the rounded P, two at a time
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const f32x16& x = st[i >> 4];
      const bf16x2 p{static_cast<__bf16>(__builtin_amdgcn_exp2f(__builtin_fmaf(x[i & 15], by, -m_run))),
                     static_cast<__bf16>(__builtin_amdgcn_exp2f(__builtin_fmaf(x[(i & 15) + 1], by, -m_run)))};
      ps[(i >> 1) & 3] = __builtin_amdgcn_fdot2_f32_bf16(p, bf16x2{static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)}, ps[(i >> 1) & 3], false);
      pb[i >> 3][i & 7] = p[0];
      pb[i >> 3][(i & 7) + 1] = p[1];
    }
    l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
  };
  auto values = [&](int v, const Kv4Tile<D>& b) __attribute__((always_inline)) {
    const int bad = __builtin_amdgcn_readfirstlane(nans);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned short* vb = &b.v[qi * VLD + 16 * j + 8 * half];
#pragma unroll
      for (int nb = 0; nb < NG; ++nb) {
        const u16x8 va = *reinterpret_cast<const u16x8*>(vb + 32 * nb * VLD);
        o[nb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, va), pb[j], o[nb], 0, 0, 0);
      }
    }
    if (bad) {  // values of NaN may be among this tile's: into the rows that see them
      const int key = tile_key(v);
      unsigned long seen = 0;
      for (int j = 0; j < kKv4Tile; ++j)
        if (key + j < cap && !b.nopage[j >> 4] && kv4_sees(key + j, pos, window, sinks)) seen |= 1ul << j;
#pragma unroll
      for (int nb = 0; nb < NG; ++nb) {
        const unsigned long lost = __ballot(b.vs[nb][lane] == kKv4Nan);
        if (seen & lost)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[nb][r] = NAN;
      }
    }
  };

  if (tid == 0) nans = 0;
  __syncthreads();
  if constexpr (NWV == 8) {
    // two tiles a barrier. Half of the waves stage the next ones before their products, the others after them, so that the two waves of a
    // SIMD are at different work
    auto put = [&](int at) {
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        store(stage[u], buf[at + u]);
        store_scales(stage[u], buf[at + u]);
      }
    };
    auto tile = [&](int v, const Kv4Tile<D>& b) __attribute__((always_inline)) {
      if (!sees_some(v)) return;
      scores(b);
      softmax(v, b);
      values(v, b);
    };
    if (nkt > 0) {
      put(0);
      fetch(UN);
      ask(2 * UN);
    }
    __syncthreads();
    const bool early = wave >= NWV / 2;
    int at = 0;
    for (int v = 0; v < nkt; v += UN) {
      const int next = UN - at;
      if (early && v + UN < nkt) {
        put(next);
        fetch(v + 2 * UN);
        ask(v + 3 * UN);
      }
#pragma unroll 1
      for (int u = 0; u < UN; ++u)
        if (u == 0 || v + u < nkt) tile(v + u, buf[at + u]);
      if (!early && v + UN < nkt) {
        put(next);
        fetch(v + 2 * UN);
        ask(v + 3 * UN);
      }
      at = next;
      __syncthreads();
    }
  } else {
    // the values of a tile and the scores of the next one together; workgroups come two a compute unit
    if (nkt > 0) {
      store(stage[0], buf[0]);
      store_scales(stage[0], buf[0]);
      fetch(1);
      ask(2);
    }
    __syncthreads();
    bool live = false;  // whether the tile before has P
    for (int v = 0; v < nkt; ++v) {
      Kv4Tile<D>&b0 = buf[v & 1], &b1 = buf[~v & 1];
      if (live) values(v - 1, b1);
      live = sees_some(v);
      if (live) scores(b0);
      __syncthreads();
      if (live) softmax(v, b0);
      if (v + 1 < nkt) {
        store(stage[0], b1);
        store_scales(stage[0], b1);
        fetch(v + 2);
        ask(v + 3);
      }
      __syncthreads();
    }
    if (live) values(nkt - 1, buf[(nkt - 1) & 1]);
  }
  l_run = kv4_sum32(l_run);
  if (run < blk.nkt) {  // a part of the rows' keys: sums and maxima as they are, a lane's 16 bytes beside its neighbours'
    if (wrow0 >= qlen) return;
    const long part = (((long)(t * SUB + sub) * gridDim.x + heads) * splits + split) * NWV + wave;
    f32x4* dst = reinterpret_cast<f32x4*>(work + part * 32 * D) + lane;
    if (wrow0 + qi >= qlen) return;
#pragma unroll
    for (int nb = 0; nb < NG; ++nb)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        dst[(4 * nb + g) * 64] = f32x4{o[nb][4 * g], o[nb][4 * g + 1], o[nb][4 * g + 2], o[nb][4 * g + 3]};
    float* ml = work + (long)gridDim.x * gridDim.y * gridDim.z * NWV * 32 * D + part * 64;
    if (half == 0) *reinterpret_cast<float2*>(ml + 2 * qi) = float2{m_run, l_run};
    return;
  }
  // ---- rows through LDS, so that a row's dims leave together
  __syncthreads();
  if (wrow0 >= qlen) return;
  const float inv = l_run == 0.f ? 0.f : 1.f / l_run;  // a row that sees nothing: zeros
  constexpr int OLD = D + 8;
  static_assert(NWV * 32 * OLD * 2 <= 2 * UN * sizeof(Kv4Tile<D>), "the waves' rows fit the tiles' LDS");
  unsigned short* ol = reinterpret_cast<unsigned short*>(smem) + wave * 32 * OLD;
#pragma unroll
  for (int nb = 0; nb < NG; ++nb)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      u16x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = f32_to_bf16(o[nb][4 * g + j] * inv);
      *reinterpret_cast<u16x4*>(ol + qi * OLD + 32 * nb + 8 * g + 4 * half) = w;
    }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // other lanes read what this one wrote
  __builtin_amdgcn_wave_barrier();
  unsigned short* op = static_cast<unsigned short*>(a.out) + (long)(q0 + wrow0) * a.out_stride + (long)h * D;
#pragma unroll
  for (int i = 0; i < 32 * D / 8; i += 64) {
    const int r = (i + lane) / (D / 8), c = (i + lane) % (D / 8);
    if (wrow0 + r < qlen)
      *reinterpret_cast<u16x8*>(op + r * a.out_stride + 8 * c) = *reinterpret_cast<const u16x8*>(ol + r * OLD + 8 * c);
  }
}

// Merges the parts of 32 rows of a head: a wave each, and each for 8 of the dims.
template <int D, int HG, int NWV>
__global__ __launch_bounds__(64) void kv4_prefill_merge_kernel(Kv4Attn a, const int* __restrict__ cu_q, int seqs,
                                                               const int* __restrict__ ctx_lens, int rows,
                                                               const int* __restrict__ tiles, const float* __restrict__ work, int splits) {
  constexpr int QR = 32 * NWV / HG, SUB = 128 / QR;
  const int heads = blockIdx.x / NWV, wave = blockIdx.x % NWV, t = blockIdx.y / SUB, sub = blockIdx.y % SUB;
  Kv4Block blk;
  if (!kv4_block<QR>(blk, a, cu_q, seqs, ctx_lens, rows, tiles, t, sub)) return;
  const int run = kv4_tile_run(blk.nkt, splits), parts = (blk.nkt + run - 1) / run;
  const int lane = threadIdx.x, qi = lane & 31, half = lane >> 5, row = blk.r0 + wave / HG * 32 + qi;
  if (parts <= 1 || row >= blk.qlen) return;
  const long part0 = ((long)blockIdx.y * (gridDim.x / NWV) + heads) * splits * NWV + wave;
  const float* ml = work + (long)gridDim.x * gridDim.y * splits * 32 * D + part0 * 64 + 2 * qi;
  const f32x4* src = reinterpret_cast<const f32x4*>(work + part0 * 32 * D) + blockIdx.z * 64 + lane;
  float M = kKv4Least;
  for (int p0 = 0; p0 < parts; p0 += 8)
#pragma unroll
    for (int u = 0; u < 8; ++u) M = fmaxf(M, ml[(long)min(p0 + u, parts - 1) * NWV * 64]);
  float l = 0.f;
  f32x4 o{0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < parts; p0 += 8)
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int p = min(p0 + u, parts - 1);
      const float2 x = *reinterpret_cast<const float2*>(ml + (long)p * NWV * 64);
      const f32x4 y = src[(long)p * NWV * 8 * D];
      if (p0 + u < parts) {
        const float w = __builtin_amdgcn_exp2f(x.x - M);
        l += w * x.y;
        o += w * y;
      }
    }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  u16x4 y;
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = f32_to_bf16(o[j] * inv);
  *reinterpret_cast<u16x4*>(static_cast<unsigned short*>(a.out) + (long)(blk.q0 + row) * a.out_stride +
                            (long)(heads * HG + wave % HG) * D + 8 * blockIdx.z + 4 * half) = y;
}

// query heads a workgroup: as many as divide a kv head's, up to 8 waves
static int kv4_prefill_heads(const Kv4Attn& a) {
  const int G = a.nq / a.cache.nkv;
  return G % 8 == 0 ? 8 : G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1;
}

int kv4_prefill_splits(const Kv4Attn& a, int seqs, int rows, int ntiles, long* floats) {
  const int HG = kv4_prefill_heads(a), NWV = HG == 1 ? 4 : 8, QR = 32 * NWV / HG;
  const long wgs = (long)ntiles * (128 / QR) * (a.nq / HG), slots = HG == 1 ? 512 : 256;  // what the chip holds at once
  const long live = min(wgs, ((long)rows / QR + seqs) * (a.nq / HG));  // that have rows, at most
  const long cap = (long)a.bt_width * a.cache.block_size;
  const long seen = a.window > 0 ? min(cap, (long)a.window + a.sinks + QR + 2 * kKv4Tile) : cap;  // at most, by a workgroup
  // a workgroup's part is 133 KB at most, and no call takes more than slots * 128 / QR of them (136 MB): tiles beyond those of its rows, as a
  // padded list has them, leave room for fewer runs
  const long most = min(slots / max(live, 1l), slots * (128 / QR) / max(wgs, 1l));
  const long splits = live <= 0 || wgs > 2048 ? 1 : max(1l, min(most, seen / kKv4Tile / kKv4LeastRun));
  *floats = splits > 1 ? wgs * splits * NWV * 32 * (a.cache.D + 2) : 0;
  return (int)splits;
}

template <int D, int HG, int NWV>
static void kv4_prefill(const Kv4Attn& a, const int* cu_q, int seqs, const int* ctx, int rows, const int* tiles, int ntiles,
                        float* work, int splits, hipStream_t s) {
  constexpr int SUB = 128 / (32 * NWV / HG);
  constexpr int UN = NWV == 8 ? 2 : 1;
  constexpr int kLds = 2 * UN * sizeof(Kv4Tile<D>);
  if (kLds > 64 * 1024) {  // more than the default limit: asked for once a device
    static std::atomic<unsigned long> asked{0};
    int dev = 0;
    (void)hipGetDevice(&dev);
    const unsigned long bit = 1ul << (dev & 63);
    if ((asked.load(std::memory_order_relaxed) & bit) == 0 &&
        hipFuncSetAttribute(reinterpret_cast<const void*>(&kv4_prefill_kernel<D, HG, NWV, UN>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, kLds) == hipSuccess)
      asked.fetch_or(bit, std::memory_order_relaxed);
  }
  const bool apart = splits > 1 || 4l * rows <= 3l * 128 * ntiles;
  const int groups = a.nq / HG;
  kv4_prefill_kernel<D, HG, NWV, UN><<<apart ? dim3(groups, ntiles, SUB * splits) : dim3(groups, SUB, ntiles), 64 * NWV, kLds, s>>>(
      a, cu_q, seqs, ctx, rows, tiles, apart, work);
  if (splits > 1)
    kv4_prefill_merge_kernel<D, HG, NWV><<<dim3(groups * NWV, ntiles * SUB, D / 8), 64, 0, s>>>(a, cu_q, seqs, ctx, rows, tiles, work, splits);
}

template <int D>
static void kv4_prefill_d(const Kv4Attn& a, const int* cu_q, int seqs, const int* ctx, int rows, const int* tiles, int ntiles,
                          float* work, int splits, hipStream_t s) {
  switch (kv4_prefill_heads(a)) {
    case 8: return kv4_prefill<D, 8, 8>(a, cu_q, seqs, ctx, rows, tiles, ntiles, work, splits, s);
    case 4: return kv4_prefill<D, 4, 8>(a, cu_q, seqs, ctx, rows, tiles, ntiles, work, splits, s);
    case 2: return kv4_prefill<D, 2, 8>(a, cu_q, seqs, ctx, rows, tiles, ntiles, work, splits, s);
    default: return kv4_prefill<D, 1, 4>(a, cu_q, seqs, ctx, rows, tiles, ntiles, work, splits, s);
  }
}

void launch_kv4_prefill(const Kv4Attn& a, const int* cu_q, int seqs, const int* ctx_lens, int rows, const int* tiles,
                        int ntiles, float* work, int splits, hipStream_t s) {
  if (ntiles <= 0) return;
  if (a.cache.D == 128) kv4_prefill_d<128>(a, cu_q, seqs, ctx_lens, rows, tiles, ntiles, work, splits, s);
  else if (a.cache.D == 96) kv4_prefill_d<96>(a, cu_q, seqs, ctx_lens, rows, tiles, ntiles, work, splits, s);
  else kv4_prefill_d<64>(a, cu_q, seqs, ctx_lens, rows, tiles, ntiles, work, splits, s);
}

}  // namespace hipserve
