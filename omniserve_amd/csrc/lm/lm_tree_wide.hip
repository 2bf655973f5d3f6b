// Attention of drafted tokens, many rows (tokens * heads per kv head): the waves of a workgroup have 16 or 32 rows each and share a ring of key and
// value tiles that DMA fills two tiles ahead.  See lm_tree_attn.hip for the formula; here a tile is 64 keys of codes, or 32 of elements.
//
// Bound by the vector units beside the matrix units (a softmax weight costs 4 vector instructions, one of them an exponential of four times the
// length, and 256 operations of the matrix units), and by the latency between them, so that what a weight does not need is done elsewhere:
//   a key is decoded with its power of two into bf16, which holds it exactly.  (Products of the codes themselves, at twice the rate and without the decoding, made
//     4 trees of 64 over 32768 keys 175 us where this takes 205, but the matrix units add products of 8-bit floats in fewer than 32 bits: a sum of 128 was off by
//     up to 2^-12 of its largest product, of bf16 by 2^-21);
//   a value's exponent (lm_tree_attn.hip) is the products' initial accumulator, e / scale;
//   2^-e and e / scale are formed by one lane per key and read back from LDS.
// 4 trees of 64 over 32768 keys, 32 heads over 8: 205 - 210 us a call, 0.65 PFLOP/s; matrix units busy 30 % of the time, vector units 53, waves wait for 43 % of
// theirs, no LDS conflicts (workgroups of half the rows 215 for 212 us, over elements 136 for 139).
#include "lm_tree.h"

namespace lm {

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

#if LM_ELEM == 0
// The 16-byte slot of a row of dk bytes that the fragments of 16 rows are read from
template <int ROWB>
__device__ __forceinline__ int key_swizzle(int row) {
  if constexpr (ROWB == 64) return (4 - (row >> 2 & 3)) & 3;
  else return Tile<ROWB>::swizzle(row);
}

// Blocks of 16 rows of a wave: what 256 registers hold
constexpr int row_blocks(int dk, int dv) { return dk > 128 || dv > 128 ? 1 : 2; }

template <int DK, int DV, int NW, bool CODES>
struct Wide {
  static constexpr int NR = row_blocks(DK, DV), ROWS = NW * 16 * NR, NVB = DV / 16;
  static constexpr int KT = CODES ? 64 : 32, NU = KT / 16;
  static constexpr int KB = CODES ? DK : 2 * DK, VB = CODES ? DV : 2 * DV;      // bytes of a row
  static constexpr int KBYTES = KT * KB, VBYTES = KT * VB, EXPS = CODES ? 128 : 0;
  static constexpr int SLOT = KBYTES + VBYTES + EXPS;                            // of the ring
  static constexpr int NBUF = NW == 2 ? 2 : 3;
  static constexpr int KP = KBYTES / 1024, VP = VBYTES / 1024, EACH = (KP + VP + NW - 1) / NW, PIECES = EACH + (CODES ? 2 : 0);      // of a wave
  static constexpr int OWN = CODES ? 512 : 0;                                     // a wave's: keys' exponents
  static constexpr int LDS = NBUF * SLOT + NW * OWN + 64;
  static constexpr float SHIFT = CODES ? 7.f : ELEMS_SHIFT;                      // weights of codes are f16: at most 2^(LAZY + 7)
  typedef Tile<2 * DV> VT;
  typedef Tile<2 * DK> KTile;
};

template <int DK, int DV, int NW, bool CODES>
__global__ __launch_bounds__(64 * NW, 2) void tree_wide_kernel(TreeArgs p) {
  typedef Wide<DK, DV, NW, CODES> W;
  constexpr int NR = W::NR, NU = W::NU, NVB = W::NVB, KT = W::KT;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  Piece s;
  int64_t part = 0;
  if (!piece_of<KT, W::ROWS>(p, s, part)) return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l15 = lane & 15, l4 = lane >> 4;
  uint8_t* own = lds + W::NBUF * W::SLOT + wave * W::OWN;
  // smallest, largest of the rows' bounds; whether a context tile has non-finite values; whether a drafted tile had some (a word of its own that nobody clears: a
  // wave may still have to read what another one would clear); whether the sums have some
  int* shared = (int*)(lds + W::NBUF * W::SLOT + NW * W::OWN);
  const int r0 = s.rb * W::ROWS + wave * 16 * NR;
  const bool live = r0 < s.R;                                         // (a wave without rows fetches its pieces and waits with the others)

  const int ta = s.t0 + min(s.from, s.nt), tb = s.t0 + min(s.to, s.nt);

  // ---- the ring ----
  // Offsets of this lane's pieces: place in the slot -> byte of the tile in memory
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  auto piece_of = [&](int j) { return min(j * NW + wave, W::KP + W::VP - 1); };      // (the last piece twice where they do not divide: equal bytes)
  uint32_t from[W::EACH];
#pragma unroll
  for (int j = 0; j < W::EACH; ++j) {
    const int pc = piece_of(j), key = pc < W::KP, at = (key ? pc : pc - W::KP) * 1024 + lane * 16, rowb = key ? W::KB : W::VB, row = at / rowb;
    const int swz = key ? (CODES ? key_swizzle<W::KB>(row) : W::KTile::swizzle(row)) : (CODES ? code_swizzle<DV>(row) : W::VT::swizzle(row));
    from[j] = row * rowb + (((at % rowb >> 4) ^ swz) << 4);
  }
  auto fetch = [&](int t, int page, int slot) {
    const int64_t at = ((int64_t)min(max(page, 0), p.pages - 1) * p.G + s.g) * PAGE + (CODES ? 0 : t * KT % PAGE);
    const uint32_t to = lds0 + slot * W::SLOT;
#pragma unroll
    for (int j = 0; j < W::EACH; ++j) {
      const int pc = piece_of(j);
      dma16_uncounted(pc < W::KP ? p.kc + at * W::KB : p.vc + at * W::VB, from[j], to + pc * 1024);
    }
    if constexpr (CODES)      // (every wave, so that all have as many pieces in flight: the same bytes to the same place)
      if (lane < 4) {
        dma16_uncounted(p.ke + at, 16 * lane, to + W::KBYTES + W::VBYTES);
        dma16_uncounted(p.ve + at, 16 * lane, to + W::KBYTES + W::VBYTES + 64);
      }
  };
  constexpr int PER_PAGE = PAGE / KT;
  // (scalar loads: a vector load's wait would take in the DMA behind it)
  const __attribute__((address_space(4))) int* bt = (const __attribute__((address_space(4))) int*)(uintptr_t)s.bt;
  auto page_of = [&](int t) { return t < tb ? bt[t / PER_PAGE] : 0; };
  int pages[W::NBUF];      // of tiles t, t + 1, ..
  auto fetch_first = [&]() {
#pragma unroll
    for (int j = 0; j < W::NBUF; ++j) pages[j] = page_of(ta + j);
#pragma unroll
    for (int j = 0; j < W::NBUF - 1; ++j)
      if (ta + j < tb) fetch(ta + j, pages[j], j);
  };
  fetch_first();

  // ---- rows ----
  auto token_of = [&](int i) { return s.f0 + min(r0 + 16 * i + l15, s.R - 1) / s.gs; };
  auto query_of = [&](int i) {
    const int tk = token_of(i);
    return p.q + (int64_t)tk * p.ldq + (int64_t)(s.g * s.gs + min(r0 + 16 * i + l15, s.R - 1) - (tk - s.f0) * s.gs) * DK;
  };
  auto row_ok = [&](int i) { return r0 + 16 * i + l15 < s.R; };
  int low[NR], low_min = INT32_MAX, low_max = INT32_MIN;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int lo = bound_of(p, p.pos[token_of(i)]);
    low_min = min(low_min, lo);
    low_max = max(low_max, lo);
    low[i] = row_ok(i) ? lo : INT32_MAX;
  }
  if (tid == 0) { shared[0] = INT32_MAX; shared[1] = INT32_MIN; shared[3] = shared[4] = 0; }
  __syncthreads();
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) {
    low_min = min(low_min, __shfl_xor(low_min, m, 64));
    low_max = max(low_max, __shfl_xor(low_max, m, 64));
  }
  if (lane == 0) { atomicMin(&shared[0], low_min); atomicMax(&shared[1], low_max); }
  __syncthreads();
  low_min = __builtin_amdgcn_readfirstlane(shared[0]);
  low_max = __builtin_amdgcn_readfirstlane(shared[1]);
  const int k0 = max(low_min, -1) + 1;

  // ---- queries ----
  frag_t qf[NR][DK / 32];      // (of codes: the order that half a slot of 16 codes has)
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const elem_t* qrow = query_of(i);
#pragma unroll
    for (int k = 0; k < DK / 32; ++k) qf[i][k] = row_ok(i) ? *(const frag_t*)(qrow + (CODES ? 64 * (k >> 1) + 16 * l4 + 8 * (k & 1) : 32 * k + 8 * l4)) : frag_t{};
  }

  f32x4 acc[NR][NVB];
  float m_run[NR], l_run[NR];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < NR; ++i) {
#pragma unroll
      for (int c = 0; c < NVB; ++c) acc[i][c] = zero4();
      m_run[i] = NEG;
      l_run[i] = 0.f;
    }
  };
  clear();
  const float inv_scale = 1.0f / p.scale;

  Loudness loud;
  // x: scores (with e / scale), unseen ones NEG -> weights; inv: 2^-e (one: there are none), mine: of the key whose number this lane has
  auto softmax = [&](int i, auto& x, const auto& inv, auto one, float mine) {
    constexpr int U = sizeof(x) / sizeof(f32x4);
    float t = NEG;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) t = fmaxf(t, x[u][r]);
    t = rows_max(t);
    t = t <= NEG ? NEG : t * p.scale;
    bool low = !one.value && loud.quiet(mine);
    const bool grows = t > m_run[i] + (low ? 0.f : LAZY);      // (the first key's always; a NaN never)
    const bool some = __any(grows);
    const float m_new = grows ? t : m_run[i], m_sub = (m_new <= NEG ? 0.f : m_new) - W::SHIFT;
    if constexpr (!one.value)
      if (some) {
        loud.set(-rows_max(lanes_max<16>(-mine)));
        low = loud.quiet(mine);
      }
    float own = 0.f, sum = 0.f;
    if (!one.value && low) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float root = __builtin_amdgcn_exp2f(__builtin_fmaf(x[u][r], 0.5f * p.scale, -0.5f * m_sub));
          own = __builtin_fmaf(root * inv[u][r], root, own);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[u][r], p.scale, -m_sub));
        if constexpr (one.value) sum += x[u][r];
        else sum = __builtin_fmaf(x[u][r], inv[u][r], sum);
      }
    if (some) {
      const float root = root_of(m_run[i], m_new);
      l_run[i] = l_run[i] * root * root;
#pragma unroll
      for (int c = 0; c < NVB; ++c) acc[i][c] = acc[i][c] * root * root;
    }
    l_run[i] += low ? own : sum;
    m_run[i] = m_new;
  };
  auto wave_sync = [&]() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  // What non-finite values among keys lo .. hi - 1 of a tile add to the rows that see them.  (They were left out of the products, where a weight of
  // zero would have made them NaN in every row; a weight's size does not matter to them.)
  auto add_nonfinite = [&](int i, int lo, int hi, auto seen, auto value) {
#pragma unroll 1
    for (int j = max(lo, 0); j < hi; ++j) {
      const bool see = seen(i, j);
#pragma unroll
      for (int c = 0; c < NVB; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float y = value(j, 16 * c + 4 * l4 + r);
          acc[i][c][r] += (int)see & (int)!(fabsf(y) < __builtin_inff()) ? y : 0.f;
        }
    }
  };
  // A tile of 32 keys and values in elements: products, weights, products; ev, inv, mine: of a codes' kernel's drafted values, as those of codes
  auto elem_products = [&](const uint8_t* kt, const uint8_t* vt, const frag_t (&q)[NR][DK / 32], bool edge, bool bad, const f32x4 (&ev)[2], const f32x4 (&inv)[2], float mine, int lo,
                           int hi, auto seen, auto value) {
    f32x4 x[NR][2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int k = 0; k < DK / 32; ++k) {
        const frag_t kf = W::KTile::frag(kt, 16 * u + l15, 4 * k + l4);
#pragma unroll
        for (int i = 0; i < NR; ++i) x[i][u] = mma(kf, q[i][k], k > 0 ? x[i][u] : CODES ? ev[u] : zero4());
      }
    quad_t pq[NR][2][2];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      if (edge) {
        const int key = here(4 * l4);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) x[i][u][r] = seen(i, key + 16 * u + r) ? x[i][u][r] : NEG;
      }
      if constexpr (CODES) softmax(i, x[i], inv, No(), mine);
      else softmax(i, x[i], inv, Yes(), mine);
#pragma unroll
      for (int u = 0; u < 2; ++u) split_quad(x[i][u], pq[i][u]);
    }
#pragma unroll
    for (int c = 0; c < NVB; ++c) {
      const quad_t v0 = W::VT::column_quad(vt, 0, c, l15, l4), v1 = W::VT::column_quad(vt, 16, c, l15, l4);
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int m = 0; m < 2; ++m) acc[i][c] = mma_quads(v0, v1, pq[i][0][m], pq[i][1][m], acc[i][c]);
    }
    if (bad) {
#pragma unroll
      for (int i = 0; i < NR; ++i) add_nonfinite(i, lo, hi, seen, value);
    }
  };
  // Values of a tile of elements that not every row sees: rows outside lo .. hi - 1 and non-finite ones become zero -> whether there were non-finite ones
  auto clean_elems = [&](uint8_t* vt, int lo, int hi) {
    if (tid == 0) shared[2] = 0;
    __syncthreads();
    bool bad = false;
    for (int i = tid; i < 32 * DV / 8; i += 64 * NW) {
      const int row = i / (DV / 8);
      frag_t* at = (frag_t*)(vt + W::VT::slot(row, i % (DV / 8)));
      frag_t f = *at;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float y = row >= lo && row < hi ? (float)f[k] : 0.f;
        const bool fine = fabsf(y) < __builtin_inff();
        bad |= !fine;
        f[k] = (elem_t)(fine ? y : 0.f);
      }
      *at = f;
    }
    if (bad) atomicOr(&shared[2], 1);
    __syncthreads();
    return shared[2] != 0;
  };

  // ---- the context ----
  int slot = 0;
  bool careful = false;      // (a second time over the tiles, where infinite elements may have become NaN: see the other kernel)
  for (int t = ta; t < tb;) {
    const int kb = t * KT, page = pages[0], hi = (uint32_t)page < (uint32_t)p.pages ? s.length - kb : 0, lo = max(k0 - kb, 0);
    const bool edge = careful || hi < KT || kb <= low_max;
    if (W::NBUF > 2 && t + 1 < tb) wait_pieces<W::PIECES>();
    else wait_pieces<0>();
    __syncthreads();      // tile t is there; everyone has read the one before it
    if (t + W::NBUF - 1 < tb) fetch(t + W::NBUF - 1, pages[W::NBUF - 1], slot + W::NBUF - 1 >= W::NBUF ? slot - 1 : slot + W::NBUF - 1);
#pragma unroll
    for (int j = 0; j + 1 < W::NBUF; ++j) pages[j] = pages[j + 1];
    pages[W::NBUF - 1] = page_of(t + W::NBUF);
    uint8_t* kt = lds + slot * W::SLOT;
    uint8_t* vt = kt + W::KBYTES;
    slot = slot + 1 == W::NBUF ? 0 : slot + 1;
    const int64_t at = ((int64_t)min(max(page, 0), p.pages - 1) * p.G + s.g) * PAGE + (CODES ? 0 : kb % PAGE);
    auto seen = [&](int i, int key) { return (bool)((int)(key >= lo) & (int)(key < hi) & (int)(kb + key > low[i])); };
    bool bad = false;
    if constexpr (!CODES) {
      if (edge) bad = clean_elems(vt, lo, hi);
      if (live) {
        const elem_t* vb = (const elem_t*)p.vc + at * DV;
        const f32x4 none[2] = {};
        elem_products(kt, vt, qf, edge, bad, none, none, 0.f, lo, min(hi, KT), seen, [&](int j, int d) { return (float)vb[j * DV + d]; });
      }
    } else {
      uint8_t* exps = vt + W::VBYTES;
      if (edge) {
        if (tid == 0) shared[2] = 0;
        __syncthreads();
        for (int i = tid; i < KT * DV / 16; i += 64 * NW) {
          const int row = i / (DV / 16);
          u32x4* to = (u32x4*)(vt + row * DV + (i % (DV / 16)) * 16);      // (a row's slots in any order)
          u32x4 w = *to;
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = row >= lo && row < hi ? drop_nan_codes(w[k], bad) : 0u;
          *to = w;
        }
        if (tid < KT && !(tid >= lo && tid < hi)) exps[64 + tid] = 127;
        if (bad) atomicOr(&shared[2], 1);
        __syncthreads();
        bad = shared[2] != 0;
      }
      if (live) {
        f32x4* both = (f32x4*)own;      // e / scale of 64 keys, then 2^-e
        const uint32_t byte = exps[64 + lane];
        const float mine = __uint_as_float((254 - byte) << 23);
        wave_sync();
        ((float*)own)[lane] = ((float)byte - 127.f) * inv_scale;
        ((float*)own)[64 + lane] = mine;
        wave_sync();
        f32x4 x[NR][NU], inv[NU];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const f32x4 ev = both[4 * u + l4];
          inv[u] = both[16 + 4 * u + l4];
          const float scale = scale_of(exps[16 * u + l15]);
#pragma unroll
          for (int j = 0; j < DK / 64; ++j) {
            const int row = 16 * u + l15;
            const u32x4 w = *(const u32x4*)(kt + row * DK + (((4 * j + l4) ^ key_swizzle<DK>(row)) << 4));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const frag_t kf = code_frag(w, h, scale);
#pragma unroll
              for (int i = 0; i < NR; ++i) x[i][u] = mma(kf, qf[i][2 * j + h], j == 0 && h == 0 ? ev : x[i][u]);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int u = 0; u < NU; ++u) asm volatile("" : "+v"(x[i][u]));      // (not later: the keys' registers are free here)
        // A column's read is requested eight products ahead: its latency is as long as six of them
        const int base = code_column<DV>(l15, l4);
        constexpr int AHEAD = NVB < 8 ? NVB : 8;
        u32x2 w[AHEAD];
#pragma unroll
        for (int c = 0; c < AHEAD; ++c) w[c] = read_code_column<DV>(vt, base, 0, c);
        __builtin_amdgcn_sched_barrier(0);
        f16x4 pq[NR][NU];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          if (edge) {
            const int key = here(4 * l4);
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
              for (int r = 0; r < 4; ++r) x[i][u][r] = seen(i, key + 16 * u + r) ? x[i][u][r] : NEG;
          }
          softmax(i, x[i], inv, No(), mine);
#pragma unroll
          for (int u = 0; u < NU; ++u) pq[i][u] = (f16x4){(_Float16)x[i][u][0], (_Float16)x[i][u][1], (_Float16)x[i][u][2], (_Float16)x[i][u][3]};
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < NVB; ++c) {
            const f16x8 vf = code_halves(w[c % AHEAD]);
            if (h * NVB + c + AHEAD < 2 * NVB) w[c % AHEAD] = read_code_column<DV>(vt, base, c + AHEAD < NVB ? h : 1, (c + AHEAD) % NVB);
#pragma unroll
            for (int i = 0; i < NR; ++i)
              acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, __builtin_shufflevector(pq[i][2 * h], pq[i][2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7), acc[i][c], 0, 0, 0);
          }
        if (bad) {
          const uint8_t* vb = p.vc + at * DV;
#pragma unroll
          for (int i = 0; i < NR; ++i) add_nonfinite(i, lo, min(hi, KT), seen, [&](int j, int d) { return (vb[j * DV + d] & 127) == 127 ? __builtin_nanf("") : 0.f; });
        }
      }
    }
    ++t;
    if constexpr (!CODES)
      if (t == tb && !careful) {
        float z = 0.f;
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int c = 0; c < NVB; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) z = __builtin_fmaf(acc[i][c][r], 0.f, z);
        if (__any(z != 0.f) && lane == 0) atomicOr(&shared[4], 1);
        __syncthreads();
        if (shared[4] != 0) {
          careful = true;
          t = ta;
          slot = 0;
          clear();
          fetch_first();
        }
      }
  }

  // ---- the drafted tokens ----
  if (s.to > s.nt) {
    typedef Wide<DK, DV, NW, false> E;      // 32 keys of elements in the ring's memory
    frag_t q[NR][DK / 32];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const elem_t* qrow = query_of(i);
#pragma unroll
      for (int k = 0; k < DK / 32; ++k) q[i][k] = row_ok(i) ? *(const frag_t*)(qrow + 32 * k + 8 * l4) : frag_t{};
    }
    for (int j0 = 32 * max(s.from - s.nt, 0); j0 < min(s.drafted, 32 * (s.to - s.nt)); j0 += 32) {
      const int rows = min(s.drafted - j0, 32);
      const int64_t row0 = s.f0 + j0;
      uint8_t* kt = lds;
      uint8_t* vt = lds + E::KBYTES;
      // Values pass through registers: non-finite ones are left out, and beside codes a token's are divided by a power of two of their own
      constexpr int VF = (32 * DV / 8 + 64 * NW - 1) / (64 * NW);
      float* exps = (float*)(lds + W::NBUF * W::SLOT);      // e / scale, from 64 on 2^-e (beside codes: the first wave's own)
      frag_t vf[VF];
      bool bad = false;
#pragma unroll
      for (int k = 0; k < VF; ++k) {
        const int i = tid + 64 * NW * k, row = i / (DV / 8), c = i % (DV / 8);
        vf[k] = row < rows ? *(const frag_t*)(p.v + (row0 + row) * p.ldv + (int64_t)s.g * DV + 8 * c) : frag_t{};
      }
      __syncthreads();      // what was there has been read
      for (int i = tid; i < 32 * DK / 8; i += 64 * NW) {
        const int row = i / (DK / 8), c = i % (DK / 8);
        *(frag_t*)(kt + W::KTile::slot(row, c)) = *(const frag_t*)(p.k + (row0 + min(row, rows - 1)) * p.ldk + (int64_t)s.g * DK + 8 * c);
      }
#pragma unroll
      for (int k = 0; k < VF; ++k) {
        const int i = tid + 64 * NW * k, row = i / (DV / 8), c = i % (DV / 8);
        float top = 0.f;
#pragma unroll
        for (int m = 0; m < 8; ++m) {
          const float y = (float)vf[k][m];
          const bool fine = fabsf(y) < __builtin_inff();
          bad |= !fine;
          vf[k][m] = fine ? vf[k][m] : (elem_t)0.f;
          top = fine ? fmaxf(top, fabsf(y)) : top;
        }
        if constexpr (CODES) {
          const int e = row < rows ? row_exponent(lanes_max<DV / 8>(top)) : 0;
          const float f = pow2(-e);
#pragma unroll
          for (int m = 0; m < 8; ++m) vf[k][m] = (elem_t)((float)vf[k][m] * f);
          if (row < 32 && c == 0) {
            exps[row] = (float)e * inv_scale;
            exps[64 + row] = f;
          }
        }
        if (row < 32) *(frag_t*)(vt + W::VT::slot(row, c)) = vf[k];
      }
      if (__any(bad) && lane == 0) atomicOr(&shared[3], 1);
      __syncthreads();
      bad = shared[3] != 0;      // (of this tile or one before: then this one is looked through for nothing)
      if (!live) continue;
      uint32_t bits[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i)
        bits[i] = row_ok(i) && (j0 >> 6) < p.words ? (uint32_t)(p.mask[(int64_t)token_of(i) * p.words + (j0 >> 6)] >> (j0 & 63)) : 0u;
      f32x4 ev[2] = {}, inv[2] = {};
      float mine = 0.f;
      if constexpr (CODES) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          ev[u] = *(const f32x4*)&exps[16 * u + 4 * l4];
          inv[u] = *(const f32x4*)&exps[64 + 16 * u + 4 * l4];
        }
        mine = exps[64 + (lane & 31)];
      }
      const elem_t* vb = p.v + row0 * p.ldv + (int64_t)s.g * DV;
      elem_products(kt, vt, q, true, bad, ev, inv, mine, 0, rows,
                    [&](int i, int key) {
                      return (bool)((int)(key < rows) & (int)(bits[i] >> key & 1) & (int)(p.pos[min((int)row0 + key, s.f0 + s.drafted - 1)] > low[i]));
                    },
                    [&](int j, int d) { return (float)vb[j * p.ldv + d]; });
    }
  }

  // ---- results ----
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const float l = column_sum(l_run[i]);
    if (!row_ok(i)) continue;
    const int r = r0 + 16 * i + l15, tk = r / s.gs, h = s.g * s.gs + r - tk * s.gs;
    if (!s.whole) {
      const int64_t at = part + wave * 16 * NR + 16 * i + l15;
#pragma unroll
      for (int c = 0; c < NVB; ++c) *(f32x4*)(p.part + at * DV + 16 * c + 4 * l4) = acc[i][c];
      if (l4 == 0) { p.ml[2 * at] = m_run[i]; p.ml[2 * at + 1] = l; }
    } else {
      const float f = l != 0.f ? 1.0f / l : 0.f;
#pragma unroll
      for (int c = 0; c < NVB; ++c) *(quad_t*)(p.o + (int64_t)(s.f0 + tk) * p.ldo + (int64_t)h * DV + 16 * c + 4 * l4) = to_quad(acc[i][c] * f);
    }
  }
}

template <int DK, int DV, int NW, bool CODES>
static int launch(const TreeArgs& a, hipStream_t s) {
  typedef Wide<DK, DV, NW, CODES> W;
  static_assert(W::NBUF * W::SLOT >= 32 * 2 * (DK + DV), "a drafted tile fits the ring");
  constexpr size_t bytes = W::LDS;
  if (allow_lds(tree_wide_kernel<DK, DV, NW, CODES>, bytes) != LM_OK) return LM_EINVAL;
  hipLaunchKernelGGL((tree_wide_kernel<DK, DV, NW, CODES>), dim3((a.workgroups + 7) / 8 * 8), dim3(64 * NW), bytes, s, a);
  return launch_status();
}

// Waves of a workgroup: as few as hold the rows, as many as share a tile
static int waves(int rows, int dk, int dv) {
  const int per = 16 * row_blocks(dk, dv);
  return rows <= 2 * per ? 2 : rows <= 4 * per ? 4 : 8;
}

bool tree_wide_takes(int rows, int dk, int dv) { return rows > 16 * row_blocks(dk, dv); }
int tree_wide_rows(int rows, int dk, int dv) { return waves(rows, dk, dv) * 16 * row_blocks(dk, dv); }

int tree_wide_fit(int rows, int dk, int dv, bool codes) {
  const int nw = waves(rows, dk, dv), each = codes ? 1 : 2;
  const int lds = (nw == 2 ? 2 : 3) * ((codes ? 64 : 32) * each * (dk + dv) + (codes ? 128 : 0)) + (codes ? 512 * nw : 0) + 64;      // (Wide::LDS)
  return 256 * min(8 / nw, 160 * 1024 / lds);      // two waves a SIMD
}

int launch_tree_wide(const TreeArgs& a, int dk, int dv, hipStream_t s) {
  const int nw = waves(a.max_draft * (a.H / a.G), dk, dv);
  const bool codes = a.ke != nullptr;
#define LM_CASE(K, V)                                                                               \
  if (dk == K && dv == V) {                                                                         \
    if (nw == 2) return codes ? launch<K, V, 2, true>(a, s) : launch<K, V, 2, false>(a, s);          \
    if (nw == 4) return codes ? launch<K, V, 4, true>(a, s) : launch<K, V, 4, false>(a, s);          \
    return codes ? launch<K, V, 8, true>(a, s) : launch<K, V, 8, false>(a, s);                       \
  }
  LM_CASE(64, 64) LM_CASE(64, 128) LM_CASE(64, 256) LM_CASE(128, 64) LM_CASE(128, 128) LM_CASE(128, 256)
  LM_CASE(256, 64) LM_CASE(256, 128) LM_CASE(256, 256)
#undef LM_CASE
  return LM_EINVAL;
}
#else
// f32, the format of verification, has the one kernel
bool tree_wide_takes(int, int, int) { return false; }
int tree_wide_rows(int, int, int) { return 1; }
int tree_wide_fit(int, int, int, bool) { return 1; }
int launch_tree_wide(const TreeArgs&, int, int, hipStream_t) { return LM_EINVAL; }
#endif

}  // namespace lm
