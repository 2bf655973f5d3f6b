// Attention of drafted tokens over a paged cache: every sequence brings a few tokens (one, a chain, a tree of guesses), each of which sees
// the cached context and, of the drafted tokens, those its mask names.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q . k_j - max),   j over the context's keys and the drafted ones that are seen
//
// The drafted tokens' query heads of one kv head are rows: R = tokens * heads per kv head, 16 of them a column block of the MFMA tiles.  A
// workgroup has NR blocks of rows of one sequence and kv head and a piece of their keys (lm_tree.h); its four waves take tiles of 64 keys (32 unless the
// cache holds codes) in turn, so that a key's codes are fetched and decoded once for all rows, and meet in LDS.  More than 32 rows (16 of heads of
// 256) go to lm_tree_wide.hip.
//
// Bound by the cache's bytes where there are enough of them: 61 tokens over 300 - 4000 keys of 8 heads of 128 71 us a call, 281 MB at 4.0 TB/s;
// one over 1501 keys 14.2 us, 4 of them the joining launch.  (Three waves a SIMD spill: 73 -> 114 us.  Eight waves a workgroup: 87.)
//
// Codes (lm_kv_codes.h).  A key's power of two scales its operand in the conversion.  A value's, 2^e, joins the softmax: with weights
// w_j = 2^(s_j + e_j - m'), m' the running maximum of s_j + e_j, the outputs are sum w_j code_j and the sum of the probabilities is
// sum w_j 2^(-e_j).  So w_j is at most 2^LAZY and is ONE f16 operand (11 bits, times 2^7 so that small ones stay normal) beside codes that f16
// holds exactly; bf16 values need two bf16 operands for theirs (16 bits).  A drafted token's values are divided by such a power of two of their own first, so
// that nothing depends on the size of values that a row does not see.  A tile with rows of values so much smaller than the others' (or none but zeros, 2^-100) that the maximum leaves
// such a weight nothing multiplies its roots with 2^(-e) one by one (Loudness): its rows count in the sum as all others do.
#include "lm_tree.h"
#include "omniserve_lm.h"

namespace lm {

// f32 of the codes' power-of-two exponents, and their reciprocals
__device__ __forceinline__ float exponent_of(uint32_t w, int i) { return (float)(w >> (8 * i) & 255) - 127.f; }
__device__ __forceinline__ float inverse_of(uint32_t w, int i) { return __uint_as_float((254 - (w >> (8 * i) & 255)) << 23); }

template <int DK, int DV, int NR, bool CODES>
struct Tree {
  static constexpr bool F16 = CODES && SPLIT;                     // weights of codes are one f16 operand
  static constexpr float SHIFT = F16 ? 7.f : CODES ? 0.f : ELEMS_SHIFT;      // an f16 weight is at most 2^(LAZY + 7)
  static constexpr int CH = DK / 64, PF = 16 / FR, NKF = CH * PF, NVB = DV / 16;
  static constexpr int KT = CODES ? 64 : 32, NU = KT / 16;        // keys of a context tile
  static constexpr int STAGE = 64 * DV;                           // bytes of a wave's V tile: 64 rows of codes, 32 of bf16
  static constexpr int NW = 4;                                    // waves
  static constexpr int EXPS = 256;                                // behind the V tiles, a wave's: exponents of 32 drafted values and 2^-exponent
  static constexpr int RED = NW * 16 * (DV + 4) * 4, LDS = SPLIT && NW * (STAGE + EXPS) > RED ? NW * (STAGE + EXPS) : RED;
  typedef Tile<SPLIT ? DV * 2 : 256> VT;

  const TreeArgs& p;
  uint8_t* stage;                   // this wave's part of the LDS
  float* exps;
  int lane, l15, l4;
  frag_t qf[NR][NKF];
  f32x4 acc[NR][NVB];
  float m_run[NR], l_run[NR];
  Loudness loud;
  int low[NR];                      // the newest position that the row does not see any more
  bool row_ok[NR];

  __device__ __forceinline__ Tree(const TreeArgs& a) : p(a) {}

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < NR; ++i) {
#pragma unroll
      for (int c = 0; c < NVB; ++c) acc[i][c] = zero4();
      m_run[i] = NEG;
      l_run[i] = 0.f;
    }
  }
  __device__ __forceinline__ bool finite() const {      // are all sums of this wave?
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int c = 0; c < NVB; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) z = __builtin_fmaf(acc[i][c][r], 0.f, z);
    return !__any(z != 0.f);
  }

  __device__ __forceinline__ void wave_sync() const {      // LDS operations of one wave are in order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // x: scores times scale plus the values' exponents, unseen ones NEG; inv: 2^-exponent (ONE: there are none), most: the largest of this lane's.  Leaves the weights
  // in x.
  template <int U, bool ONE>
  __device__ __forceinline__ void softmax(int i, f32x4 (&x)[U], const f32x4 (&inv)[U], float most) {
    float t = NEG;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) t = fmaxf(t, x[u][r]);
    t = rows_max(t);
    bool low = !ONE && loud.quiet(most);
    const bool grows = t > m_run[i] + (low ? 0.f : LAZY);      // (the first key's always; a NaN never)
    const bool some = __any(grows);
    const float m_new = grows ? t : m_run[i], m_sub = (m_new <= NEG ? 0.f : m_new) - SHIFT;
    if constexpr (!ONE)
      if (some) {
        float least = inv[0][0];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) least = fminf(least, inv[u][r]);
        loud.set(-rows_max(-least));
        low = loud.quiet(most);
      }
    float own = 0.f, sum = 0.f;
    if (!ONE && low) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float root = __builtin_amdgcn_exp2f(__builtin_fmaf(x[u][r], 0.5f, -0.5f * m_sub));
          own = __builtin_fmaf(root * inv[u][r], root, own);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[u][r] = __builtin_amdgcn_exp2f(x[u][r] - m_sub);
        sum = ONE ? sum + x[u][r] : __builtin_fmaf(x[u][r], inv[u][r], sum);
      }
    if (some) {
      const float root = root_of(m_run[i], m_new);
      l_run[i] = l_run[i] * root * root;
#pragma unroll
      for (int c = 0; c < NVB; ++c) acc[i][c] = acc[i][c] * root * root;
    }
    l_run[i] += low ? own : sum;
    m_run[i] = m_new;
  }

  // What non-finite values among keys lo .. hi - 1 of a tile add to the rows that see them.  (They were left out of the products, where a weight of
  // zero would have made them NaN in every row; a weight's size does not matter to them.)
  template <typename Seen, typename Value>
  __device__ __forceinline__ void add_nonfinite(int lo, int hi, Seen seen, Value value) {
#pragma unroll
    for (int i = 0; i < NR; ++i)
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
  }

  // ---- context tiles of codes ----
  struct Codes {
    u32x4 k[NU][CH], v[SPLIT ? DV / 16 : 1];
    uint32_t kx[NU], vx[NU];
    int64_t at;        // first row of the tile in the pools
  };

  __device__ __forceinline__ void load_codes(Codes& c, int page, int g) const {
    c.at = ((int64_t)min(max(page, 0), p.pages - 1) * p.G + g) * PAGE;
    const uint8_t* kp = p.kc + c.at * DK;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
#pragma unroll
      for (int j = 0; j < CH; ++j) c.k[u][j] = *(const u32x4*)(kp + (16 * u + l15) * DK + 64 * j + 16 * l4);
      c.kx[u] = p.ke[c.at + 16 * u + l15];
      c.vx[u] = *(const uint32_t*)(p.ve + c.at + 16 * u + 4 * l4);
    }
    if constexpr (SPLIT) {
      const uint8_t* vp = p.vc + c.at * DV;
#pragma unroll
      for (int i = 0; i < DV / 16; ++i) c.v[i] = *(const u32x4*)(vp + (64 * i + lane) * 16);
    }
  }

  // Scores of the tile's keys, and the next tile's request behind them; keys lo .. hi - 1 of the tile exist.
  template <typename Next>
  __device__ __forceinline__ void code_tile(Codes& c, int kb, int lo, int hi, bool edge, Next next) {
    f32x4 x[NR][NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
#pragma unroll
      for (int i = 0; i < NR; ++i) x[i][u] = zero4();
      const float scale = scale_of(c.kx[u]);
#pragma unroll
      for (int j = 0; j < CH; ++j)
#pragma unroll
        for (int h = 0; h < PF; ++h) {
          const frag_t kf = code_frag(c.k[u][j], h, scale);
#pragma unroll
          for (int i = 0; i < NR; ++i) x[i][u] = mma(kf, qf[i][j * PF + h], x[i][u]);
        }
    }
    const uint8_t* vp = p.vc + c.at * DV;
    bool bad = false;
    if (edge) {
      const int k4 = here(4 * l4);
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        uint32_t w = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = k4 + 16 * u + r;
          w |= (key >= lo && key < hi ? c.vx[u] >> (8 * r) & 255 : 127u) << (8 * r);
        }
        c.vx[u] = w;
      }
    }
    if constexpr (SPLIT) {
      if (edge) {
        const int first = here(lane / (DV / 16));
#pragma unroll
        for (int i = 0; i < DV / 16; ++i) {
          const int row = first + 64 * i / (DV / 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            c.v[i][e] = row >= lo && row < hi ? drop_nan_codes(c.v[i][e], bad) : 0u;
          }
        }
        bad = __any(bad);
      }
      __builtin_amdgcn_wave_barrier();       // the previous tile has been read
#pragma unroll
      for (int i = 0; i < DV / 16; ++i) {
        const int at = 64 * i + lane, row = at / (DV / 16), slot = at % (DV / 16);
        *(u32x4*)(stage + row * DV + ((slot ^ code_swizzle<DV>(row)) << 4)) = c.v[i];
      }
    }
    const int64_t page_at = c.at;
    uint32_t vx[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) vx[u] = c.vx[u];
    next();
    if constexpr (SPLIT) wave_sync();
    f32x4 ev[NU], inv[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) { ev[u][r] = exponent_of(vx[u], r); inv[u][r] = inverse_of(vx[u], r); }
    float most = inv[0][0];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) most = fmaxf(most, inv[u][r]);
    f16x4 pq[NR][NU];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[i][u][r] = __builtin_fmaf(x[i][u][r], p.scale, ev[u][r]);
      if (edge) {
        const int k4 = here(4 * l4);
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = k4 + 16 * u + r;
            x[i][u][r] = (int)(key >= lo) & (int)(key < hi) & (int)(kb + key > low[i]) ? x[i][u][r] : NEG;
          }
      }
      softmax<NU, false>(i, x[i], inv, most);
      if constexpr (SPLIT) {
#pragma unroll
        for (int u = 0; u < NU; ++u) pq[i][u] = (f16x4){(_Float16)x[i][u][0], (_Float16)x[i][u][1], (_Float16)x[i][u][2], (_Float16)x[i][u][3]};
      }
    }
    if constexpr (SPLIT) {
      const int base = code_column<DV>(l15, l4);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int cb = 0; cb < NVB; ++cb) {
          const f16x8 vf = code_halves(read_code_column<DV>(stage, base, h, cb));
#pragma unroll
          for (int i = 0; i < NR; ++i)
            acc[i][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, __builtin_shufflevector(pq[i][2 * h], pq[i][2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7), acc[i][cb], 0, 0, 0);
        }
    } else {
#pragma unroll
      for (int h = 0; h < NU / 2; ++h)
#pragma unroll
        for (int cb = 0; cb < NVB; ++cb) {
          quad_t v[2];
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int key = 32 * h + 16 * s + 4 * l4 + r;
              float y = decode4(vp[key * DV + 16 * cb + l15], 1.0f)[0];
              if (edge) {
                y = key >= lo && key < hi ? y : 0.f;
                bad |= y != y;
                y = y != y ? 0.f : y;
              }
              v[s][r] = (elem_t)y;
            }
#pragma unroll
          for (int i = 0; i < NR; ++i) acc[i][cb] = mma_quads(v[0], v[1], to_quad(x[i][2 * h]), to_quad(x[i][2 * h + 1]), acc[i][cb]);
        }
      bad = __any(bad);
    }
    if (bad) {
      const uint8_t* vb = p.vc + page_at * DV;
      add_nonfinite(lo, min(hi, KT), [&](int i, int j) { return kb + j > low[i]; }, [&](int j, int d) { return (vb[j * DV + d] & 127) == 127 ? __builtin_nanf("") : 0.f; });
    }
  }

  // ---- 32 keys and values in elements: drafted ones, or a part of a page ----
  struct Elems {
    frag_t k[2][NKF], v[SPLIT ? DV / 16 : 1];
    const elem_t* kp; const elem_t* vp;
    int64_t ldk, ldv;
    int rows;        // that exist
  };

  __device__ __forceinline__ void load_elems(Elems& c, const elem_t* kp, int64_t ldk, const elem_t* vp, int64_t ldv, int rows) const {
    c.kp = kp; c.vp = vp; c.ldk = ldk; c.ldv = ldv; c.rows = rows;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const elem_t* row = kp + min(16 * u + l15, rows - 1) * ldk;
#pragma unroll
      for (int j = 0; j < CH; ++j)
#pragma unroll
        for (int h = 0; h < PF; ++h) c.k[u][j * PF + h] = *(const frag_t*)(row + 64 * j + 16 * l4 + FR * h);
    }
    if constexpr (SPLIT) {
#pragma unroll
      for (int i = 0; i < DV / 16; ++i) {
        const int at = 64 * i + lane, row = at / (DV / 8), col = at % (DV / 8);
        c.v[i] = *(const frag_t*)(vp + min(row, rows - 1) * ldv + 8 * col);
      }
    }
  }

  // seen(i, key): does row block i's row of this lane see key (of 32)?  lo .. hi - 1: keys that any row may see
  template <typename Next, typename Seen>
  __device__ __forceinline__ void elem_tile(Elems& c, int lo, int hi, bool edge, Seen seen, Next next) {
    f32x4 x[NR][2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        x[i][u] = zero4();
#pragma unroll
        for (int s = 0; s < NKF; ++s) x[i][u] = mma(c.k[u][s], qf[i][s], x[i][u]);
      }
    bool bad = false;
    const elem_t* vp = c.vp;
    const int64_t ldv = c.ldv;
    f32x4 ev[2], inv[2];      // of this lane's keys, as those of codes
    if constexpr (SPLIT) {
      __builtin_amdgcn_wave_barrier();       // the previous tile has been read
      if (edge) {
#pragma unroll
        for (int i = 0; i < DV / 16; ++i) {
          const int at = 64 * i + lane, row = at / (DV / 8);
          int e = 0;
          if (64 * i / (DV / 8) >= hi) {      // (a step without drafts has one row)
            c.v[i] = frag_t{};
          } else {
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              float y = row >= lo && row < hi ? (float)c.v[i][k] : 0.f;
              const bool fine = fabsf(y) < __builtin_inff();
              bad |= !fine;
              y = fine ? y : 0.f;
              top = fmaxf(top, fabsf(y));
              c.v[i][k] = (elem_t)y;
            }
            if constexpr (CODES) {
              e = row >= lo && row < hi ? row_exponent(lanes_max<DV / 8>(top)) : 0;
              const float f = pow2(-e);
#pragma unroll
              for (int k = 0; k < 8; ++k) c.v[i][k] = (elem_t)((float)c.v[i][k] * f);
            }
          }
          if constexpr (CODES)
            if (at % VT::NS == 0) {
              exps[row] = (float)e;
              exps[32 + row] = pow2(-e);
            }
        }
        bad = __any(bad);
      }
#pragma unroll
      for (int i = 0; i < DV / 16; ++i) {
        const int at = 64 * i + lane;
        *(frag_t*)(stage + VT::slot(at / VT::NS, at % VT::NS)) = c.v[i];
      }
    } else if constexpr (CODES) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = 16 * s + 4 * l4 + r;
          float top = 0.f;
#pragma unroll
          for (int cb = 0; cb < NVB; ++cb) {
            const float m = fabsf((float)vp[min(key, c.rows - 1) * ldv + 16 * cb + l15]);
            top = m < __builtin_inff() ? fmaxf(top, m) : top;
          }
          const int e = key >= lo && key < hi ? row_exponent(lanes_max<16>(top)) : 0;
          ev[s][r] = (float)e;
          inv[s][r] = pow2(-e);
        }
    }
    next();
    if constexpr (SPLIT) wave_sync();
    if constexpr (SPLIT && CODES) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        ev[u] = *(const f32x4*)&exps[16 * u + 4 * l4];
        inv[u] = *(const f32x4*)&exps[32 + 16 * u + 4 * l4];
      }
    }
    float most = 0.f;
    if constexpr (CODES) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) most = fmaxf(most, inv[u][r]);
    }
    quad_t pq[NR][2][NOPND];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[i][u][r] = CODES ? __builtin_fmaf(x[i][u][r], p.scale, ev[u][r]) : x[i][u][r] * p.scale;
      if (edge) {
        const int key = here(4 * l4);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) x[i][u][r] = seen(i, key + 16 * u + r) ? x[i][u][r] : NEG;
      }
      softmax<2, !CODES>(i, x[i], inv, most);
#pragma unroll
      for (int u = 0; u < 2; ++u) split_quad(x[i][u], pq[i][u]);
    }
#pragma unroll
    for (int cb = 0; cb < NVB; ++cb) {
      quad_t v[2];
      if constexpr (SPLIT) {
        v[0] = VT::column_quad(stage, 0, cb, l15, l4);
        v[1] = VT::column_quad(stage, 16, cb, l15, l4);
      } else {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = 16 * s + 4 * l4 + r;
            float y = (float)vp[min(key, c.rows - 1) * ldv + 16 * cb + l15];
            if (edge) {
              y = key >= lo && key < hi ? y : 0.f;
              const bool fine = fabsf(y) < __builtin_inff();
              bad |= !fine;
              y = fine ? y : 0.f;
              if constexpr (CODES) y *= inv[s][r];
            }
            v[s][r] = (elem_t)y;
          }
      }
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int m = 0; m < NOPND; ++m) acc[i][cb] = mma_quads(v[0], v[1], pq[i][0][m], pq[i][1][m], acc[i][cb]);
    }
    if constexpr (!SPLIT) bad = __any(bad);
    if (bad) add_nonfinite(lo, min(hi, 32), seen, [&](int j, int d) { return (float)vp[j * ldv + d]; });
  }
};

template <int DK, int DV, int NR, bool CODES>
__global__ __launch_bounds__(256, NR == 1 && DK + DV <= 256 ? 2 : 1) void tree_attn_kernel(TreeArgs p) {
  typedef Tree<DK, DV, NR, CODES> T;
  __shared__ __attribute__((aligned(16))) uint8_t lds[T::LDS];
  constexpr int NW = T::NW;
  __shared__ float wm[NW][16], wl[NW][16];
  Piece s;
  int64_t part = 0;
  if (!piece_of<T::KT, 16 * NR>(p, s, part)) return;
  const int g = s.g, f0 = s.f0, drafted = s.drafted, gs = s.gs, R = s.R, r0 = s.rb * 16 * NR, length = s.length;
  const __attribute__((address_space(4))) int* bt = (const __attribute__((address_space(4))) int*)(uintptr_t)s.bt;      // (scalar loads)

  T t(p);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  t.lane = tid & 63; t.l15 = tid & 15; t.l4 = t.lane >> 4;
  t.stage = lds + wave * (SPLIT ? T::STAGE : 0);
  t.exps = (float*)(lds + T::NW * T::STAGE + wave * T::EXPS);      // (SPLIT alone uses it)
  int low_min = INT32_MAX, low_max = INT32_MIN, token[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = r0 + 16 * i + t.l15, rc = min(r, R - 1), tk = rc / gs;
    token[i] = f0 + tk;
    t.row_ok[i] = r < R;
    const int lo = bound_of(p, p.pos[token[i]]);
    low_min = min(low_min, lo);
    low_max = max(low_max, lo);
    t.low[i] = r < R ? lo : INT32_MAX;
    const elem_t* q = p.q + (int64_t)token[i] * p.ldq + (int64_t)(g * gs + rc - tk * gs) * DK;
#pragma unroll
    for (int j = 0; j < T::CH; ++j)
#pragma unroll
      for (int h = 0; h < T::PF; ++h) t.qf[i][j * T::PF + h] = r < R ? *(const frag_t*)(q + 64 * j + 16 * t.l4 + FR * h) : frag_t{};
  }
  t.clear();
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) {
    low_min = min(low_min, __shfl_xor(low_min, m, 64));
    low_max = max(low_max, __shfl_xor(low_max, m, 64));
  }
  low_min = __builtin_amdgcn_readfirstlane(low_min);
  low_max = __builtin_amdgcn_readfirstlane(low_max);

  // ---- the context ----
  const int k0 = max(low_min, -1) + 1, ta = s.t0 + min(s.from, s.nt), tb = s.t0 + min(s.to, s.nt);
  constexpr int PER_PAGE = PAGE / T::KT;
  int tile = ta + wave;
  if (tile < tb) {
    int page = bt[tile / PER_PAGE];
    if constexpr (CODES) {
      typename T::Codes c;
      t.load_codes(c, page, g);
      int ahead = tile + NW < tb ? bt[tile + NW] : 0;
      for (; tile < tb; tile += NW) {
        const int kb = tile * T::KT, hi = (uint32_t)page < (uint32_t)p.pages ? length - kb : 0;
        const bool edge = hi < T::KT || kb <= low_max;
        page = ahead;
        t.code_tile(c, kb, max(k0 - kb, 0), hi, edge, [&]() {
          if (tile + NW >= tb) return;
          t.load_codes(c, page, g);
          ahead = tile + 2 * NW < tb ? bt[tile + 2 * NW] : 0;
        });
      }
    } else {
      typename T::Elems c;
      const elem_t* kc = (const elem_t*)p.kc;
      const elem_t* vc = (const elem_t*)p.vc;
      auto load = [&](int tl, int pg) {
        const int64_t at = ((int64_t)min(max(pg, 0), p.pages - 1) * p.G + g) * PAGE + tl * T::KT % PAGE;
        t.load_elems(c, kc + at * DK, DK, vc + at * DV, DV, T::KT);
      };
      int ahead;
      auto begin = [&]() {
        tile = ta + wave;
        page = bt[tile / PER_PAGE];
        load(tile, page);
        ahead = tile + NW < tb ? bt[(tile + NW) / PER_PAGE] : 0;
      };
      begin();
      // An infinite value in a tile that all rows see whole passes through the products, where the second half of a weight, or a weight of zero, makes it NaN.  A
      // wave whose sums are not finite goes over its tiles once more with such values taken out, as those of partly seen tiles always are.
      for (bool careful = false; tile < tb;) {
        const int kb = tile * T::KT, hi = (uint32_t)page < (uint32_t)p.pages ? length - kb : 0, lo = max(k0 - kb, 0);
        const bool edge = careful || hi < T::KT || kb <= low_max;
        page = ahead;
        t.elem_tile(c, lo, hi, edge, [&](int i, int key) { return (bool)((int)(key >= lo) & (int)(key < hi) & (int)(kb + key > t.low[i])); },
                    [&]() {
                      if (tile + NW >= tb) return;
                      load(tile + NW, page);
                      ahead = tile + 2 * NW < tb ? bt[(tile + 2 * NW) / PER_PAGE] : 0;
                    });
        tile += NW;
        if (tile >= tb && !careful && !t.finite()) {
          careful = true;
          t.clear();
          begin();
        }
      }
    }
  }
  // ---- the drafted tokens: waves that had a tile less come first ----
  if (s.to > s.nt) {
    for (int j0 = 32 * (max(s.from - s.nt, 0) + ((wave - (tb - ta)) & (NW - 1))); j0 < min(drafted, 32 * (s.to - s.nt)); j0 += 32 * NW) {
      typename T::Elems c;
      const int64_t row = f0 + j0;
      t.load_elems(c, p.k + row * p.ldk + (int64_t)g * DK, p.ldk, p.v + row * p.ldv + (int64_t)g * DV, p.ldv, min(drafted - j0, 32));
      uint32_t bits[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i)
        bits[i] = t.row_ok[i] && (j0 >> 6) < p.words ? (uint32_t)(p.mask[(int64_t)token[i] * p.words + (j0 >> 6)] >> (j0 & 63)) : 0u;
      const int hi = min(drafted - j0, 32);
      t.elem_tile(c, 0, hi, true,
                  [&](int i, int key) {
                    return (bool)((int)(key < hi) & (int)(bits[i] >> key & 1) & (int)(p.pos[min((int)row + key, f0 + drafted - 1)] > t.low[i]));
                  },
                  []() {});
    }
  }

  // ---- the waves' results ----
  float(*res)[16][DV + 4] = (float(*)[16][DV + 4])lds;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const float l = column_sum(t.l_run[i]);
    __syncthreads();      // V tiles, or the block before, have been read
#pragma unroll
    for (int c = 0; c < T::NVB; ++c) *(f32x4*)&res[wave][t.l15][16 * c + 4 * t.l4] = t.acc[i][c];
    if (t.l4 == 0) { wm[wave][t.l15] = t.m_run[i]; wl[wave][t.l15] = l; }
    __syncthreads();
    const int rows = min(16, R - r0 - 16 * i);
    for (int at = tid; at < rows * (DV / 4); at += 64 * NW) {
      const int rr = at / (DV / 4), d = (at - rr * (DV / 4)) * 4, r = r0 + 16 * i + rr, tk = r / gs, h = g * gs + r - tk * gs;
      float m = wm[0][rr];
#pragma unroll
      for (int w = 1; w < NW; ++w) m = fmaxf(m, wm[w][rr]);
      f32x4 y = zero4();
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float root = wl[w][rr] != 0.f ? root_of(wm[w][rr], m) : 0.f;
        sum += wl[w][rr] * root * root;
        y += *(const f32x4*)&res[w][rr][d] * root * root;
      }
      if (!s.whole) {
        const int64_t at = part + 16 * i + rr;
        *(f32x4*)(p.part + at * DV + d) = y;
        if (d == 0) { p.ml[2 * at] = m; p.ml[2 * at + 1] = sum; }
      } else {
        y *= sum != 0.f ? 1.0f / sum : 0.f;
        *(quad_t*)(p.o + (int64_t)(f0 + tk) * p.ldo + (int64_t)h * DV + d) = to_quad(y);
      }
    }
  }
}

// Joins the pieces of a segment's rows.  A lane has four columns, so that a wave has four, two or one rows (of 64, 128, 256), each with pieces of its own to
// add up, or (few rows, whose pieces are many) the four waves of a workgroup the same rows and a quarter of the pieces each.  Lane l of a row holds the maximum
// and sum of every l-th piece.
template <int DV>
constexpr int rows_of_wave() { return 256 / DV; }
template <int ROWS, int DV>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs p, int rows, int waves) {
  constexpr int RW = rows_of_wave<DV>(), LR = 64 / RW;      // rows of a wave, lanes of a row
  __shared__ f32x4 res[3][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane % LR, each = 4 / waves * RW, per = (rows + each - 1) / each;
  const int seg = blockIdx.x / per, rr = (blockIdx.x - seg * per) * each + (waves == 1 ? wave * RW : 0) + lane / LR, w = waves == 1 ? 0 : wave;
  const int rb = seg % p.blocks, g = seg / p.blocks % p.G, b = seg / p.blocks / p.G, gs = p.H / p.G, r = rb * ROWS + rr;
  const int f0 = min(max(p.first[b], 0), p.n), drafted = min(max(p.first[b + 1] - f0, 0), min(p.max_draft, p.n - f0));
  if (rb * ROWS >= drafted * gs) return;      // (such a segment is none, and nothing says how it is cut)
  const int parts = p.cuts[2 * seg + 1];
  if (parts == 1) return;                     // written by its piece
  const bool mine = rr < ROWS && r < drafted * gs;
  const int64_t at0 = (int64_t)p.cuts[2 * seg] * ROWS + min(rr, ROWS - 1), step = (int64_t)((drafted * gs + ROWS - 1) / ROWS) * ROWS;
  float m = NEG;
  for (int s = l; s < parts; s += LR) m = fmaxf(m, p.ml[2 * (at0 + s * step)]);
#pragma unroll
  for (int k = LR / 2; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor(m, k, 64));
  float sum = 0.f;
  f32x4 y = zero4();
  for (int s0 = 0; s0 < parts; s0 += LR) {
    f32x4 v[8];
    auto load = [&](int s1) {
#pragma unroll
      for (int s = 0; s < 8; ++s) {      // (those behind a row's lanes come with the next pass; here they would count as zero times theirs, NaN of an infinity)
        const int at = s1 + s * waves;
        v[s] = at < min(LR, parts - s0) ? *(const f32x4*)(p.part + (at0 + (s0 + at) * step) * DV + 4 * l) : zero4();
      }
    };
    load(w);      // (beside the sums' request)
    const bool in = s0 + l < parts;
    const float ms = in ? p.ml[2 * (at0 + (s0 + l) * step)] : NEG, ls = in ? p.ml[2 * (at0 + (s0 + l) * step) + 1] : 0.f;
    const float root = ls != 0.f ? root_of(ms, m) : 0.f;
    float t = ls * root * root;
#pragma unroll
    for (int k = LR / 2; k > 0; k >>= 1) t += __shfl_xor(t, k, 64);
    sum += t;
    const int end = min(LR, parts - s0);
    for (int s1 = w; s1 < end; s1 += 8 * waves) {
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const float f = s1 + s * waves < LR ? __shfl(root, lane - l + (s1 + s * waves) % LR, 64) : 0.f;
        y += v[s] * f * f;
      }
      if (s1 + 8 * waves < end) load(s1 + 8 * waves);
    }
  }
  if (waves > 1) {      // (uniform over the workgroup, as are the returns above)
    if (w > 0) res[w - 1][lane] = y;
    __syncthreads();
    if (w > 0) return;
    y += res[0][lane] + res[1][lane] + res[2][lane];
  }
  if (!mine) return;
  y *= sum != 0.f ? 1.0f / sum : 0.f;
  const int tk = f0 + r / gs, h = g * gs + r % gs;
  *(quad_t*)(p.o + (int64_t)tk * p.ldo + (int64_t)h * DV + 4 * l) = to_quad(y);
}

// Blocks of 16 rows of a workgroup
static int row_blocks(int rows) { return rows <= 16 || !SPLIT ? 1 : 2; }

template <int DK, int DV, bool CODES>
static int launch_tree(const TreeArgs& a, int nr, hipStream_t s) {
  const dim3 grid((a.workgroups + 7) / 8 * 8);
  if (nr == 1) hipLaunchKernelGGL((tree_attn_kernel<DK, DV, 1, CODES>), grid, dim3(256), 0, s, a);
  if constexpr (SPLIT && DK <= 128 && DV <= 128)
    if (nr == 2) hipLaunchKernelGGL((tree_attn_kernel<DK, DV, 2, CODES>), grid, dim3(256), 0, s, a);
  return launch_status();
}

template <int ROWS>
static void launch_merge(const TreeArgs& a, int dv, hipStream_t s) {
  const int rows = min(ROWS, a.max_draft * (a.H / a.G));      // of a segment, at most
  const int64_t segments = (int64_t)a.B * a.G * a.blocks;
  const int waves = segments * rows <= 512 ? 4 : 1, each = 4 / waves * (256 / dv);
  const dim3 grid((unsigned)(segments * ((rows + each - 1) / each)));
  if (dv == 64) hipLaunchKernelGGL((tree_merge_kernel<ROWS, 64>), grid, dim3(256), 0, s, a, rows, waves);
  else if (dv == 128) hipLaunchKernelGGL((tree_merge_kernel<ROWS, 128>), grid, dim3(256), 0, s, a, rows, waves);
  else hipLaunchKernelGGL((tree_merge_kernel<ROWS, 256>), grid, dim3(256), 0, s, a, rows, waves);
}

struct Plan {
  bool wide, cut;
  int each;                   // rows of a workgroup
  int64_t run, blocks, workgroups, target, scratch;
};
// Cut where the segments are fewer than four rounds of workgroups and the longest has more tiles than joining is worth: 20 of the narrow kernel, 8 of the wide
// one (one token, 1501 keys of 8 heads in one piece each 14.9 us, in pieces of 4 tiles 14.4; 16 of 1024 keys 13.6 and 19.3; a tree of 26, 500 keys, in one
// piece 25.7, in pieces of 3 tiles 20.8).  Into as many pieces as workgroups fit the chip, or twice as many where the segments alone are half of that (61 tokens of
// 300 - 4000 keys: 74 us and 70; the wide kernel, whose pieces have more sums to write, not: 4 trees of 64 over 32768 keys 240 instead of 212, a tree of 26 for each
// of 16 sequences 58 instead of 47).
static Plan plan_of(int B, int max_draft, int max_context, int H, int G, int dk, int dv, bool codes) {
  Plan q{};
  const int rows = max_draft * (H / G), kt = codes ? 64 : 32;
  q.wide = tree_wide_takes(rows, dk, dv);
  q.each = q.wide ? tree_wide_rows(rows, dk, dv) : 16 * row_blocks(rows);
  q.blocks = (rows + q.each - 1) / q.each;
  const int64_t segments = (int64_t)B * G * q.blocks, tiles = max_context / kt + (max_context % kt > 0) + (max_draft + 31) / 32;
  const int64_t fit = q.wide ? tree_wide_fit(rows, dk, dv, codes) : q.each == 16 && dk + dv <= 256 ? 512 : 256;
  q.run = q.wide ? 3 : 4;
  q.cut = tiles > (q.wide ? 8 : 20) && segments < 4 * fit;
  q.target = min(segments > fit / 2 ? 2 * fit : fit, (segments * tiles + q.run - 1) / q.run);
  q.workgroups = q.cut ? segments + q.target : segments;
  q.scratch = q.cut ? q.workgroups * q.each * (dv + 2) + 2 * segments : 0;
  return q;
}

}  // namespace lm

using namespace lm;

// (an exponent of 127 over the scale is far above NEG, and a score times the scale finite)
static constexpr float MIN_SCALE = 0x1p-60f;

extern "C" int64_t lm_tree_attn_scratch(int B, int max_draft, int max_context, int H, int G, int dk, int dv, int codes) {
  if (B <= 0 || G <= 0 || H <= 0 || H % G || max_draft <= 0 || max_context < 0 || (int64_t)max_draft * H > 1 << 24) return 0;
  return plan_of(B, max_draft, max_context, H, G, dk, dv, codes != 0).scratch;
}

extern "C" int lm_tree_attn(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, const void* kc, const void* vc, const uint8_t* ke,
                            const uint8_t* ve, int64_t pages, const int* bt, int bt_stride, int bt_width, const int* length, const int* first, const int* pos,
                            const int64_t* mask, int words, void* o, int64_t ldo, float* part, float scale, int window, int B, int n, int max_draft,
                            int max_context, int H, int G, int dk, int dv, void* stream) {
  if (B < 0 || n < 0 || max_draft < 0 || G <= 0 || H <= 0 || H % G || !(scale >= MIN_SCALE && scale <= 1.0f / MIN_SCALE) || window <= 0 || words < 0 || bt_width < 0 || bt_stride < bt_width ||
      bt_width > INT32_MAX / PAGE || pages < 0 || pages > INT32_MAX / PAGE || (bt_width > 0 && pages == 0) || max_context < 0 || (ke == nullptr) != (ve == nullptr) || ldq % FR || ldk % FR || ldv % FR || ldo % 4 || (int64_t)max_draft * H > 1 << 24 ||
      // (tiles are counted in 32 bits)
      (int64_t)B * G * (max_draft * (H / G) / 16 + 1) * (2 * (int64_t)bt_width + max_draft / 32 + 2) > INT32_MAX)
    return LM_EINVAL;
  if (B == 0 || n == 0 || max_draft == 0) return LM_OK;
  if (!q || !k || !v || !length || !first || !pos || !mask || !o || (bt_width > 0 && (!bt || !kc || !vc)) ||
      ((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)ke | (uintptr_t)ve | (uintptr_t)part) % 16 || (uintptr_t)o % 8)
    return LM_EINVAL;
  TreeArgs a{};
  a.q = (const elem_t*)q; a.ldq = ldq; a.k = (const elem_t*)k; a.ldk = ldk; a.v = (const elem_t*)v; a.ldv = ldv;
  a.kc = (const uint8_t*)kc; a.vc = (const uint8_t*)vc; a.ke = ke; a.ve = ve; a.pages = (int)pages;
  a.bt = bt; a.bt_stride = bt_stride; a.bt_width = bt_width; a.length = length; a.first = first; a.pos = pos;
  a.mask = (const unsigned long long*)mask; a.words = words; a.o = (elem_t*)o; a.ldo = ldo;
  a.scale = scale * LOG2E; a.window = window; a.n = n; a.H = H; a.G = G; a.B = B; a.max_draft = max_draft;
  Plan plan = plan_of(B, max_draft, max_context, H, G, dk, dv, ke != nullptr);
  if (!part && plan.cut) { plan.cut = false; plan.workgroups = (int64_t)B * G * plan.blocks; }
  a.blocks = (int)plan.blocks;
  a.workgroups = (int)plan.workgroups;
  a.target = (int)plan.target;
  a.run = (int)plan.run;
  if (plan.cut) { a.part = part; a.ml = part + plan.workgroups * plan.each * dv; a.cuts = (int*)(a.ml + plan.workgroups * plan.each * 2); }
  hipStream_t s = (hipStream_t)stream;
  int rc = LM_EINVAL;
  if (plan.wide) rc = launch_tree_wide(a, dk, dv, s);
#define LM_CASE(K, V) else if (dk == K && dv == V) rc = ke ? launch_tree<K, V, true>(a, plan.each / 16, s) : launch_tree<K, V, false>(a, plan.each / 16, s);
  LM_CASE(64, 64) LM_CASE(64, 128) LM_CASE(64, 256) LM_CASE(128, 64) LM_CASE(128, 128) LM_CASE(128, 256)
  LM_CASE(256, 64) LM_CASE(256, 128) LM_CASE(256, 256)
#undef LM_CASE
  if (rc != LM_OK) return rc;
  if (plan.cut) {
#define LM_CASE(ROWS) if (plan.each == ROWS) launch_merge<ROWS>(a, dv, s);
    LM_CASE(16) LM_CASE(32) LM_CASE(64) LM_CASE(128) LM_CASE(256)
#undef LM_CASE
  }
  return launch_status();
}
