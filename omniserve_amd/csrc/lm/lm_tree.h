// What the two kernels of drafted tokens' attention share (lm_tree_attn.hip: few rows, lm_tree_wide.hip: many).
#pragma once
#include "lm_attn.h"
#include <initializer_list>
#include "lm_kv_codes.h"

namespace lm {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

struct TreeArgs {
  const elem_t* q; int64_t ldq;                      // [n][H][dk]
  const elem_t* k; int64_t ldk;                      // drafted keys [n][G][dk]
  const elem_t* v; int64_t ldv;
  const uint8_t* kc; const uint8_t* vc;              // pools: codes, or elements
  const uint8_t* ke; const uint8_t* ve;
  int pages;
  const int* bt; int bt_stride, bt_width;
  const int* length; const int* first; const int* pos;
  const unsigned long long* mask; int words;
  elem_t* o; int64_t ldo;
  float* ml; float* part;                            // of cut pieces: [workgroups][rows][2] and [workgroups][rows][dv]; null: nothing is cut
  int* cuts;                                         // [B * G * blocks][2]: a segment's first piece and how many it has
  float scale;                                       // includes log2(e)
  int window;                                        // NO_WINDOW: none
  int n, H, G, B, max_draft, blocks, workgroups;     // blocks: of rows, the most a sequence has
  int target, run;                                   // pieces that there should be; tiles of one at least
};
constexpr int NO_WINDOW = INT32_MAX;

// The newest position that a token does not see any more
__device__ __forceinline__ int bound_of(const TreeArgs& p, int pos) { return p.window == NO_WINDOW ? INT32_MIN : max(pos, INT32_MIN + p.window) - p.window; }

// A row's weights are relative to a maximum that is followed only when it has grown by so much (in powers of two): what has been added up is rescaled in a
// few tiles, not in every second one
constexpr float LAZY = 8.f;
// The largest weight over elements is 2^(LAZY + ELEMS_SHIFT): a sum of 2^24 values near the largest of their type stays finite
constexpr float ELEMS_SHIFT = -32.f;
// A weight is 2^(s + e - m'), and a probability it times 2^-e, so that a weight may be too small for 32 bits whose probability is not: where a tile has exponents
// SPREAD below that of the keys which have set the maximum, or below LOWEST (the sum of many probabilities, each 2^-e times a weight, could pass 32
// bits), the weights' roots are multiplied with 2^-e one by one.  What is lost otherwise is below 2^-30 of the largest probability.
constexpr int LOWEST = -63, SPREAD = 96;

// The root of the factor by which what has been added up is brought from maximum m to m_new.  It is multiplied with twice: a sum of 2^100 (of values of zero) may
// count where the whole factor is zero in 32 bits, and an infinite value that a row sees counts whatever its weight is (zero times it would be NaN; what is
// finite is below 2^-124 after two times the least)
__device__ __forceinline__ float root_of(float m, float m_new) { return fmaxf(__builtin_amdgcn_exp2f(0.5f * (m - m_new)), 0x1p-126f); }

// Which tiles those are, of one wave.  Exponents are looked at as the bits of 2^-e, in scalar registers.
struct Loudness {
  static constexpr uint32_t FROM = (uint32_t)(127 - LOWEST) << 23;
  uint32_t loudest = ~0u, limit = FROM;      // of the keys that have set a maximum; of the tiles that go without roots
  __device__ __forceinline__ bool quiet(float most) const { return __any(__float_as_uint(most) > limit); }      // most: the largest of this lane's
  // a tile sets a row's maximum; least: the smallest of all its keys'
  __device__ __forceinline__ void set(float least) {
    loudest = min(loudest, (uint32_t)__builtin_amdgcn_readfirstlane(__float_as_uint(least)));
    limit = min(FROM, loudest + ((uint32_t)SPREAD << 23));
  }
};

// Largest of the four lanes that share l15, by lane swaps (column_max goes through LDS: two latencies in every tile's chain)
__device__ __forceinline__ float rows_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
template <int C>
struct Dpp { static constexpr int value = C; };
// Largest of N neighbouring lanes, 8 to 32 (lane swaps inside a row of 16, then of two rows)
template <int N>
__device__ __forceinline__ float lanes_max(float v) {
  auto with = [&](auto ctrl) { v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, false))); };
  with(Dpp<0xb1>());       // lane ^ 1
  with(Dpp<0x4e>());       // lane ^ 2
  with(Dpp<0x141>());      // the other four of eight
  if constexpr (N > 8) with(Dpp<0x140>());
  if constexpr (N > 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  return v;
}
// x in a place that few tiles come to: nothing formed from it moves in front of the branch
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// The 16-byte slot of a row of dv codes in LDS, so that the eight rows of both 16-lane groups of a transposed read lie in different banks.
template <int DV>
__device__ __forceinline__ int code_swizzle(int row) {
  if constexpr (DV == 64) return ((row >> 2) & 1) | ((row >> 4) & 1) << 1;
  if constexpr (DV == 128) return ((row >> 1) & 3) | ((row >> 4) & 1) << 2;
  return (row & 7) | ((row >> 4) & 1) << 3;
}

// Eight keys' codes of one column, keys 4 l4 + (0..3) and 16 + 4 l4 + (0..3) of a tile of rows of DV codes; base: code_column(..), h: which 32 keys
template <int DV>
__device__ __forceinline__ int code_column(int l15, int l4) {
  const int i = l15 >> 1, row = i < 4 ? 4 * l4 + i : 12 + 4 * l4 + i;
  return row * DV + (code_swizzle<DV>(row) << 4) + 8 * (l15 & 1);
}
template <int DV>
__device__ __forceinline__ u32x2 read_code_column(const uint8_t* tile, int base, int h, int cb) {
  typedef int tr2 __attribute__((__vector_size__(8)));
  const tr2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
      (__attribute__((address_space(3))) tr2*)(__attribute__((address_space(3))) void*)(tile + (base ^ (cb << 4)) + h * 32 * DV));
  return (u32x2){(uint32_t)w[0], (uint32_t)w[1]};
}

__device__ __forceinline__ f16x8 code_halves(u32x2 w) {
  f16x8 f;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[m], 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[m], 1.0f, true);
    f[4 * m] = a[0]; f[4 * m + 1] = a[1]; f[4 * m + 2] = b[0]; f[4 * m + 3] = b[1];
  }
  return f;
}

// Half h of 16 codes times a power of two, as an operand
__device__ __forceinline__ frag_t code_frag(const u32x4& w, int h, float scale) {
  frag_t f;
#pragma unroll
  for (int m = 0; m < FR / 4; ++m) {
    const quad_t z = decode4(w[h * (FR / 4) + m], scale);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[4 * m + e] = z[e];
  }
  return f;
}

// w without its NaN codes (seven low bits ones); bad: there was one
__device__ __forceinline__ uint32_t drop_nan_codes(uint32_t w, bool& bad) {
  const uint32_t nan = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  bad |= nan != 0;
  return w & ~(nan - (nan >> 7) | nan);
}

// ---- how the work is dealt out ----
// A segment is the keys of one (sequence, kv head, block of rows): its context tiles that any row sees and, behind them, tiles of 32 drafted tokens.
// Where segments are few or of different lengths they are cut into equal pieces of at most run_length() tiles, a workgroup each.  The length follows from
// the tiles of all of them, so that there are as many pieces as suit the chip whatever the sequences' lengths are (a fixed number of parts a sequence
// leaves the short ones' places idle: 16 trees of 26 over 500 - 4000 keys took 65 us where pieces of one length took 58, when the pieces themselves were slower than now).  A segment of one piece is written by it, others are joined by tree_merge_kernel.  The division depends on the
// lengths alone.

struct Segments {            // of one sequence
  int f0, drafted, length, t0, nt, nd, blocks;
  __device__ __forceinline__ int tiles() const { return nt + nd; }
};
template <int KT, int ROWS>
__device__ __forceinline__ Segments segments_of(const TreeArgs& p, int b) {
  Segments q;
  q.f0 = min(max(p.first[b], 0), p.n);
  q.drafted = min(max(p.first[b + 1] - q.f0, 0), min(p.max_draft, p.n - q.f0));
  q.length = min(max(p.length[b], 0), p.bt_width * PAGE);
  q.blocks = (q.drafted * (p.H / p.G) + ROWS - 1) / ROWS;
  int low = INT32_MIN;
  if (p.window != NO_WINDOW && q.drafted > 0) {
    low = INT32_MAX;
    for (int i = 0; i < q.drafted; ++i) low = min(low, bound_of(p, p.pos[q.f0 + i]));
  }
  q.t0 = min(max(low, -1) + 1, q.length) / KT;
  q.nt = (q.length + KT - 1) / KT - q.t0;
  q.nd = (q.drafted + 31) / 32;
  return q;
}

__device__ __forceinline__ int pieces_of(const Segments& q, int run) { return (q.tiles() + run - 1) / run; }      // of one segment

// All sequences, 64 at a time, a lane each; the first 64 are looked up once
template <int KT, int ROWS>
struct Batch {
  const TreeArgs& p;
  Segments mine;
  int lane;
  __device__ __forceinline__ Batch(const TreeArgs& a) : p(a), lane(threadIdx.x & 63) { mine = look(lane); }
  __device__ __forceinline__ Segments look(int b) const {
    Segments q{};
    if (b < p.B) q = segments_of<KT, ROWS>(p, b);
    return q;
  }
  __device__ __forceinline__ Segments at(int b0) const { return b0 == 0 ? mine : look(b0 + lane); }
  // f(segments) times heads and row blocks, summed over the sequences in front of `upto`
  template <typename F>
  __device__ __forceinline__ uint32_t sum(int upto, F f) const {
    uint32_t total = 0;
    for (int b0 = 0; b0 < upto; b0 += 64) {
      const Segments q = at(b0);
      uint32_t t = b0 + lane < upto ? (uint32_t)f(q) * q.blocks * p.G : 0;
#pragma unroll
      for (int m = 32; m > 0; m >>= 1) t += __shfl_xor(t, m, 64);
      total += __builtin_amdgcn_readfirstlane(t);
    }
    return total;
  }
  // The shortest that makes no more pieces than `target` (a piece more than places is a round more), looked for between total / target and three times
  // that, a length per lane; where none does (more segments than `target`), total / target: at most `target` pieces beyond one a segment.
  __device__ __forceinline__ int run_length() const {
    const uint32_t total = sum(p.B, [](const Segments& q) { return q.tiles(); });
    const uint32_t least = max((uint32_t)p.run, (total + p.target - 1) / p.target);
    if (p.B > 64) return (int)least;
    // (counted in f32: a length that makes a piece more than it seems is as good)
    const uint32_t run = least + least * lane / 32;
    const float each = (float)mine.tiles(), many = (float)(mine.blocks * p.G), inv = 1.0f / (float)run;
    float count = 0.f;
    for (int b = 0; b < p.B; ++b)
      count = __builtin_fmaf(ceilf(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(each), b)) * inv), __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(many), b)), count);
    const uint64_t fits = __ballot(count <= (float)p.target);
    return (int)(fits ? __builtin_amdgcn_readlane(run, __builtin_ctzll(fits)) : least);
  }
};

struct Piece : Segments {
  int b, g, rb, gs, R, from, to;      // tiles from .. to - 1 of the segment
  const int* bt;
  bool whole;
};

template <int KT, int ROWS>
__device__ __forceinline__ bool piece_of(const TreeArgs& p, Piece& s, int64_t& part) {
  int id, j = 0, n = 1;      // piece j of n
  if (!p.part) {             // row blocks of the same keys are neighbours: one XCD's L2 serves them
    id = xcd_contiguous(blockIdx.x, p.workgroups);
    if (id < 0) return false;
    s.rb = id % p.blocks; s.g = id / p.blocks % p.G; s.b = id / p.blocks / p.G;
    (Segments&)s = segments_of<KT, ROWS>(p, s.b);
    if (s.rb >= s.blocks) return false;
  } else {
    const Batch<KT, ROWS> all(p);
    const int run = all.run_length();
    const uint32_t total = all.sum(p.B, [&](const Segments& q) { return pieces_of(q, run); }), per = (total + 7) >> 3;
    if ((blockIdx.x >> 3) >= per) return false;
    id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);      // (the pieces that there are, evenly over the XCDs)
    if ((uint32_t)id >= total) return false;
    part = id;
    bool found = false;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      const Segments q = all.at(b0);
      const uint32_t t = (uint32_t)pieces_of(q, run) * q.blocks * p.G;
      uint32_t upto = t;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const uint32_t y = __shfl_up(upto, m, 64);
        upto += all.lane >= m ? y : 0;
      }
      const uint64_t has = __ballot((uint32_t)id < upto);
      if (has) {
        const int l = __builtin_ctzll(has);
        id -= __builtin_amdgcn_readlane(upto - t, l);
        s.b = b0 + l;
        s.f0 = __builtin_amdgcn_readlane(q.f0, l); s.drafted = __builtin_amdgcn_readlane(q.drafted, l); s.length = __builtin_amdgcn_readlane(q.length, l);
        s.t0 = __builtin_amdgcn_readlane(q.t0, l); s.nt = __builtin_amdgcn_readlane(q.nt, l); s.nd = __builtin_amdgcn_readlane(q.nd, l);
        s.blocks = __builtin_amdgcn_readlane(q.blocks, l);
        found = true;
        break;
      }
      id -= __builtin_amdgcn_readlane(upto, 63);
    }
    if (!found) return false;
    n = pieces_of(s, run);
    // row blocks of the same keys are neighbours
    s.rb = id % s.blocks; id /= s.blocks;
    j = id % n; s.g = id / n;
    if (j == 0 && threadIdx.x == 0) {
      int* c = p.cuts + 2 * ((s.b * p.G + s.g) * p.blocks + s.rb);
      c[0] = (int)part; c[1] = n;      // (its pieces are s.blocks apart)
    }
  }
  s.from = (int)((int64_t)j * s.tiles() / n);
  s.to = (int)((int64_t)(j + 1) * s.tiles() / n);
  s.whole = n == 1;
  // (all of it is uniform; says so where the compiler does not see it)
  for (int* f : {&s.f0, &s.drafted, &s.length, &s.t0, &s.nt, &s.nd, &s.blocks, &s.b, &s.g, &s.rb, &s.from, &s.to}) *f = __builtin_amdgcn_readfirstlane(*f);
  part *= ROWS;          // rows of the scratch in front of this piece's
  s.gs = p.H / p.G;
  s.R = s.drafted * s.gs;
  s.bt = p.bt + (int64_t)s.b * p.bt_stride;
  return true;
}

// Many rows (lm_tree_wide.hip)
bool tree_wide_takes(int rows, int dk, int dv);
int tree_wide_fit(int rows, int dk, int dv, bool codes);      // workgroups on the chip
int tree_wide_rows(int rows, int dk, int dv);      // of a workgroup
int launch_tree_wide(const TreeArgs& a, int dk, int dv, hipStream_t s);

}  // namespace lm
