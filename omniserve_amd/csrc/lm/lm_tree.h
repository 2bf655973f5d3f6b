// What the two kernels of drafted tokens' attention share (lm_tree_attn.hip: few rows, lm_tree_wide.hip: many).
#pragma once
#include "lm_attn.h"
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
  float* ml; float* part;                            // nsplit > 1: [n * H][nsplit][2] and [n * H][nsplit][dv]
  float scale;                                       // includes log2(e)
  int window, n, H, G, B, nsplit, max_draft, blocks;
};

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

// w without its NaN codes (seven low bits ones); bad: there was one
__device__ __forceinline__ uint32_t drop_nan_codes(uint32_t w, bool& bad) {
  const uint32_t nan = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  bad |= nan != 0;
  return w & ~(nan - (nan >> 7) | nan);
}

// Which sequence's tokens, rows and keys a workgroup has
struct Share {
  int rb, split, g, b, f0, drafted, gs, R, length;
  const int* bt;
};
__device__ __forceinline__ bool share_of(const TreeArgs& p, Share& s, int rows) {
  const int id = xcd_contiguous(blockIdx.x, p.B * p.G * p.nsplit * p.blocks);
  if (id < 0) return false;
  // row blocks of the same keys are neighbours: one XCD's L2 serves them
  s.rb = id % p.blocks; s.split = id / p.blocks % p.nsplit; s.g = id / p.blocks / p.nsplit % p.G; s.b = id / p.blocks / p.nsplit / p.G;
  s.f0 = min(max(p.first[s.b], 0), p.n);
  s.drafted = min(max(p.first[s.b + 1] - s.f0, 0), min(p.max_draft, p.n - s.f0));
  s.gs = p.H / p.G;
  s.R = s.drafted * s.gs;
  s.length = min(max(p.length[s.b], 0), p.bt_width * PAGE);
  s.bt = p.bt + (int64_t)s.b * p.bt_stride;
  return s.rb * rows < s.R;
}

// Many rows (lm_tree_wide.hip): returns false where the kernel does not exist
bool tree_wide_takes(int rows, int dk, int dv);
int tree_wide_rows(int rows, int dk, int dv);      // of a workgroup
int launch_tree_wide(TreeArgs& a, int dk, int dv, hipStream_t s);

}  // namespace lm
