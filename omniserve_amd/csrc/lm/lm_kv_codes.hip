// Rotary positions of queries and keys, and the cache of 8-bit keys and values (lm_kv_codes.h): written with the rotation in the same
// launch, read back as rows.  All three are bound by memory: kernels of 12001 tokens of 40 heads of 128, half of each turned, 38.7 us, of 64 heads over 8 turned and stored 109,
// of 100000 tokens of 8 heads read back 125 (6.4, 4.3 and 4.9 TB/s read and written; a copy of 8 GB 4.8).
//
// Angles: position * frequency in 64 bits (32 hold an angle of a million radians to 2^-5 of one, a two-hundredth of a turn), taken
// modulo a turn and through sincospi once per token and pair, by the workgroup, for all of its heads.
//
// A workgroup takes a few tokens, so that its threads have several 16-byte pieces each and the sines are formed by all of them; few
// tokens (decode steps) are dealt out by heads too.
#include "lm_kv_codes.h"
#include "omniserve_lm.h"

namespace lm {

struct Turn {
  const double* freq;      // per pair; half = 0: nothing turns
  const int* pos;          // < 0: an empty place
  int half, halves;        // pairs (i, i + half) instead of (2 i, 2 i + 1)
  double factor;
};

struct RopeArgs {
  Turn turn;
  const elem_t* x; int64_t ldx;
  elem_t* o; int64_t ldo;
  int tokens, heads, dk, per, hpb;      // tokens, heads of a workgroup
  Divisor items, wg_items, half;        // pieces of a head; of a token's heads in this workgroup
  int vec;
};

template <typename T>
struct alignas(2 * sizeof(T)) CosSin { T c, s; };

// cos, sin of token t0 + i, pair k at out[i * half + k]
template <typename T>
__device__ __forceinline__ void sines(const Turn& r, CosSin<T>* out, const Divisor& half, int t0, int n) {
  for (int i = threadIdx.x; i < n * r.half; i += 256) {
    const int t = half.quotient(i), k = i - t * r.half;
    const double turns = (double)r.pos[t0 + t] * r.freq[k] * 0.31830988618379067;      // in half turns
    double s, c;
    sincospi(turns, &s, &c);
    out[i].c = (T)(c * r.factor);
    out[i].s = (T)(s * r.factor);
  }
  __syncthreads();
}

// Turns (and, to another place, copies) heads h0 .. h0 + nh - 1 of tokens t0 .. t0 + n - 1.
template <bool VEC>
__device__ __forceinline__ void rope_heads(const RopeArgs& p, const CosSin<float>* cs, int t0, int n, int h0, int nh) {
  constexpr int W = VEC ? FR : 1, U = VEC ? 4 : 2;
  const Turn& r = p.turn;
  const int half = r.half, pieces = r.halves ? half / W : 2 * half / (VEC ? FR : 2);      // that turn
  const uint32_t total = (uint32_t)n * nh * p.items.d;
  for (uint32_t i0 = threadIdx.x; i0 < total; i0 += 256 * U) {
    const elem_t* src[U];
    elem_t* dst[U];
    int at[U], cd[U];      // first pair in cs; distance of the second part, 0: pairs inside, -1: a copy
    frag_t a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = i0 + 256 * u;
      src[u] = nullptr;
      if (i >= total) continue;
      const int th = p.items.quotient(i), item = i - th * p.items.d, t = nh == (int)p.wg_items.d ? p.wg_items.quotient(th) : th / nh;
      const int h = h0 + th - t * nh;
      if (half && r.pos[t0 + t] < 0) continue;
      const int64_t base = (int64_t)h * p.dk;
      int d;
      if (item < pieces) {
        d = r.halves ? item * W : item * (VEC ? FR : 2);
        cd[u] = r.halves ? half : 0;
        at[u] = t * half + (r.halves ? d : d >> 1);
      } else {
        d = 2 * half + (item - pieces) * W;
        cd[u] = -1;
        at[u] = 0;
      }
      src[u] = p.x + (int64_t)(t0 + t) * p.ldx + base + d;
      dst[u] = p.o + (int64_t)(t0 + t) * p.ldo + base + d;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!src[u]) continue;
      if constexpr (VEC) {
        a[u] = *(const frag_t*)src[u];
        if (cd[u] > 0) b[u] = *(const frag_t*)(src[u] + cd[u]);
      } else {
        a[u][0] = src[u][0];
        if (cd[u] == 0) a[u][1] = src[u][1];
        if (cd[u] > 0) b[u][0] = src[u][cd[u]];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!src[u]) continue;
      if (cd[u] > 0) {
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float c = cs[at[u] + e].c, s = cs[at[u] + e].s, y = (float)a[u][e], z = (float)b[u][e];
          a[u][e] = (elem_t)__builtin_fmaf(y, c, -z * s);
          b[u][e] = (elem_t)__builtin_fmaf(z, c, y * s);
        }
        if constexpr (VEC) __builtin_nontemporal_store(b[u], (frag_t*)(dst[u] + cd[u]));
        else dst[u][cd[u]] = b[u][0];
      } else if (cd[u] == 0) {
#pragma unroll
        for (int e = 0; e < (VEC ? FR : 2); e += 2) {
          const float c = cs[at[u] + e / 2].c, s = cs[at[u] + e / 2].s, y = (float)a[u][e], z = (float)a[u][e + 1];
          a[u][e] = (elem_t)__builtin_fmaf(y, c, -z * s);
          a[u][e + 1] = (elem_t)__builtin_fmaf(z, c, y * s);
        }
      }
      if constexpr (VEC) __builtin_nontemporal_store(a[u], (frag_t*)dst[u]);
      else {
        dst[u][0] = a[u][0];
        if (cd[u] == 0) dst[u][1] = a[u][1];
      }
    }
  }
}

template <bool VEC>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int t0 = blockIdx.x * p.per, n = min(p.per, p.tokens - t0), h0 = blockIdx.y * p.hpb;
  CosSin<float>* cs = (CosSin<float>*)lds;
  sines(p.turn, cs, p.half, t0, n);
  rope_heads<VEC>(p, cs, t0, n, h0, min(p.hpb, p.heads - h0));
}

struct StoreArgs {
  RopeArgs q;                             // o null: queries are left alone
  const int* rows; int x_rows;            // token i is row rows[i] of x (null: row i), rows outside of x are none
  const int* slot;
  uint8_t* kc; uint8_t* vc; uint8_t* ke; uint8_t* ve;
  int64_t places;                         // pages * 64
  int H, G, dk, dv;
  Divisor kl, vl, heads;                  // lanes of a key, of a value row; kv heads
};

// The f32 next to d whose lowest bit says whether it is inexact: rounding it again to fewer bits gives what rounding d does.
__device__ __forceinline__ float to_odd(double d) {
  const float f = (float)d;
  uint32_t u = __float_as_uint(f);
  if ((double)f != d) u = (fabs((double)f) > fabs(d) ? u - 1 : u) | 1u;
  return __uint_as_float(u);
}

// One lane's FR values of a row -> codes; the `lanes` lanes of the row are neighbours
__device__ __forceinline__ void store_row(const float* y, int lanes, int l, uint8_t* codes, uint8_t* exp, bool live) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < FR; ++e) {
    const float m = fabsf(y[e]);
    top = m < __builtin_inff() ? fmaxf(top, m) : top;
  }
  for (int m = 1; m < lanes; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
  if (!live) return;
  const int e = row_exponent(top);
#if LM_ELEM == 0
  *(u32x2*)(codes + 8 * l) = (u32x2){encode4(y, e), encode4(y + 4, e)};
#else
  *(uint32_t*)(codes + 4 * l) = encode4(y, e);
#endif
  if (l == 0) *exp = (uint8_t)(e + 127);
}

// blockIdx.y 0: keys and values; the others: the queries' heads.  A row of codes is dk / FR neighbouring lanes (8 codes each in bf16), its
// largest magnitude 3 to 6 shuffles.  Keys are turned in 64 bits and rounded once: three fraction bits make an error in the last place of
// an intermediate format visible (a code next to the right one, 2^-4 of the value), and keys are the small part of a row.
template <bool VEC>
__global__ __launch_bounds__(256) void kv_store_kernel(StoreArgs p) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const RopeArgs& q = p.q;
  const Turn& r = q.turn;
  const int t0 = blockIdx.x * q.per, n = min(q.per, q.tokens - t0), tid = threadIdx.x;
  if (blockIdx.y > 0) {
    CosSin<float>* cs = (CosSin<float>*)lds;
    const int h0 = (blockIdx.y - 1) * q.hpb;
    if (r.half) sines(r, cs, q.half, t0, n);
    rope_heads<VEC>(q, cs, t0, n, h0, min(q.hpb, p.H - h0));
    return;
  }
  CosSin<double>* cs = (CosSin<double>*)lds;
  if (r.half) sines(r, cs, q.half, t0, n);
  for (int value = 0; value < 2; ++value) {
    const Divisor& lanes = value ? p.vl : p.kl;
    const int size = value ? p.dv : p.dk, total = n * p.G * (int)lanes.d;
    const int64_t col = (int64_t)(p.H + (value ? p.G : 0)) * p.dk;
    for (int i = tid; i < (total + 255) / 256 * 256; i += 256) {
      const int th = lanes.quotient(i), l = i - th * lanes.d, t = p.heads.quotient(th), g = th - t * p.G, d = l * FR;
      bool live = i < total;
      int slot = 0, row = 0;
      if (live) {
        row = p.rows ? p.rows[t0 + t] : t0 + t;
        slot = p.slot[t0 + t];
        live = (uint32_t)row < (uint32_t)p.x_rows && slot >= 0 && slot < p.places && !(r.half && r.pos[t0 + t] < 0);
      }
      float y[FR] = {};
      if (live) {
        const elem_t* src = q.x + (int64_t)row * q.ldx + col + (int64_t)g * size;
        frag_t a;
        if constexpr (VEC) a = *(const frag_t*)(src + d);
        else
#pragma unroll
          for (int e = 0; e < FR; ++e) a[e] = src[d + e];
        if (value || d >= 2 * r.half) {
#pragma unroll
          for (int e = 0; e < FR; ++e) y[e] = (float)a[e];
        } else if (r.halves) {
          frag_t b;
          if (VEC && r.half % FR == 0) b = *(const frag_t*)(src + (d < r.half ? d + r.half : d - r.half));
          else
#pragma unroll
            for (int e = 0; e < FR; ++e) b[e] = d + e >= 2 * r.half ? (elem_t)0.f : src[d + e < r.half ? d + e + r.half : d + e - r.half];
#pragma unroll
          for (int e = 0; e < FR; ++e) {
            const bool second = d + e >= r.half;
            if (d + e >= 2 * r.half) { y[e] = (float)a[e]; continue; }
            const CosSin<double> w = cs[t * r.half + (second ? d + e - r.half : d + e)];
            y[e] = to_odd(fma((double)a[e], w.c, (double)b[e] * (second ? w.s : -w.s)));
          }
        } else {
#pragma unroll
          for (int e = 0; e < FR; e += 2) {
            if (d + e >= 2 * r.half) { y[e] = (float)a[e]; y[e + 1] = (float)a[e + 1]; continue; }
            const CosSin<double> w = cs[t * r.half + ((d + e) >> 1)];
            y[e] = to_odd(fma((double)a[e], w.c, -(double)a[e + 1] * w.s));
            y[e + 1] = to_odd(fma((double)a[e + 1], w.c, (double)a[e] * w.s));
          }
        }
      }
      const int64_t at = ((int64_t)(slot / PAGE) * p.G + g) * PAGE + slot % PAGE;
      store_row(y, lanes.d, l, (value ? p.vc : p.kc) + at * size, (value ? p.ve : p.ke) + at, live);
    }
  }
}

struct LoadArgs {
  const uint8_t* codes[2]; const uint8_t* exps[2];
  elem_t* out[2]; int64_t ld[2];
  const int* slot;
  int64_t places;
  int G, size[2];
  int tokens, per;
  Divisor row, piece[2];                  // pieces of a token's keys and values; of one head's key, value
};

// 16 codes a thread: 16 bytes in, 32 (bf16) out; a piece each (several requests a thread, or streamed stores, took 135 - 160 us for 100000 tokens of 8
// heads, this 125: 4.9 TB/s read and written)
__global__ __launch_bounds__(256) void kv_load_kernel(LoadArgs p) {
  const int t0 = blockIdx.x * p.per, n = min(p.per, p.tokens - t0);
  const uint32_t total = (uint32_t)n * p.row.d, keys = (uint32_t)p.G * p.piece[0].d;
  for (uint32_t i = threadIdx.x; i < total; i += 256) {
    const int t = p.row.quotient(i);
    uint32_t j = i - t * p.row.d;
    const int v = j >= keys;
    j -= v ? keys : 0;
    const Divisor& pc = p.piece[v];
    const int g = pc.quotient(j), c = j - g * pc.d, slot = p.slot[t0 + t];
    u32x4 w = {0, 0, 0, 0};
    float f = 1.f;
    if (slot >= 0 && slot < p.places) {
      const int64_t at = ((int64_t)(slot / PAGE) * p.G + g) * PAGE + slot % PAGE;
      w = *(const u32x4*)(p.codes[v] + at * p.size[v] + 16 * c);
      f = scale_of(p.exps[v][at]);
    }
    elem_t* dst = p.out[v] + (int64_t)(t0 + t) * p.ld[v] + (int64_t)g * p.size[v] + 16 * c;
#pragma unroll
    for (int k = 0; k < 16 / FR; ++k) {
      frag_t y;
#pragma unroll
      for (int m = 0; m < FR / 4; ++m) {
        const quad_t z = decode4(w[k * (FR / 4) + m], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[4 * m + e] = z[e];
      }
      *(frag_t*)(dst + k * FR) = y;
    }
  }
}

constexpr int MOST_PAIRS = 512, MOST_HEADS = 4096;      // of a head; of a row

// Tokens of a workgroup: four pieces a thread where that leaves a thousand workgroups (12001 tokens of 40 heads: 2 tokens 40 us, 1 43.5, 4 41.4)
static int tokens_per_group(int tokens, int pieces, int half) {
  return max(1, min(min((1024 + pieces - 1) / max(pieces, 1), tokens / 1024), min(16, 2048 / max(half, 1))));
}

// How many heads a workgroup takes: all of them unless tokens are few
static int heads_per_group(int tokens, int heads) { return tokens >= 512 ? heads : tokens >= 64 ? min(heads, 16) : min(heads, 8); }

static bool aligned(const void* p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % FR == 0; }

static bool good_turn(const double* freq, int half, const int* pos, int dk) { return half >= 0 && half <= MOST_PAIRS && 2 * half <= dk && (half == 0 || (freq && pos)); }

static RopeArgs rope_args(const void* x, int64_t ldx, void* o, int64_t ldo, const Turn& t, int tokens, int heads, int dk) {
  RopeArgs a{};
  a.turn = t;
  a.x = (const elem_t*)x; a.ldx = ldx; a.o = (elem_t*)o; a.ldo = ldo;
  a.tokens = tokens; a.heads = heads; a.dk = dk;
  a.hpb = heads_per_group(tokens, heads);
  const int turning = t.halves ? t.half : 2 * t.half;      // elements of the pieces that turn
  a.vec = aligned(x, ldx) && aligned(o, ldo) && dk % FR == 0 && turning % FR == 0 && (dk - 2 * t.half) % FR == 0;
  const bool in_place = o == x && ldo == ldx;
  const int rest = in_place ? 0 : dk - 2 * t.half;
  a.items = Divisor(a.vec ? (turning + rest) / FR : t.half + rest);
  a.per = tokens_per_group(tokens, a.hpb * a.items.d, t.half);
  a.wg_items = Divisor(a.hpb);
  a.half = Divisor(t.half > 0 ? t.half : 1);
  return a;
}

}  // namespace lm

using namespace lm;

extern "C" int lm_rope(const void* x, int64_t ldx, void* o, int64_t ldo, const double* freq, int half, const int* pos, int halves, double factor,
                       int tokens, int heads, int dk, void* stream) {
  if (tokens < 0 || heads <= 0 || heads > MOST_HEADS || dk <= 0 || half < 1 || !good_turn(freq, half, pos, dk) || (tokens && (!x || !o))) return LM_EINVAL;
  if (tokens == 0) return LM_OK;
  const RopeArgs a = rope_args(x, ldx, o, ldo, Turn{freq, pos, half, halves, factor}, tokens, heads, dk);
  if ((int64_t)a.per * a.hpb * a.items.d >= 1 << 20 || a.items.d > 4096) return LM_EINVAL;      // (Divisor)
  const dim3 grid((tokens + a.per - 1) / a.per, (heads + a.hpb - 1) / a.hpb);
  const size_t bytes = (size_t)a.per * half * sizeof(CosSin<float>);
  if (a.vec) hipLaunchKernelGGL((rope_kernel<true>), grid, dim3(256), bytes, (hipStream_t)stream, a);
  else hipLaunchKernelGGL((rope_kernel<false>), grid, dim3(256), bytes, (hipStream_t)stream, a);
  return launch_status();
}

static bool code_size(int d) { return d == 64 || d == 128 || d == 256; }

extern "C" int lm_kv_store(const void* x, int64_t ldx, int x_rows, const int* rows, const double* freq, int half, const int* pos, int halves, double factor, void* q,
                           int64_t ldq, const int* slot, uint8_t* kc, uint8_t* vc, uint8_t* ke, uint8_t* ve, int64_t pages, int tokens, int H, int G, int dk,
                           int dv, void* stream) {
  if (tokens < 0 || H < 0 || G <= 0 || H + G > MOST_HEADS || !code_size(dk) || !code_size(dv) || !good_turn(freq, half, pos, dk) || pages < 0 || pages * PAGE > INT32_MAX ||
      (q && (H == 0 || rows)) || x_rows < 0 || (tokens && (!x || !slot || !kc || !vc || !ke || !ve)) || (uintptr_t)kc % 8 || (uintptr_t)vc % 8)
    return LM_EINVAL;
  if (tokens == 0) return LM_OK;
  StoreArgs a{};
  a.q = rope_args(x, ldx, q, ldq, Turn{freq, pos, half, halves, factor}, tokens, H > 0 ? H : 1, dk);
  if (!q) {
    a.q.vec = aligned(x, ldx);
    a.q.per = tokens_per_group(tokens, G * (dk + dv) / FR, half);
  }
  a.rows = rows; a.x_rows = x_rows; a.slot = slot;
  a.kc = kc; a.vc = vc; a.ke = ke; a.ve = ve; a.places = pages * PAGE;
  a.H = H; a.G = G; a.dk = dk; a.dv = dv;
  a.kl = Divisor(dk / FR); a.vl = Divisor(dv / FR); a.heads = Divisor(G);
  if ((int64_t)a.q.per * G * (dk > dv ? dk : dv) >= 1 << 22) return LM_EINVAL;      // (Divisor)
  const dim3 grid((tokens + a.q.per - 1) / a.q.per, q ? 1 + (H + a.q.hpb - 1) / a.q.hpb : 1);
  const size_t bytes = (size_t)a.q.per * half * sizeof(CosSin<double>);
  if (a.q.vec) hipLaunchKernelGGL((kv_store_kernel<true>), grid, dim3(256), bytes, (hipStream_t)stream, a);
  else hipLaunchKernelGGL((kv_store_kernel<false>), grid, dim3(256), bytes, (hipStream_t)stream, a);
  return launch_status();
}

extern "C" int lm_kv_load(void* k, int64_t ldk, void* v, int64_t ldv, const uint8_t* kc, const uint8_t* vc, const uint8_t* ke, const uint8_t* ve, int64_t pages,
                          const int* slot, int tokens, int G, int dk, int dv, void* stream) {
  if (tokens < 0 || G <= 0 || G > MOST_HEADS || !code_size(dk) || !code_size(dv) || pages < 0 || pages * PAGE > INT32_MAX || ldk % FR || ldv % FR ||
      (tokens && (!k || !v || !kc || !vc || !ke || !ve || !slot)) || ((uintptr_t)k | (uintptr_t)v | (uintptr_t)kc | (uintptr_t)vc) % 16)
    return LM_EINVAL;
  if (tokens == 0) return LM_OK;
  LoadArgs a{};
  a.codes[0] = kc; a.codes[1] = vc; a.exps[0] = ke; a.exps[1] = ve;
  a.out[0] = (elem_t*)k; a.out[1] = (elem_t*)v; a.ld[0] = ldk; a.ld[1] = ldv;
  a.slot = slot; a.places = pages * PAGE; a.G = G; a.size[0] = dk; a.size[1] = dv;
  a.tokens = tokens;
  a.row = Divisor(G * (dk + dv) / 16);
  a.piece[0] = Divisor(dk / 16); a.piece[1] = Divisor(dv / 16);
  a.per = max(1u, 256 / a.row.d);
  if ((int64_t)a.row.d * a.row.d >= 1ll << 32) return LM_EINVAL;
  hipLaunchKernelGGL(kv_load_kernel, dim3((tokens + a.per - 1) / a.per), dim3(256), 0, (hipStream_t)stream, a);
  return launch_status();
}
