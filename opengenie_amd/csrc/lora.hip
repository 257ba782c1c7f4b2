// Low-rank adapters of many requests beside a shared projection, and their
// backward pass.
//
// Rows (tokens) are divided into segments, each with an adapter l (or none):
//   y' = y + s_l B_l (A_l x)          A_l [r, K], B_l [N, r]
//   dx = A_l^T dlow,  dlow = s_l B_l^T dy
//   dA_l = sum_rows dlow x^T,  dB_l = sum_rows dy low^T,  low = s_l A_l x.
// r is small, so every product is bound by moving x, y and dy once:
//  * k_lora_shrink: low (or dlow) [rows, r], float32, from the long rows. The
//    waves of a workgroup divide the long axis and add up in LDS; where rows
//    are few, several workgroups divide it too and each leaves its part.
//  * k_lora_expand: the [rows, N] (or [rows, K]) result from low, added to y;
//    it adds the parts of low up as it reads them, in order.
//  * k_lora_wgrad: dA and dB, one workgroup per adapter, 512 columns and part
//    of the adapter's rows; k_lora_join adds the parts, if any, in order.
// The sums low and dlow stay float32 in memory and enter the matrix products
// as two 16-bit halves (v = hi + lo), so only results are rounded.
//
// The segments are device data (no host synchronisation): a row tile of BM
// rows is paired with each segment it meets. With the bounds b_0 = 0,
// b_1 .. b_{S+1} (the starts) and b_{S+2} = T of S + 2 segments (the first and
// last without an adapter), pair number floor(b_s / BM) + s + j is tile
// floor(b_s / BM) + j of segment s: unique, since each next segment begins in
// the last tile of the one before or later, and below ceil(T / BM) + S + 2.
#include "common.h"
#include "host.h"

namespace oga {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// C[16 x 16] += A[16 x 32] B[32 x 16]: lane l has row (A) or column (B) l % 16
// at k = 8 (l / 16) .. +7, and of C column l % 16, rows 4 (l / 16) .. +3.
template <int XDT>
OGA_DEVICE f32x4 mfma16(const uint4& a, const uint4& b, const f32x4& c) {
  if constexpr (XDT == OGA_DT_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

template <int XDT>
OGA_DEVICE uint32_t pack2x(float a, float b) {
  return XDT == OGA_DT_F16 ? pack_f16(a, b) : pack_bf16(a, b);
}
template <int XDT>
OGA_DEVICE uint4 pack8x(const float* f) {
  return make_uint4(pack2x<XDT>(f[0], f[1]), pack2x<XDT>(f[2], f[3]), pack2x<XDT>(f[4], f[5]),
                    pack2x<XDT>(f[6], f[7]));
}
// The two 16-bit halves of 8 floats.
template <int XDT>
OGA_DEVICE void split8x(const float* f, uint4& hi, uint4& lo) {
  hi = pack8x<XDT>(f);
  float h[8], d[8];
  unpack8x<XDT>(hi, h);
#pragma unroll
  for (int i = 0; i < 8; ++i) d[i] = f[i] - h[i];
  lo = pack8x<XDT>(d);
}

// Bytes of a buffer resource, and an offset outside it.
constexpr int kPast = INT32_MAX - 15;

struct Segments {
  const int32_t* starts;  // [count + 1]
  const int32_t* ids;     // [count]
  int count;
  int adapters;
  int64_t rows;
};

// Bounds of segment s of count + 2 (see above), inside [0, rows] whatever
// the starts say.
OGA_DEVICE int64_t seg_bound(const Segments& g, int s) {
  if (s <= 0) return 0;
  if (s > g.count + 1) return g.rows;
  return min(max((int64_t)g.starts[s - 1], (int64_t)0), g.rows);
}

struct Pair {
  int64_t lo, hi, tile0;  // rows lo .. hi - 1 (none: hi <= lo) of the tile that begins at row tile0
  int adapter;            // -1: none
};

// Pair number p for tiles of bm rows. Lanes test 64 segments at a time, each
// with its bounds and adapter loaded side by side (one memory latency).
OGA_DEVICE Pair seg_pair(const Segments& g, int bm, int64_t p, int lane) {
  const int all = g.count + 2;
  int seg = 0, b0 = 0, b1 = 0, id = -1;
  for (int s0 = 0; s0 < all; s0 += 64) {
    const int s = s0 + lane;
    const int lo = (int)seg_bound(g, s), hi = (int)seg_bound(g, s + 1);  // (rows stay below 2^31)
    const int own = s >= 1 && s <= g.count ? g.ids[s - 1] : -1;
    const unsigned long long m = __ballot(s < all && lo / bm + s <= p);
    if (!m) break;
    const int top = 63 - __builtin_clzll(m);
    seg = s0 + top;
    b0 = __builtin_amdgcn_readlane(lo, top);
    b1 = __builtin_amdgcn_readlane(hi, top);
    id = __builtin_amdgcn_readlane(own, top);
    if (top < 63) break;
  }
  Pair r;
  r.tile0 = (p - seg) * bm;  // floor(b0 / bm) + j tiles down
  r.lo = max((int64_t)b0, r.tile0);
  r.hi = min((int64_t)b1, r.tile0 + bm);
  r.adapter = id >= 0 && id < g.adapters ? id : -1;
  return r;
}

static int64_t seg_pairs(int64_t rows, int64_t count, int bm) { return (rows + bm - 1) / bm + count + 2; }

// ------------------------------------------------------------------ shrink
struct ShrinkArgs {
  Segments g;
  const void* x;  // [rows, k], row stride xs
  int64_t xs;
  const void* w;  // [adapters, rank, k]
  const float* scale;
  float* low;     // [parts][rows, rank]
  int64_t k;
  int rank;
};

constexpr int kShrinkWaves = 4;

// 16 TB rows x 16 RB ranks per workgroup, part blockIdx.y of the long axis in
// chunks of 64 (a 128-byte line of each row), the waves in turn. The fragments
// come straight from memory; two chunks of loads are in flight. Each tile reads
// all of A, so larger ones read less of it through L2 (9216 rows x 4096, rank
// 64: 35.3 us with 32 rows, 28.1 with 64: 2.7 TB/s of x).
template <int XDT, int RB, int TB>
__global__ __launch_bounds__(64 * kShrinkWaves, 2) void k_lora_shrink(ShrinkArgs a) {
  __shared__ f32x4 red[kShrinkWaves][TB * RB][64];
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const Pair p = seg_pair(a.g, 16 * TB, blockIdx.x, lane);
  if (p.adapter < 0 || p.hi <= p.lo) return;  // (uniform over the workgroup)
  const int c = lane & 15, kg = 8 * (lane >> 4);
  const uint16_t* xr[TB];
#pragma unroll
  for (int t = 0; t < TB; ++t)
    xr[t] = (const uint16_t*)a.x + min(max(p.tile0 + 16 * t + c, p.lo), p.hi - 1) * a.xs + kg;
  const uint16_t* wr[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r)
    wr[r] = (const uint16_t*)a.w + ((int64_t)p.adapter * a.rank + min(16 * r + c, a.rank - 1)) * a.k + kg;
  f32x4 acc[TB][RB];
#pragma unroll
  for (int t = 0; t < TB; ++t)
#pragma unroll
    for (int r = 0; r < RB; ++r) acc[t][r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  struct Chunk {
    uint4 x[2][TB], w[2][RB];
  };
  const int chunks = (int)((a.k + 63) / 64), whole = (int)(a.k / 64);
  const int c0 = (int)((int64_t)chunks * blockIdx.y / gridDim.y), c1 = (int)((int64_t)chunks * (blockIdx.y + 1) / gridDim.y);
  auto load = [&](Chunk& f, int ch) {
    const int k0 = 64 * ch;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int t = 0; t < TB; ++t) f.x[h][t] = *(const uint4*)(xr[t] + k0 + 32 * h);
#pragma unroll
      for (int r = 0; r < RB; ++r) f.w[h][r] = *(const uint4*)(wr[r] + k0 + 32 * h);
    }
  };
  auto mul = [&](const Chunk& f) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int t = 0; t < TB; ++t) acc[t][r] = mfma16<XDT>(f.w[h][r], f.x[h][t], acc[t][r]);
  };
  // (no load behind a branch inside the loop: the wait before its products
  // would then be for every load)
  const int end = min(c1, whole);
  Chunk f0, f1;
  // This wave's n chunks, c0 + wv + 4 i, beginning with i = first: all tiles
  // would otherwise read the same columns of their rows at one time, which are
  // powers of two apart and so in the same few memory channels.
  const int n = end > c0 + wv ? (end - c0 - wv + kShrinkWaves - 1) / kShrinkWaves : 0;
  int ch = n ? c0 + wv + kShrinkWaves * (int)(blockIdx.x % (uint32_t)n) : 0;
  auto next = [&] {
    const int now = ch;
    ch = ch + kShrinkWaves < end ? ch + kShrinkWaves : c0 + wv;
    return now;
  };
  if (n) {
    load(f0, next());
    int i = 2;
    for (; i < n; i += 2) {
      load(f1, next());
      mul(f0);
      load(f0, next());
      mul(f1);
    }
    if (i == n) {
      load(f1, next());
      mul(f0);
      mul(f1);
    } else {
      mul(f0);
    }
  }
  if (c1 > whole && wv == (whole - c0) % kShrinkWaves) {  // the last 8 .. 56 of the axis
    const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool in = 64 * whole + 32 * h + kg < a.k;
#pragma unroll
      for (int t = 0; t < TB; ++t) {
        f0.x[h][t] = none;
        if (in) f0.x[h][t] = *(const uint4*)(xr[t] + 64 * whole + 32 * h);
      }
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        f0.w[h][r] = none;
        if (in) f0.w[h][r] = *(const uint4*)(wr[r] + 64 * whole + 32 * h);
      }
    }
    mul(f0);
  }
#pragma unroll
  for (int t = 0; t < TB; ++t)
#pragma unroll
    for (int r = 0; r < RB; ++r) red[wv][t * RB + r][lane] = acc[t][r];
  __syncthreads();
  const float scale = a.scale ? a.scale[p.adapter] : 1.0f;
  float* const low = a.low + blockIdx.y * a.g.rows * a.rank;
  for (int o = wv; o < TB * RB; o += kShrinkWaves) {
    f32x4 v = red[0][o][lane];
#pragma unroll
    for (int w = 1; w < kShrinkWaves; ++w) v += red[w][o][lane];
    const int64_t row = p.tile0 + 16 * (o / RB) + c;
    const int rank = 16 * (o % RB) + 4 * (lane >> 4);
    if (row >= p.lo && row < p.hi && rank < a.rank) *(f32x4*)(low + row * a.rank + rank) = v * scale;
  }
}

// ------------------------------------------------------------------ expand
struct ExpandArgs {
  Segments g;
  const float* low;  // [parts][rows, rank]
  float* low_sum;    // [rows, rank], their sum, or null
  const void* w;     // [adapters, n, rank]
  const void* y;     // [rows, n] or null (zero)
  void* out;         // [rows, n]; may be y
  int64_t ys, os;    // row strides
  int64_t n;
  int rank, parts;
  int bm;
  uint32_t col_blocks;
};

// Up to bm rows x 128 columns per wave, 16 rows at a time: operand A is low
// (16 rows, its two halves as fragments in LDS, shared by the waves), operand B
// of product j the eight columns' j-th, 8 (l % 16) + j for lane l, so that a
// lane ends with 8 consecutive columns of 4 rows and y moves in pieces of 256
// bytes a row (16 rows x 64 bytes at a time, as the other orientation has it,
// moved 2.9 TB/s). The weights' fragments stay in registers over the rows; y
// runs RING x 16 rows ahead. Rows and columns past the end are offsets past the
// end of a buffer resource, which loads give 0 for and stores drop: no branch
// stands between the loads and the wait counts. 9216 rows x 4096, rank 64: 38.4
// us, 3.9 TB/s of y (a bias add of that size 24.9 us); 48 with a tile's loads,
// products and stores one after the other (50 of them with 4 waves).
template <int XDT, int KS, int RING, int W>
__global__ __launch_bounds__(64 * W) void k_lora_expand(ExpandArgs a) {
  extern __shared__ uint4 lows[];  // [bm / 16, a multiple of RING][KS][2][64]
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  // column blocks in turn: the tile's low is read while it is in a cache
  const uint32_t tile = blockIdx.x / a.col_blocks, col_block = blockIdx.x % a.col_blocks;
  const Pair p = seg_pair(a.g, RING == 1 ? 16 : a.bm, tile, lane);
  if (p.hi <= p.lo || (p.adapter < 0 && a.y == a.out)) return;  // (rows without an adapter keep y)
  const int c = lane & 15, g4 = lane >> 4, kg = 8 * g4;
  const int64_t f0 = ((int64_t)col_block * W + wv) * 128, f = f0 + 8 * c;  // this lane's 8 columns
  const int rows = (int)(p.hi - p.lo), nb = (rows + 15) / 16;
  const uint32_t yo = f < a.n ? 2 * ((uint32_t)(4 * g4) * (uint32_t)a.ys + (uint32_t)f) : kPast;
  const uint32_t oo = f < a.n ? 2 * ((uint32_t)(4 * g4) * (uint32_t)a.os + (uint32_t)f) : kPast;
  // rows 16 b + 4 g4 .. + 3 of the pair
  auto fetch = [&](int b, u32x4(&v)[4]) {
    const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)((const uint16_t*)a.y + (p.lo + 16 * b) * a.ys), 0,
                                                      a.y ? kPast : 0, 0x00027000);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = __builtin_amdgcn_raw_buffer_load_b128(
          rs, 16 * b + 4 * g4 + i < rows ? min(yo + 2 * (uint32_t)(i * a.ys), (uint32_t)kPast) : kPast, 0, 0);
  };
  auto store = [&](int b, int i, const uint4& v) {
    const auto rs =
        __builtin_amdgcn_make_buffer_rsrc((uint16_t*)a.out + (p.lo + 16 * b) * a.os, 0, kPast, 0x00027000);
    __builtin_amdgcn_raw_buffer_store_b128(
        u32x4{v.x, v.y, v.z, v.w}, rs,
        16 * b + 4 * g4 + i < rows ? min(oo + 2 * (uint32_t)(i * a.os), (uint32_t)kPast) : kPast, 0, 2 /* nt */);
  };
  u32x4 yv[RING][4];
#pragma unroll
  for (int u = 0; u < RING; ++u) fetch(u, yv[u]);
  if (p.adapter < 0) {  // (dx: zero)
    for (int b = 0; b < nb; b += RING)
#pragma unroll
      for (int u = 0; u < RING; ++u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) store(b + u, i, make_uint4(yv[u][i][0], yv[u][i][1], yv[u][i][2], yv[u][i][3]));
        fetch(b + u + RING, yv[u]);
      }
    return;
  }
  const uint4 none = make_uint4(0, 0, 0, 0);
  uint4 w[8][KS];
  {
    const uint16_t* wa = (const uint16_t*)a.w + (int64_t)p.adapter * a.n * a.rank;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int s = 0; s < KS; ++s)
        w[j][s] = *(const uint4*)(wa + min(f + j, a.n - 1) * a.rank + min(32 * s + kg, a.rank - 8));
  }
  // wave w makes fragments w, w + W, ... of the pair's nb x KS
  for (int u = wv; u < nb * KS; u += W) {
    const int s = u % KS;
    const int64_t row = p.lo + 16 * (u / KS) + c, rc = min(row, p.hi - 1);
    float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (32 * s + kg < a.rank) {
      const int64_t step = a.g.rows * a.rank;
      const float* l = a.low + rc * a.rank + 32 * s + kg;
      for (int q = 0; q < a.parts; q += 4) {  // four parts' loads in flight
        float4 x[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float* m = l + min(q + e, a.parts - 1) * step;
          x[e] = *(const float4*)m, y[e] = *(const float4*)(m + 4);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (q + e >= a.parts) break;
          f[0] += x[e].x, f[1] += x[e].y, f[2] += x[e].z, f[3] += x[e].w;
          f[4] += y[e].x, f[5] += y[e].y, f[6] += y[e].z, f[7] += y[e].w;
        }
      }
      if (a.low_sum && row == rc && col_block == 0) {
        float* o = a.low_sum + row * a.rank + 32 * s + kg;
        *(float4*)o = make_float4(f[0], f[1], f[2], f[3]);
        *(float4*)(o + 4) = make_float4(f[4], f[5], f[6], f[7]);
      }
    }
    uint4 hi, lo;
    split8x<XDT>(f, hi, lo);
    lows[2 * u * 64 + lane] = hi;
    lows[(2 * u + 1) * 64 + lane] = lo;
  }
  // Every load so far has ended here, seen by the compiler too: its waits in the
  // loop would otherwise be for the weights as well, and so for every load.
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
  if (f0 >= a.n) return;  // (no barrier follows)
  if (a.rank < 32 * KS) {  // what is read past the rank counts as 0, whatever it holds
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int s = 0; s < KS; ++s)
        if (32 * s + kg >= a.rank) w[j][s] = none;
  }
  auto block = [&](int b, u32x4(&v)[4]) {
    f32x4 acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 1; h >= 0; --h) {
        const uint4 l = lows[(2 * (b * KS + s) + h) * 64 + lane];
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = mfma16<XDT>(l, w[j][s], acc[j]);
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float o[8];
      asm volatile("" : "+v"(v[i]));  // unpacked here, not ahead of the other blocks' loads
      unpack8x<XDT>(make_uint4(v[i][0], v[i][1], v[i][2], v[i][3]), o);  // (0 where there is no y)
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] += acc[j][i];
      store(b, i, pack8x<XDT>(o));
    }
  };
  // (a round's blocks past the last have nothing loaded or stored; an exit
  // between blocks would make the waits of all of them those of the first)
  for (int b = 0; b < nb; b += RING)
#pragma unroll
    for (int u = 0; u < RING; ++u) {
      block(b + u, yv[u]);
      if constexpr (RING > 1) fetch(b + u + RING, yv[u]);
    }
}

// -------------------------------------------------------- 16-bit transpose
// dst[l][c][r] = src[l][r][c] for the two weights (A and B) of one call.
struct TransposeArgs {
  const uint16_t* src[2];
  uint16_t* dst[2];
  int64_t rows[2], cols[2];
  int64_t blocks0;     // workgroups of the first
  int64_t tiles[2];    // 64 x 64 tiles per adapter
  int64_t col_tiles[2];
};
// 16 bytes a lane in and out (rows and cols are multiples of 8); the 66-element
// rows put the eight rows of a lane's column piece into eight banks.
__global__ __launch_bounds__(256) void k_lora_transpose(TransposeArgs a) {
  __shared__ uint32_t tile[64][33];
  const int i = (int64_t)blockIdx.x >= a.blocks0;
  const int64_t u = (int64_t)blockIdx.x - (i ? a.blocks0 : 0);
  const int64_t rows = i ? a.rows[1] : a.rows[0], cols = i ? a.cols[1] : a.cols[0];
  const int64_t tiles = i ? a.tiles[1] : a.tiles[0], ct = i ? a.col_tiles[1] : a.col_tiles[0];
  const int64_t l = u / tiles, t = u - l * tiles;
  const int64_t r0 = t / ct * 64, c0 = t % ct * 64;
  const uint16_t* src = (i ? a.src[1] : a.src[0]) + l * rows * cols;
  uint16_t* dst = (i ? a.dst[1] : a.dst[0]) + l * rows * cols;
  const int x = threadIdx.x & 7, y = threadIdx.x >> 3;
#pragma unroll
  for (int j = 0; j < 64; j += 32)
    if (r0 + y + j < rows && c0 + 8 * x < cols) {
      const uint4 v = *(const uint4*)(src + (r0 + y + j) * cols + c0 + 8 * x);
      uint32_t* o = &tile[y + j][4 * x];
      o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
    }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 64; j += 32)
    if (c0 + y + j < cols && r0 + 8 * x < rows) {
      uint32_t v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = tile[8 * x + e][(y + j) >> 1];
      const uint32_t sel = y & 1 ? 0x07060302u : 0x05040100u;  // (j is even)
      *(uint4*)(dst + (c0 + y + j) * rows + r0 + 8 * x) =
          make_uint4(__builtin_amdgcn_perm(v[1], v[0], sel), __builtin_amdgcn_perm(v[3], v[2], sel),
                     __builtin_amdgcn_perm(v[5], v[4], sel), __builtin_amdgcn_perm(v[7], v[6], sel));
    }
}

// ------------------------------------------------------- weight gradients
struct WgradSide {
  const void* x;     // [rows, c]: x for dA, dy for dB
  int64_t xs;
  const float* u;    // [rows, rank]: dlow for dA, low for dB
  int64_t c;
  float* part;       // [adapters][splits][rank][c]
  uint16_t* out;     // where the rows are not split
  int col_tiles;     // of 512 columns
};
struct WgradArgs {
  Segments g;
  WgradSide side[2];
  int rank, splits;
};

constexpr int kWgradRows = 128;  // rows of one pass over LDS
constexpr int kWgradPad = kWgradRows + 8;

// (4608 rows of x and dy of 4096, rank 32: 23.8 us, 3.2 TB/s; 26.5 with each
// step's rows waited for by a register copy.)
// One adapter, 4 x 128 columns, ranks 16 RB z .. , every splits-th 128-row
// tile of the adapter's segments. A lane loads 8 rows x 8 columns (16 lanes
// cover 256 bytes of a row) and regroups them by column with one v_perm per
// dword: column c of lanes is an MFMA operand whose k runs over rows.
template <int XDT, int RB>
__global__ __launch_bounds__(256) void k_lora_wgrad(WgradArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t uh[16 * RB * kWgradPad], ul[16 * RB * kWgradPad];
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const bool second = (int)blockIdx.x >= a.side[0].col_tiles;
  const WgradSide& sd = second ? a.side[1] : a.side[0];
  const int ct = (int)blockIdx.x - (second ? a.side[0].col_tiles : 0);
  const int adapter = blockIdx.y / a.splits, split = blockIdx.y % a.splits;
  const int r0 = 16 * RB * blockIdx.z;
  const int c = lane & 15, g8 = 8 * (lane >> 4);
  const int64_t col = (int64_t)ct * 512 + wv * 128 + 8 * c;
  const int64_t colc = min(col, sd.c - 8);
  f32x4 acc[8][RB];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int r = 0; r < RB; ++r) acc[j][r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  int64_t seen = 0;  // tiles of this adapter so far
  typedef u32x4 Rows8[8];
  const uint32_t xs2 = 2 * (uint32_t)sd.xs, x0 = (uint32_t)g8 * xs2 + 2 * (uint32_t)colc;
  auto tile = [&](int64_t lo, int64_t hi) {
    const int rows = (int)min(hi - lo, (int64_t)kWgradRows), steps = (rows + 31) / 32;
    // rows 32 st + g8 .. + 7; 0 past the segment's end, whose rows may hold anything
    auto rows8 = [&](Rows8& x, int st) {
      const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)((const uint16_t*)sd.x + (lo + 32 * st) * sd.xs), 0,
                                                        kPast, 0x00027000);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x[j] = __builtin_amdgcn_raw_buffer_load_b128(rs, 32 * st + g8 + j < rows ? x0 + j * xs2 : (uint32_t)kPast, 0, 0);
    };
    Rows8 cur, nxt;
    rows8(cur, 0);  // in flight while the tile's u goes to LDS
    rows8(nxt, 1);
    __syncthreads();  // the last tile's reads are done
    // a lane: four ranks of rows 2 i, 2 i + 1, which are neighbours in LDS
    constexpr int kQ = 4 * RB, kIt = kWgradRows / 2 * kQ / 256, kAhead = kIt < 2 ? kIt : 2;
    const int q = threadIdx.x % kQ, row0 = 2 * (int)(threadIdx.x / kQ);
    const bool in = r0 + 4 * q < a.rank;
    const float* up = sd.u + (in ? r0 + 4 * q : 0);
    for (int it = 0; it < kIt && it * (512 / kQ) < 64 * ((steps + 1) / 2); it += kAhead) {
      float4 v[2 * kAhead];
#pragma unroll
      for (int e = 0; e < 2 * kAhead; ++e)
        v[e] = *(const float4*)(up + min(lo + row0 + (it + e / 2) * (512 / kQ) + e % 2, hi - 1) * a.rank);
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const int row = row0 + (it + e) * (512 / kQ);
        const bool in0 = in && lo + row < hi, in1 = in && lo + row + 1 < hi;
        const float4 &x = v[2 * e], &y = v[2 * e + 1];
        const float f0[4] = {x.x, x.y, x.z, x.w}, f1[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a0 = in0 ? f0[i] : 0.0f, a1 = in1 ? f1[i] : 0.0f;
          const uint32_t h = pack2x<XDT>(a0, a1);
          *(uint32_t*)(uh + (4 * q + i) * kWgradPad + row) = h;
          *(uint32_t*)(ul + (4 * q + i) * kWgradPad + row) =
              pack2x<XDT>(a0 - x16_bits<XDT>(h & 0xFFFFu), a1 - x16_bits<XDT>(h >> 16));
        }
      }
    }
    __syncthreads();
    auto mul = [&](const Rows8& x, int st) {
      uint4 fh[RB], fl[RB];
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const int at = (16 * r + c) * kWgradPad + 32 * st + g8;
        fh[r] = *(const uint4*)(uh + at);
        fl[r] = *(const uint4*)(ul + at);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
        const uint4 xf = make_uint4(__builtin_amdgcn_perm(x[1][j >> 1], x[0][j >> 1], sel),
                                    __builtin_amdgcn_perm(x[3][j >> 1], x[2][j >> 1], sel),
                                    __builtin_amdgcn_perm(x[5][j >> 1], x[4][j >> 1], sel),
                                    __builtin_amdgcn_perm(x[7][j >> 1], x[6][j >> 1], sel));
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          acc[j][r] = mfma16<XDT>(fl[r], xf, acc[j][r]);
          acc[j][r] = mfma16<XDT>(fh[r], xf, acc[j][r]);
        }
      }
    };
    // Two steps at a time (a copy of rows in flight would wait for them), and
    // none of the second's work before the first's next loads.
    for (int st = 0; st < steps; st += 2) {
      mul(cur, st);
      rows8(cur, st + 2);
      __builtin_amdgcn_sched_barrier(0);
      mul(nxt, st + 1);
      rows8(nxt, st + 3);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (int s0 = 0; s0 < a.g.count; s0 += 64) {
    const int s = s0 + lane;
    const bool mine = s < a.g.count && a.g.ids[s] == adapter;
    const int64_t b0 = mine ? seg_bound(a.g, s + 1) : 0, b1 = mine ? seg_bound(a.g, s + 2) : 0;
    unsigned long long m = __ballot(mine && b0 < b1);
    while (m) {
      const int l = __builtin_ctzll(m);
      m &= m - 1;
      const int64_t lo = __builtin_amdgcn_readlane((int)b0, l), hi = __builtin_amdgcn_readlane((int)b1, l);
      for (int64_t t = lo; t < hi; t += kWgradRows, ++seen)
        if (seen % a.splits == split) tile(t, hi);
    }
  }
  if (col >= sd.c) return;
  if (a.splits == 1) {
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const int rank = r0 + 16 * r + 4 * (lane >> 4);  // .. + 3 (ranks are multiples of 8)
      if (rank >= a.rank) continue;
      if (!second) {  // dA [rank][k]
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f[8] = {acc[0][r][i], acc[1][r][i], acc[2][r][i], acc[3][r][i],
                              acc[4][r][i], acc[5][r][i], acc[6][r][i], acc[7][r][i]};
          *(uint4*)(sd.out + ((int64_t)adapter * a.rank + rank + i) * sd.c + col) = pack8x<XDT>(f);
        }
      } else {  // dB [n][rank]
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *(uint2*)(sd.out + ((int64_t)adapter * sd.c + col + j) * a.rank + rank) =
              make_uint2(pack2x<XDT>(acc[j][r][0], acc[j][r][1]), pack2x<XDT>(acc[j][r][2], acc[j][r][3]));
      }
    }
    return;
  }
  float* part = sd.part + ((int64_t)adapter * a.splits + split) * a.rank * sd.c;
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rank = r0 + 16 * r + 4 * (lane >> 4) + i;
      if (rank >= a.rank) continue;
      float* o = part + (int64_t)rank * sd.c + col;
      *(float4*)o = make_float4(acc[0][r][i], acc[1][r][i], acc[2][r][i], acc[3][r][i]);
      *(float4*)(o + 4) = make_float4(acc[4][r][i], acc[5][r][i], acc[6][r][i], acc[7][r][i]);
    }
}

struct JoinArgs {
  const float* part[2];  // [adapters][splits][rank][c]
  uint16_t* out[2];      // dA [adapters][rank][k], dB [adapters][n][rank]
  int64_t c[2];
  int64_t blocks0;       // workgroups of the first
  int64_t adapters;
  int rank, splits;
};
// Four columns of one rank (dA) or one column's four ranks (dB) a thread.
template <int XDT>
__global__ __launch_bounds__(256) void k_lora_join(JoinArgs a) {
  const bool second = (int64_t)blockIdx.x >= a.blocks0;
  const int64_t c = second ? a.c[1] : a.c[0];
  const int64_t i = ((int64_t)blockIdx.x - (second ? a.blocks0 : 0)) * 256 + threadIdx.x;
  const int64_t per = a.rank * c / 4;
  if (i >= a.adapters * per) return;
  const int64_t l = i / per, e = i - l * per;
  const float* part = (second ? a.part[1] : a.part[0]) + l * a.splits * a.rank * c;
  float v[4] = {0, 0, 0, 0};
  if (!second) {
    for (int s = 0; s < a.splits; ++s) {
      const float4 u = *(const float4*)(part + (int64_t)s * a.rank * c + 4 * e);
      v[0] += u.x, v[1] += u.y, v[2] += u.z, v[3] += u.w;
    }
    *(uint2*)(a.out[0] + l * a.rank * c + 4 * e) = make_uint2(pack2x<XDT>(v[0], v[1]), pack2x<XDT>(v[2], v[3]));
  } else {
    const int64_t q = e / c, col = e - q * c;  // ranks 4q .. 4q + 3: a wave reads consecutive columns
    for (int s = 0; s < a.splits; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += part[((int64_t)s * a.rank + 4 * q + r) * c + col];
    *(uint2*)(a.out[1] + (l * c + col) * a.rank + 4 * q) = make_uint2(pack2x<XDT>(v[0], v[1]), pack2x<XDT>(v[2], v[3]));
  }
}

// -------------------------------------------------------------------- host
// Blocks of 16 rows in a tile: more where segments are long and each fragment
// of the weights serves more rows, one where they are single tokens. 2048 rows,
// 4096 x 4096, rank 32, shrink + expand in us for 1 / 2 / 4 blocks: 200 requests
// 41 / 53 / 65, 64 requests 32 / 29 / 32, 32 requests 26 / 27 / 24.
static int row_blocks(int64_t rows, int64_t segments, int most) {
  const int64_t mean = rows / segments;
  return mean >= 48 ? most : mean >= 16 ? min(most, 2) : 1;
}

// (Rank 128 holds its weights' fragments for 32 rows at most.)
static int shrink_tiles(int64_t rank) { return rank > 64 ? 2 : 4; }

// Parts of the long axis: with two (64-row tiles, rank 128) or three workgroups a CU at
// a time, the number whose rounds times a part's length is least (each wave
// with two chunks or more).
static int shrink_parts(int64_t rows, int64_t segments, int64_t k, int64_t rank) {
  const int tb = row_blocks(rows, segments, shrink_tiles(rank));
  const int64_t pairs = seg_pairs(rows, segments, 16 * tb), slots = (tb == 4 || rank > 64 ? 2 : 3) * (int64_t)cu_count();
  const int64_t most = min((k + 63) / 64 / (2 * kShrinkWaves), (int64_t)8);
  int best = 1;
  double least = 1e30;
  for (int p = 1; p <= most; ++p) {
    const double cost = (double)((pairs * p + slots - 1) / slots) / p + 0.01 * p;
    if (cost < least) least = cost, best = p;
  }
  return best;
}

template <int XDT, int RB>
static void shrink_launch(const ShrinkArgs& a, int parts, hipStream_t s) {
  constexpr int most = RB >= 8 ? 2 : 4;
  const int tb = row_blocks(a.g.rows, a.g.count, most);
  const dim3 grid((unsigned)seg_pairs(a.g.rows, a.g.count, 16 * tb), parts), block(64 * kShrinkWaves);
  if (tb == 4)
    k_lora_shrink<XDT, RB, most><<<grid, block, 0, s>>>(a);
  else if (tb == 2)
    k_lora_shrink<XDT, RB, 2><<<grid, block, 0, s>>>(a);
  else
    k_lora_shrink<XDT, RB, 1><<<grid, block, 0, s>>>(a);
}
template <int XDT>
static void shrink(const ShrinkArgs& a, int parts, hipStream_t s) {
  if (a.rank <= 16)
    shrink_launch<XDT, 1>(a, parts, s);
  else if (a.rank <= 32)
    shrink_launch<XDT, 2>(a, parts, s);
  else if (a.rank <= 64)
    shrink_launch<XDT, 4>(a, parts, s);
  else
    shrink_launch<XDT, 8>(a, parts, s);
}

// Rows of an expand workgroup where segments are long: the number whose rounds
// of the CUs cost least, a workgroup's start counted as 24 rows (9216 rows, rank
// 64: 46.6 us with 64, 43.4 with 80, 42.0 with 144, 38.3 with 160, 38.1 with 192,
// 44.2 with 256; 4608 rows, rank 32: 22.5 with 64, 17.9 with 80, 22.2 with 144).
static int expand_rows(int64_t rows, int64_t segments, int64_t col_blocks, int most) {
  int best = 16;
  double least = 1e30;
  for (int bm = 16; bm <= most; bm += 16) {
    const int64_t wgs = ((rows + bm - 1) / bm + segments - 1) * col_blocks;
    const double cost = (double)((wgs + cu_count() - 1) / cu_count()) * (bm + 24);
    if (cost < least) least = cost, best = bm;
  }
  return best;
}

template <int XDT, int KS, int RING, int W>
static void expand_launch(ExpandArgs a, hipStream_t s) {
  a.col_blocks = (uint32_t)((a.n + 128 * W - 1) / (128 * W));
  a.bm = RING == 1 ? 16 : RING == 2 && a.g.rows / a.g.count < 48 ? 32 : expand_rows(a.g.rows, a.g.count, a.col_blocks, 512 / KS);
  const dim3 grid((unsigned)(seg_pairs(a.g.rows, a.g.count, a.bm) * a.col_blocks));
  k_lora_expand<XDT, KS, RING, W><<<grid, dim3(64 * W), (a.bm / 16 + RING - 1) / RING * RING * KS * 2048, s>>>(a);
}
template <int XDT, int KS>
static void expand_tiles(const ExpandArgs& a, hipStream_t s) {
  constexpr int most = KS >= 4 ? 2 : 4;
  const int tb = row_blocks(a.g.rows, a.g.count, most);
  if (tb == 4)
    expand_launch<XDT, KS, most, 8>(a, s);
  else if (tb == 2)
    expand_launch<XDT, KS, 2, 8>(a, s);
  else
    expand_launch<XDT, KS, 1, 4>(a, s);
}
template <int XDT>
static void expand(const ExpandArgs& a, hipStream_t s) {
  if (a.rank <= 32)
    expand_tiles<XDT, 1>(a, s);
  else if (a.rank <= 64)
    expand_tiles<XDT, 2>(a, s);
  else
    expand_tiles<XDT, 4>(a, s);
}

static int wgrad_rank_blocks(int rank) { return rank <= 16 ? 1 : rank <= 32 ? 2 : 4; }

// Parts of each adapter's rows: enough workgroups for one a CU, but no more
// than tiles of 128 rows an adapter has on average.
static int wgrad_splits(int64_t rows, int64_t adapters, int64_t k, int64_t n, int64_t rank) {
  const int64_t rz = (rank + 16 * wgrad_rank_blocks((int)rank) - 1) / (16 * wgrad_rank_blocks((int)rank));
  const int64_t wgs = ((k + 511) / 512 + (n + 511) / 512) * adapters * rz;
  const int64_t want = ((int64_t)cu_count() + wgs - 1) / wgs;
  const int64_t tiles = (rows + kWgradRows * adapters - 1) / (kWgradRows * adapters);
  return (int)max((int64_t)1, min(min(want, tiles), (int64_t)32));
}

template <int XDT>
static void wgrad(const WgradArgs& a, hipStream_t s) {
  const int rb = wgrad_rank_blocks(a.rank);
  const dim3 grid((unsigned)(a.side[0].col_tiles + a.side[1].col_tiles), (unsigned)(a.g.adapters * a.splits),
                  (unsigned)((a.rank + 16 * rb - 1) / (16 * rb)));
  if (rb == 1)
    k_lora_wgrad<XDT, 1><<<grid, dim3(256), 0, s>>>(a);
  else if (rb == 2)
    k_lora_wgrad<XDT, 2><<<grid, dim3(256), 0, s>>>(a);
  else
    k_lora_wgrad<XDT, 4><<<grid, dim3(256), 0, s>>>(a);
}

static int lora_shape(int x_dtype, int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t adapters,
                      int64_t segments, const void* starts, const void* ids) {
  if (x_dtype != OGA_DT_BF16 && x_dtype != OGA_DT_F16) return fail("x dtype code %d", x_dtype);
  if (rows < 1 || k < 8 || n < 8 || k % 8 || n % 8) return fail("shape rows %lld, k %lld, n %lld", (long long)rows,
                                                                (long long)k, (long long)n);
  if (rank < 8 || rank > 128 || rank % 8) return unsupported("rank %lld", (long long)rank);
  if (adapters < 1 || segments < 1 || adapters > 2000 || segments > (1 << 20))
    return fail("%lld adapters, %lld segments", (long long)adapters, (long long)segments);
  if (rows > (1 << 30) || k > (1 << 22) || n > (1 << 22))
    return unsupported("rows %lld, k %lld, n %lld", (long long)rows, (long long)k, (long long)n);
  // a grid holds less than 2^32 threads: 256 for 16 rows and 512 columns
  if (((rows + 15) / 16 + segments + 2) * ((max(k, n) + 511) / 512) >= 1 << 24)
    return unsupported("%lld rows, %lld segments of %lld, %lld columns", (long long)rows, (long long)segments, (long long)k,
                       (long long)n);
  if (!starts || !ids || !aligned(starts, 4) || !aligned(ids, 4)) return fail("segments");
  return OGA_OK;
}
static bool rows_ok(const void* p, int64_t stride) { return p && aligned(p, 16) && stride % 8 == 0; }
// Offsets inside 16 or 32 rows are 32-bit.
static bool near_rows(int64_t stride) { return stride >= 0 && stride < (1 << 25); }

static int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

// Layout of the backward workspace: the parts of dlow and dlow, A^T, B^T, the
// partial dA and dB.
struct LoraBwdSpace {
  int64_t dlow, at, bt, pa, pb, total;
  int parts, splits;
};
static LoraBwdSpace lora_bwd_space(int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t adapters,
                                   int64_t segments) {
  LoraBwdSpace w;
  w.parts = shrink_parts(rows, segments, n, rank);
  w.splits = wgrad_splits(rows, adapters, k, n, rank);
  w.dlow = align256(w.parts * rows * rank * 4);
  w.at = w.dlow + (w.parts > 1 ? align256(rows * rank * 4) : 0);
  w.bt = w.at + align256(adapters * rank * k * 2);
  w.pa = w.bt + align256(adapters * rank * n * 2);
  w.pb = w.pa + align256(adapters * w.splits * rank * k * 4);
  w.total = w.pb + align256(adapters * w.splits * rank * n * 4);
  if (w.splits == 1) w.pb = w.total = w.pa;  // (written straight away)
  if (w.parts == 1) w.dlow = 0;
  return w;
}

}  // namespace oga

using namespace oga;

extern "C" int64_t oga_lora_add_workspace_bytes(int64_t rows, int64_t k, int64_t rank, int64_t segments) {
  if (rows < 1 || k < 8 || rank < 8 || rank > 128 || segments < 1) return 0;
  return align256(shrink_parts(rows, segments, k, rank) * rows * rank * 4);
}

extern "C" int oga_lora_add(int x_dtype, const void* y, int64_t y_stride, const void* x, int64_t x_stride,
                            const void* a, const void* b, const float* scale, const int32_t* segment_starts,
                            const int32_t* segment_adapters, int64_t segments, int64_t adapters, float* low, void* out,
                            int64_t out_stride, int64_t rows, int64_t k, int64_t n, int64_t rank, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  if (int rc = lora_shape(x_dtype, rows, k, n, rank, adapters, segments, segment_starts, segment_adapters)) return rc;
  if (!rows_ok(y, y_stride) || !rows_ok(x, x_stride) || !rows_ok(out, out_stride) || !rows_ok(a, k) ||
      !rows_ok(b, rank) || !aligned(low, 16))
    return fail("operand alignment");
  if (!near_rows(y_stride) || !near_rows(out_stride))
    return unsupported("row strides %lld, %lld", (long long)y_stride, (long long)out_stride);
  const int64_t need = oga_lora_add_workspace_bytes(rows, k, rank, segments);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < need)
    return fail("workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  const Segments g = {segment_starts, segment_adapters, (int)segments, (int)adapters, rows};
  const int parts = shrink_parts(rows, segments, k, rank);
  const ShrinkArgs sa = {g, x, x_stride, a, scale, (float*)workspace, k, (int)rank};
  const ExpandArgs ea = {g, (const float*)workspace, low, b, y, out, y_stride, out_stride, n, (int)rank, parts, 0, 0};
  const hipStream_t s = (hipStream_t)stream;
  if (x_dtype == OGA_DT_F16) {
    shrink<OGA_DT_F16>(sa, parts, s);
    expand<OGA_DT_F16>(ea, s);
  } else {
    shrink<OGA_DT_BF16>(sa, parts, s);
    expand<OGA_DT_BF16>(ea, s);
  }
  return launch_status();
}

extern "C" int64_t oga_lora_bwd_workspace_bytes(int64_t rows, int64_t k, int64_t n, int64_t rank, int64_t adapters,
                                                int64_t segments) {
  if (rows < 1 || k < 8 || n < 8 || rank < 8 || rank > 128 || adapters < 1 || segments < 1) return 0;
  return lora_bwd_space(rows, k, n, rank, adapters, segments).total;
}

extern "C" int oga_lora_bwd(int x_dtype, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                            const float* low, const void* a, const void* b, const float* scale,
                            const int32_t* segment_starts, const int32_t* segment_adapters, int64_t segments,
                            int64_t adapters, void* dx, int64_t dx_stride, void* da, void* db, int64_t rows, int64_t k,
                            int64_t n, int64_t rank, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = lora_shape(x_dtype, rows, k, n, rank, adapters, segments, segment_starts, segment_adapters)) return rc;
  if (!rows_ok(dy, dy_stride) || !rows_ok(x, x_stride) || !rows_ok(dx, dx_stride) || !rows_ok(a, k) ||
      !rows_ok(b, rank) || !rows_ok(low, 8) || !rows_ok(da, 8) || !rows_ok(db, 8))
    return fail("operand alignment");
  if (!near_rows(dy_stride) || !near_rows(x_stride) || !near_rows(dx_stride))
    return unsupported("row strides %lld, %lld, %lld", (long long)dy_stride, (long long)x_stride, (long long)dx_stride);
  const LoraBwdSpace w = lora_bwd_space(rows, k, n, rank, adapters, segments);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < w.total)
    return fail("workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)w.total);
  char* const ws = (char*)workspace;
  float* const parts = (float*)ws;
  float* const dlow = (float*)(ws + w.dlow);  // the parts themselves where there is one
  const hipStream_t s = (hipStream_t)stream;

  TransposeArgs t = {};
  t.src[0] = (const uint16_t*)a, t.dst[0] = (uint16_t*)(ws + w.at), t.rows[0] = rank, t.cols[0] = k;
  t.src[1] = (const uint16_t*)b, t.dst[1] = (uint16_t*)(ws + w.bt), t.rows[1] = n, t.cols[1] = rank;
  for (int i = 0; i < 2; ++i) {
    t.col_tiles[i] = (t.cols[i] + 63) / 64;
    t.tiles[i] = (t.rows[i] + 63) / 64 * t.col_tiles[i];
  }
  t.blocks0 = adapters * t.tiles[0];
  k_lora_transpose<<<dim3((unsigned)(adapters * (t.tiles[0] + t.tiles[1]))), dim3(256), 0, s>>>(t);

  const Segments g = {segment_starts, segment_adapters, (int)segments, (int)adapters, rows};
  const ShrinkArgs sa = {g, dy, dy_stride, ws + w.bt, scale, parts, n, (int)rank};
  const ExpandArgs ea = {g, parts, w.parts > 1 ? dlow : nullptr, ws + w.at, nullptr, dx, 0, dx_stride, k, (int)rank,
                         w.parts, 0, 0};
  WgradArgs wa = {};
  wa.g = g, wa.rank = (int)rank, wa.splits = w.splits;
  wa.side[0] = {x, x_stride, dlow, k, (float*)(ws + w.pa), (uint16_t*)da, (int)((k + 511) / 512)};
  wa.side[1] = {dy, dy_stride, low, n, (float*)(ws + w.pb), (uint16_t*)db, (int)((n + 511) / 512)};
  JoinArgs j = {};
  j.part[0] = wa.side[0].part, j.part[1] = wa.side[1].part;
  j.out[0] = (uint16_t*)da, j.out[1] = (uint16_t*)db;
  j.c[0] = k, j.c[1] = n;
  j.adapters = adapters, j.rank = (int)rank, j.splits = w.splits;
  j.blocks0 = (adapters * rank * k / 4 + 255) / 256;
  const dim3 jgrid((unsigned)(j.blocks0 + (adapters * rank * n / 4 + 255) / 256));
  if (x_dtype == OGA_DT_F16) {
    shrink<OGA_DT_F16>(sa, w.parts, s);
    expand<OGA_DT_F16>(ea, s);
    wgrad<OGA_DT_F16>(wa, s);
    if (w.splits > 1) k_lora_join<OGA_DT_F16><<<jgrid, dim3(256), 0, s>>>(j);
  } else {
    shrink<OGA_DT_BF16>(sa, w.parts, s);
    expand<OGA_DT_BF16>(ea, s);
    wgrad<OGA_DT_BF16>(wa, s);
    if (w.splits > 1) k_lora_join<OGA_DT_BF16><<<jgrid, dim3(256), 0, s>>>(j);
  }
  return launch_status();
}
