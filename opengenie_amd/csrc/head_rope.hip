// RMSNorm of each query and key head with the position rotation in the same
// pass, its backward pass, and the rotation alone.
//
// Per head row x of D elements, with r = (mean(x^2) + eps)^-1/2:
//   n = x r w,  y = Rot(n);
//   dn = Rot^T(dy),  dx = r (w dn - x r mean(w dn x r)),  dw = sum_rows dn x r.
// Rot turns the first R elements of the head in R / 2 planes by the token's
// angles, (a, b) -> (a cos - b sin, b cos + a sin), the planes being elements
// (i, i + R/2) (half layout) or (2i, 2i + 1) (interleaved); Rot^T is Rot with
// the sines negated. Everything is float32, rounded once to x's dtype.
//
// All of it is bound by HBM: x read and y written (backward: x and dy read,
// dx written). A lane holds 8 consecutive elements (16 bytes), LPH = D / 8
// lanes a head row, so a wave's load covers 64 / LPH rows; the mean goes
// through DPP within the LPH lanes, and in the half layout the other element
// of a plane comes from the lane R / 16 further by ds_bpermute, as packed
// 16-bit inputs (4 dwords for 8 elements; its norm factor is the same row's).
// A wave takes one token's heads (several tokens' where a token has fewer
// heads than the wave has rows) NV rows a lane at a time, so the token's
// angles are read once for NV rows. 9216 tokens, 32 + 32 heads of 128: 68 us,
// 4.5 TB/s; 4999 tokens, 64 heads of 64: 18.4 us forward, 28.5 back, 4.4 TB/s.
#include "common.h"
#include "host.h"

namespace oga {

struct HeadTensor {
  const void* x;
  const void* dy;  // backward only
  void* out;       // y, or dx
  const void* w;   // [D] or null
  int64_t xs[3], ds[3], os[3];  // element strides (batch, token, head); unit along D
  int heads;
  int hp;        // rows of one token side by side in a wave (power of two)
  int slices;    // NV x hp heads each
  int64_t units; // token groups x slices
  float* part;   // backward: [blocks][D] partial dw, or null
  int blocks;    // of the launch, this tensor's share
};

struct HeadRopeArgs {
  HeadTensor t[2];
  const void* cos;
  const void* sin;
  int64_t cs_row;     // row stride of the tables
  int64_t table_len;
  const void* pos;    // null: token n has table row n
  int pos64;
  int64_t pos_sb, pos_sn;
  int64_t batch, tokens;
  int rot;            // rotated elements of a head
  int wdt, tdt;
  int norm;
  float sin_sign;     // -1 turns back
  float eps;
};

constexpr int kHeadWaves = 4;

template <int XDT>
OGA_DEVICE uint4 pack8x(const float* f) {
  if constexpr (XDT == OGA_DT_F16)
    return make_uint4(pack_f16(f[0], f[1]), pack_f16(f[2], f[3]), pack_f16(f[4], f[5]), pack_f16(f[6], f[7]));
  else
    return pack8(f);
}

// Sum over the LPH (8, 16 or 32) lanes of a head row; every lane gets it.
template <int LPH>
OGA_DEVICE float head_sum(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v += dpp(v, IC<0xB1>{});                        // lane ^ 1
  v += dpp(v, IC<0x4E>{});                        // lane ^ 2
  v += dpp(v, IC<0x141>{});                       // mirror within 8: the other quad
  if constexpr (LPH >= 16) v += dpp(v, IC<0x140>{});  // mirror within 16: the other 8
  if constexpr (LPH >= 32)
    v += __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), 0x401F));  // lane ^ 16
  return v;
}

// What a lane needs of its token's angles and of the weight, for its 8
// elements (and the weight of the other element of each plane).
template <int LPH, bool INTER>
struct HeadLane {
  float c[INTER ? 4 : 8], s[INTER ? 4 : 8];  // s carries the sign of the plane's other element
  float w[8], wp[INTER ? 1 : 8];
  int partner;  // byte index for ds_bpermute
  bool turned;

  OGA_DEVICE void load(const HeadRopeArgs& a, const void* weight, int lane, int64_t row) {
    const int ch = lane % LPH;
    turned = 8 * ch < a.rot;
    const int half = a.rot / 16;  // lanes of half the rotated part
    const bool first = ch < half;
    const int pch = !INTER && turned ? (first ? ch + half : ch - half) : ch;
    partner = 4 * (lane - ch + pch);
    const int64_t at = row * a.cs_row + (!turned ? 0 : INTER ? 4 * ch : 8 * (first ? ch : ch - half));
    constexpr int N = INTER ? 4 : 8;
    if (a.tdt == OGA_DT_F32) {
      const float* pc = (const float*)a.cos + at;
      const float* ps = (const float*)a.sin + at;
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 u = *(const float4*)(pc + i), v = *(const float4*)(ps + i);
        c[i] = u.x, c[i + 1] = u.y, c[i + 2] = u.z, c[i + 3] = u.w;
        s[i] = v.x, s[i + 1] = v.y, s[i + 2] = v.z, s[i + 3] = v.w;
      }
    } else {
      const uint16_t* pc = (const uint16_t*)a.cos + at;
      const uint16_t* ps = (const uint16_t*)a.sin + at;
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const uint2 u = *(const uint2*)(pc + i), v = *(const uint2*)(ps + i);
        c[i] = bf16_lo(u.x), c[i + 1] = bf16_hi(u.x), c[i + 2] = bf16_lo(u.y), c[i + 3] = bf16_hi(u.y);
        s[i] = bf16_lo(v.x), s[i + 1] = bf16_hi(v.x), s[i + 2] = bf16_lo(v.y), s[i + 3] = bf16_hi(v.y);
      }
    }
    const float sg = !INTER && first ? -a.sin_sign : a.sin_sign;
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] *= sg;
    if (weight) {
      load8(weight, a.wdt, 8 * ch, 1, true, w);
      if constexpr (!INTER) load8(weight, a.wdt, 8 * pch, 1, true, wp);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = 1.0f;
      if constexpr (!INTER) {
#pragma unroll
        for (int i = 0; i < 8; ++i) wp[i] = 1.0f;
      }
    }
  }

  // Rot of 8 elements n, np those of the planes' other elements (half layout).
  OGA_DEVICE void turn(const float* n, const float* np, float* y) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (INTER) {
        const float o = (i & 1) ? n[i - 1] : -n[i + 1];
        y[i] = turned ? fmaf(n[i], c[i / 2], o * s[i / 2]) : n[i];
      } else {
        y[i] = turned ? fmaf(n[i], c[i], np[i] * s[i]) : n[i];
      }
    }
  }

  // The planes' other elements, unscaled, from the lane that holds them.
  template <int XDT>
  OGA_DEVICE void other(const uint4& u, float* f) const {
    uint4 v;
    v.x = __builtin_amdgcn_ds_bpermute(partner, u.x);
    v.y = __builtin_amdgcn_ds_bpermute(partner, u.y);
    v.z = __builtin_amdgcn_ds_bpermute(partner, u.z);
    v.w = __builtin_amdgcn_ds_bpermute(partner, u.w);
    unpack8x<XDT>(v, f);
  }
};

// Where unit u's lane works: its token (batch b, token n, valid or clamped)
// and the first of its heads.
struct HeadSpot {
  int64_t b, n, row;
  int h0;
  bool valid;
};
template <int LPH, int NV>
OGA_DEVICE HeadSpot head_spot(const HeadRopeArgs& a, const HeadTensor& t, int64_t u, int lane) {
  HeadSpot p;
  const int g = lane / LPH;
  const int per = 64 / LPH / t.hp;  // tokens side by side
  const int64_t all = a.batch * a.tokens;
  const int64_t tg = u / t.slices;
  const int64_t tok = tg * per + g / t.hp;
  p.valid = tok < all;
  const int64_t tc = p.valid ? tok : all - 1;
  p.b = tc / a.tokens;
  p.n = tc - p.b * a.tokens;
  p.h0 = (int)(u - tg * t.slices) * NV * t.hp + g % t.hp;
  p.row = p.n;
  if (a.pos) {
    const int64_t at = p.b * a.pos_sb + p.n * a.pos_sn;
    p.row = a.pos64 ? ((const int64_t*)a.pos)[at] : (int64_t)((const int32_t*)a.pos)[at];
  }
  p.row = min(max(p.row, (int64_t)0), a.table_len - 1);  // a position outside the tables reads their end
  return p;
}

template <int XDT, int LPH, bool INTER, int NV>
__global__ __launch_bounds__(64 * kHeadWaves) void k_head_rope(HeadRopeArgs a) {
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const bool second = (int)blockIdx.x >= a.t[0].blocks;
  const HeadTensor& t = second ? a.t[1] : a.t[0];
  const int64_t u = (int64_t)(blockIdx.x - (second ? a.t[0].blocks : 0)) * kHeadWaves + wv;
  if (u >= t.units) return;
  const HeadSpot p = head_spot<LPH, NV>(a, t, u, lane);
  const int ch = lane % LPH;
  const uint16_t* x = (const uint16_t*)t.x + p.b * t.xs[0] + p.n * t.xs[1] + 8 * ch;
  uint4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = *(const uint4*)(x + min(p.h0 + i * t.hp, t.heads - 1) * t.xs[2]);
  HeadLane<LPH, INTER> l;
  l.load(a, t.w, lane, p.row);
  uint16_t* out = (uint16_t*)t.out + p.b * t.os[0] + p.n * t.os[1] + 8 * ch;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float f[8], fp[8], y[8];
    unpack8x<XDT>(v[i], f);
    float inv = 1.0f;
    if (a.norm) {
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
      inv = 1.0f / sqrtf(head_sum<LPH>(ss) * (1.0f / (8 * LPH)) + a.eps);
    }
    if constexpr (!INTER) l.template other<XDT>(v[i], fp);
    if (a.norm) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = f[e] * inv * l.w[e];
      if constexpr (!INTER) {
#pragma unroll
        for (int e = 0; e < 8; ++e) fp[e] = fp[e] * inv * l.wp[e];
      }
    }
    l.turn(f, fp, y);
    const int h = p.h0 + i * t.hp;
    if (p.valid && h < t.heads) *(uint4*)(out + h * t.os[2]) = pack8x<XDT>(y);
  }
}

// Backward. The waves of a workgroup walk the units of one tensor, each lane
// keeping dw of its 8 elements; at the end the workgroup adds its lanes' and
// leaves one row of D sums for k_head_dw.
template <int XDT, int LPH, bool INTER, int NV>
__global__ __launch_bounds__(64 * kHeadWaves) void k_head_rope_bwd(HeadRopeArgs a) {
  __shared__ float red[kHeadWaves * 64 * 9];  // 9: a lane's 8 sums, rows of different lanes on different banks
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const bool second = (int)blockIdx.x >= a.t[0].blocks;
  const HeadTensor& t = second ? a.t[1] : a.t[0];
  const int block = (int)blockIdx.x - (second ? a.t[0].blocks : 0);
  const int ch = lane % LPH;
  float dw[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[e] = 0.0f;
  for (int64_t u = (int64_t)block * kHeadWaves + wv; u < t.units; u += (int64_t)t.blocks * kHeadWaves) {
    const HeadSpot p = head_spot<LPH, NV>(a, t, u, lane);
    const uint16_t* x = (const uint16_t*)t.x + p.b * t.xs[0] + p.n * t.xs[1] + 8 * ch;
    const uint16_t* dy = (const uint16_t*)t.dy + p.b * t.ds[0] + p.n * t.ds[1] + 8 * ch;
    uint4 xv[NV], dv[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int h = min(p.h0 + i * t.hp, t.heads - 1);
      xv[i] = *(const uint4*)(x + h * t.xs[2]);
      dv[i] = *(const uint4*)(dy + h * t.ds[2]);
    }
    HeadLane<LPH, INTER> l;
    l.load(a, t.w, lane, p.row);
    uint16_t* out = (uint16_t*)t.out + p.b * t.os[0] + p.n * t.os[1] + 8 * ch;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[8], d[8], dp[8], dn[8];
      unpack8x<XDT>(xv[i], f);
      unpack8x<XDT>(dv[i], d);
      if constexpr (!INTER) l.template other<XDT>(dv[i], dp);
      l.turn(d, dp, dn);
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
      const float inv = 1.0f / sqrtf(head_sum<LPH>(ss) * (1.0f / (8 * LPH)) + a.eps);
      float along = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] *= inv;
        along = fmaf(dn[e] * l.w[e], f[e], along);
      }
      along = head_sum<LPH>(along) * (1.0f / (8 * LPH));
      const int h = p.h0 + i * t.hp;
      const bool live = p.valid && h < t.heads;
      float g[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        g[e] = inv * (dn[e] * l.w[e] - f[e] * along);
        if (live) dw[e] = fmaf(dn[e], f[e], dw[e]);
      }
      if (live) *(uint4*)(out + h * t.os[2]) = pack8x<XDT>(g);
    }
  }
  if (!t.part) return;  // (uniform over the workgroup)
#pragma unroll
  for (int e = 0; e < 8; ++e) red[(wv * 64 + lane) * 9 + e] = dw[e];
  __syncthreads();
  for (int d = threadIdx.x; d < 8 * LPH; d += 64 * kHeadWaves) {
    float sum = 0.0f;
    for (int r = d / 8; r < kHeadWaves * 64; r += LPH) sum += red[r * 9 + (d & 7)];
    t.part[(int64_t)block * (8 * LPH) + d] = sum;
  }
}

// dw of one tensor per workgroup from the rows the workgroups left: four
// columns a thread, each strip of threads every strips-th row in order (eight
// loads in flight; one at a time took 18 us for 1024 rows), then the strips in
// order, in float64.
struct HeadDwArgs {
  const float* part[2];
  void* dw[2];
  int blocks[2];
  int dim, wdt;
};
__global__ __launch_bounds__(1024) void k_head_dw(HeadDwArgs a) {
  __shared__ double red[1024][4];
  const int i = blockIdx.x;
  const float* part = i ? a.part[1] : a.part[0];
  const int blocks = i ? a.blocks[1] : a.blocks[0];
  const int lanes = a.dim / 4, c = threadIdx.x % lanes, strip = threadIdx.x / lanes, strips = 1024 / lanes;
  double sum[4] = {0, 0, 0, 0};
  auto add = [&](const float4& v) { sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w; };
  int r = strip;
  for (; r + 7 * strips < blocks; r += 8 * strips) {
    float4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = *(const float4*)(part + (int64_t)(r + u * strips) * a.dim + 4 * c);
#pragma unroll
    for (int u = 0; u < 8; ++u) add(v[u]);
  }
  for (; r < blocks; r += strips) add(*(const float4*)(part + (int64_t)r * a.dim + 4 * c));
#pragma unroll
  for (int e = 0; e < 4; ++e) red[threadIdx.x][e] = sum[e];
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= a.dim) return;
  double all = 0.0;
  for (int s = 0; s < strips; ++s) all += red[s * lanes + d / 4][d & 3];
  void* out = i ? a.dw[1] : a.dw[0];
  if (a.wdt == OGA_DT_F32)
    ((float*)out)[d] = (float)all;
  else
    ((uint16_t*)out)[d] = (uint16_t)(pack_bf16((float)all, 0.0f) & 0xFFFFu);
}

static int pow2_ceil(int64_t v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

// Waves' worth of rows per lane: NV rows keep NV loads in flight and read the
// angles once for NV rows, but a call of few tokens then fills few CUs.
template <int NV>
static void head_plan(HeadTensor& t, int64_t all_tokens, int head_dim) {
  const int rows = 512 / head_dim;  // rows of a wave
  t.hp = min(rows, pow2_ceil(t.heads));
  const int per = rows / t.hp;
  t.slices = (int)((t.heads + (int64_t)NV * t.hp - 1) / ((int64_t)NV * t.hp));
  t.units = (all_tokens + per - 1) / per * t.slices;
}

template <int XDT, bool BWD, int NV, int LPH>
static void head_launch2(const HeadRopeArgs& a, bool inter, dim3 grid, hipStream_t s) {
  const dim3 block(64 * kHeadWaves);
  if constexpr (BWD) {
    if (inter)
      k_head_rope_bwd<XDT, LPH, true, NV><<<grid, block, 0, s>>>(a);
    else
      k_head_rope_bwd<XDT, LPH, false, NV><<<grid, block, 0, s>>>(a);
  } else {
    if (inter)
      k_head_rope<XDT, LPH, true, NV><<<grid, block, 0, s>>>(a);
    else
      k_head_rope<XDT, LPH, false, NV><<<grid, block, 0, s>>>(a);
  }
}

template <int XDT, bool BWD, int NV>
static void head_launch(HeadRopeArgs& a, bool inter, int head_dim, int max_blocks, hipStream_t s) {
  for (int i = 0; i < 2; ++i) {
    HeadTensor& t = a.t[i];
    if (!t.heads) {
      t.units = 0, t.blocks = 0, t.hp = 1, t.slices = 1;
      continue;
    }
    head_plan<NV>(t, a.batch * a.tokens, head_dim);
    const int64_t blocks = (t.units + kHeadWaves - 1) / kHeadWaves;
    t.blocks = (int)blocks;
    if (BWD) {  // as many units for every workgroup
      const int64_t turns = (blocks + max_blocks - 1) / max_blocks;
      t.blocks = (int)((blocks + turns - 1) / turns);
    }
  }
  const dim3 grid((unsigned)(a.t[0].blocks + a.t[1].blocks));
  if (head_dim == 64)
    head_launch2<XDT, BWD, NV, 8>(a, inter, grid, s);
  else if (head_dim == 128)
    head_launch2<XDT, BWD, NV, 16>(a, inter, grid, s);
  else
    head_launch2<XDT, BWD, NV, 32>(a, inter, grid, s);
}

// Workgroups of the backward kernel per tensor: each leaves one row of dw.
constexpr int kHeadBwdBlocks = 1024;

static bool strides_ok(const void* p, const int64_t* s) {
  return aligned(p, 16) && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0;
}

static int head_common(HeadRopeArgs& a, int x_dtype, const void* q_weight, const void* k_weight, int weight_dtype,
                       const void* cos, const void* sin, int cs_dtype, int64_t cs_stride, int64_t table_len,
                       const void* positions, int positions64, const int64_t* pos_strides, int64_t batch,
                       int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rotary_dim,
                       float eps) {
  if (x_dtype != OGA_DT_BF16 && x_dtype != OGA_DT_F16) return fail("x dtype code %d", x_dtype);
  if (!dt_ok(cs_dtype)) return fail("cos/sin dtype code %d", cs_dtype);
  if ((q_weight || k_weight) && !dt_ok(weight_dtype)) return fail("weight dtype code %d", weight_dtype);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return unsupported("head_dim %lld", (long long)head_dim);
  if (rotary_dim < 16 || rotary_dim > head_dim || rotary_dim % 16)
    return fail("rotary_dim %lld of head_dim %lld", (long long)rotary_dim, (long long)head_dim);
  if (batch < 1 || tokens < 1 || heads < 1 || kv_heads < 0 || heads > 65536 || kv_heads > 65536)
    return fail("shape (%lld, %lld, %lld, %lld)", (long long)batch, (long long)tokens, (long long)heads,
                (long long)kv_heads);
  if (batch > (INT64_C(1) << 31) / tokens / (heads + kv_heads)) return unsupported("more than 2^31 head rows");
  if (!cos || !sin || table_len < 1) return fail("no cos/sin table");
  if (!positions && table_len < tokens) return fail("table of %lld rows for %lld tokens", (long long)table_len,
                                                    (long long)tokens);
  const int64_t es = dt_size(cs_dtype);
  if (!aligned(cos, 4 * es) || !aligned(sin, 4 * es) || cs_stride % 4) return fail("cos/sin alignment");
  if (cs_stride < 0) return fail("cos/sin row stride");
  if ((q_weight && !aligned(q_weight, 8 * (int64_t)dt_size(weight_dtype))) ||
      (k_weight && !aligned(k_weight, 8 * (int64_t)dt_size(weight_dtype))))
    return fail("weight alignment");
  a.cos = cos, a.sin = sin, a.cs_row = cs_stride, a.table_len = table_len;
  a.pos = positions, a.pos64 = positions64;
  a.pos_sb = positions ? pos_strides[0] : 0, a.pos_sn = positions ? pos_strides[1] : 0;
  a.batch = batch, a.tokens = tokens, a.rot = (int)rotary_dim;
  a.wdt = weight_dtype, a.tdt = cs_dtype, a.eps = eps;
  a.t[0].heads = (int)heads, a.t[1].heads = (int)kv_heads;
  a.t[0].w = q_weight, a.t[1].w = k_weight;
  return OGA_OK;
}

static void set3(int64_t* d, const int64_t* s) { d[0] = s[0], d[1] = s[1], d[2] = s[2]; }

}  // namespace oga

using namespace oga;

extern "C" int oga_head_rmsnorm_rope(int x_dtype, const void* q, const int64_t q_strides[3], const void* k,
                                     const int64_t k_strides[3], const void* q_weight, const void* k_weight,
                                     int weight_dtype, const void* cos, const void* sin, int cs_dtype,
                                     int64_t cs_stride, int64_t table_len, const void* positions, int positions64,
                                     const int64_t pos_strides[2], void* q_out, const int64_t qo_strides[3],
                                     void* k_out, const int64_t ko_strides[3], int64_t batch, int64_t tokens,
                                     int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rotary_dim,
                                     int interleaved, int inverse, int norm, float eps, void* stream) {
  HeadRopeArgs a = {};
  if (int rc = head_common(a, x_dtype, norm ? q_weight : nullptr, norm ? k_weight : nullptr, weight_dtype, cos, sin,
                           cs_dtype, cs_stride, table_len, positions, positions64, pos_strides, batch, tokens, heads,
                           kv_heads, head_dim, rotary_dim, eps))
    return rc;
  if (!q || !q_out || !strides_ok(q, q_strides) || !strides_ok(q_out, qo_strides)) return fail("q layout");
  if (kv_heads && (!k || !k_out || !strides_ok(k, k_strides) || !strides_ok(k_out, ko_strides)))
    return fail("k layout");
  a.norm = norm ? 1 : 0;
  a.sin_sign = inverse ? -1.0f : 1.0f;
  a.t[0].x = q, a.t[0].out = q_out, set3(a.t[0].xs, q_strides), set3(a.t[0].os, qo_strides);
  if (kv_heads) a.t[1].x = k, a.t[1].out = k_out, set3(a.t[1].xs, k_strides), set3(a.t[1].os, ko_strides);
  if (x_dtype == OGA_DT_F16)
    head_launch<OGA_DT_F16, false, 4>(a, interleaved, (int)head_dim, 0, (hipStream_t)stream);
  else
    head_launch<OGA_DT_BF16, false, 4>(a, interleaved, (int)head_dim, 0, (hipStream_t)stream);
  return launch_status();
}

extern "C" int64_t oga_head_rmsnorm_rope_bwd_workspace_bytes(int64_t head_dim) {
  return head_dim == 64 || head_dim == 128 || head_dim == 256 ? 2 * kHeadBwdBlocks * head_dim * 4 : 0;
}

extern "C" int oga_head_rmsnorm_rope_bwd(
    int x_dtype, const void* dq_out, const int64_t dqo_strides[3], const void* dk_out, const int64_t dko_strides[3],
    const void* q, const int64_t q_strides[3], const void* k, const int64_t k_strides[3], const void* q_weight,
    const void* k_weight, int weight_dtype, const void* cos, const void* sin, int cs_dtype, int64_t cs_stride,
    int64_t table_len, const void* positions, int positions64, const int64_t pos_strides[2], void* dq,
    const int64_t dq_strides[3], void* dk, const int64_t dk_strides[3], void* dq_weight, void* dk_weight,
    int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rotary_dim,
    int interleaved, float eps, void* workspace, int64_t workspace_bytes, void* stream) {
  HeadRopeArgs a = {};
  if (int rc = head_common(a, x_dtype, q_weight, k_weight, weight_dtype, cos, sin, cs_dtype, cs_stride, table_len,
                           positions, positions64, pos_strides, batch, tokens, heads, kv_heads, head_dim, rotary_dim,
                           eps))
    return rc;
  if (!q || !dq_out || !dq || !strides_ok(q, q_strides) || !strides_ok(dq_out, dqo_strides) ||
      !strides_ok(dq, dq_strides))
    return fail("q layout");
  if (kv_heads && (!k || !dk_out || !dk || !strides_ok(k, k_strides) || !strides_ok(dk_out, dko_strides) ||
                   !strides_ok(dk, dk_strides)))
    return fail("k layout");
  if ((dq_weight && !q_weight) || (dk_weight && (!k_weight || !kv_heads))) return fail("gradient of no weight");
  if ((dq_weight || dk_weight) &&
      (!workspace || !aligned(workspace, 16) || workspace_bytes < oga_head_rmsnorm_rope_bwd_workspace_bytes(head_dim)))
    return fail("workspace of %lld bytes", (long long)workspace_bytes);
  a.norm = 1;
  a.sin_sign = -1.0f;
  HeadTensor &tq = a.t[0], &tk = a.t[1];
  tq.x = q, tq.dy = dq_out, tq.out = dq;
  set3(tq.xs, q_strides), set3(tq.ds, dqo_strides), set3(tq.os, dq_strides);
  tq.part = dq_weight ? (float*)workspace : nullptr;
  if (kv_heads) {
    tk.x = k, tk.dy = dk_out, tk.out = dk;
    set3(tk.xs, k_strides), set3(tk.ds, dko_strides), set3(tk.os, dk_strides);
    tk.part = dk_weight ? (float*)workspace + kHeadBwdBlocks * head_dim : nullptr;
  }
  const hipStream_t s = (hipStream_t)stream;
  if (x_dtype == OGA_DT_F16)
    head_launch<OGA_DT_F16, true, 4>(a, interleaved, (int)head_dim, kHeadBwdBlocks, s);
  else
    head_launch<OGA_DT_BF16, true, 4>(a, interleaved, (int)head_dim, kHeadBwdBlocks, s);
  if (int rc = launch_status()) return rc;
  if (!dq_weight && !dk_weight) return OGA_OK;
  // one workgroup per weight that has a gradient
  HeadDwArgs d = {};
  d.dim = (int)head_dim, d.wdt = weight_dtype;
  int n = 0;
  for (int i = 0; i < 2; ++i) {
    void* dw = i ? dk_weight : dq_weight;
    if (!dw) continue;
    d.part[n] = a.t[i].part, d.dw[n] = dw, d.blocks[n] = a.t[i].blocks;
    ++n;
  }
  k_head_dw<<<dim3(n), dim3(1024), 0, s>>>(d);
  return launch_status();
}
