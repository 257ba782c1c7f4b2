// Attention that is trained: a forward pass that keeps each row's log-sum-exp
// and a backward pass that recomputes the probabilities from it. bf16 in and
// out, head dimension 64 or 128, shared key/value heads, padded batches
// (k_lens) and causal masks; float32 softmax and sums.
//
//   S = c q k^T,  L_i = log sum_j exp S_ij,  P = exp(S - L),  O = P v
//   Delta_i = sum_d dO_id O_id,  dP = dO v^T,  dS = P (dP - Delta)
//   dv = P^T dO,  dq = c dS k,  dk = c dS^T q  (dk, dv: sums over the query
//   heads that share the key head)
// P and dS enter the second products rounded to bf16, everything else stays
// float32 until the results are rounded once.
//
// Three kernels share one loop shape: a wave keeps its own rows in registers
// and walks 64-row tiles of the other side, which LDS-DMA brings into a ring
// of three tile pairs, two steps ahead, or two where steps are few
// (k_attn_lse: 32 queries a wave over K and V; k_attn_dq: the same for dq;
// k_attn_dkv: 32 keys a wave over Q and dO of all query heads of the group).
// No sum crosses a workgroup by atomics: recomputing S and dP in both gradient
// kernels (7 products where 5 would do) costs less than writing and joining
// partial dq, and results do not depend on the order of workgroups. Blocks that
// would leave CUs idle are cut over their steps and joined in a fixed order.
//
// What bounds them: at D 128 the MFMAs and the power they draw (9216 x 9216, 32
// heads: busy 0.56 to 0.60 of the cycles), at D 64, with half the products per
// score, the exponentials and conversions (VALU 0.58 to 0.70, MFMA 0.41 to 0.50
// at 4099 x 4099 causal), over 256 keys the rows of Q, dO, out and the results
// (2 x 2304 rows: MFMA 0.22 to 0.32).
#include "common.h"
#include "host.h"

namespace oga {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kGT = 64;        // rows of a tile
constexpr int kMaxParts = 16;  // of a split block
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnGradArgs {
  const uint16_t *q, *k, *v, *dout, *out;
  uint16_t *o, *dq, *dk, *dv;
  int64_t q_s[3], k_s[3], v_s[3], do_s[3], o_s[3], dq_s[3], dk_s[3], dv_s[3];  // (batch, token, head); unit along D
  float* lse;          // [B, H, Nq]
  float* ld;           // [B, H, ceil(Nq / 64)][64 lse2 | 64 -Delta] (backward)
  float* part;         // what the parts of split blocks leave, float32
  float* part_ml;      // k_attn_lse: their running maxima and sums
  const int32_t* k_lens;
  int64_t nq, nk, batch;
  int heads, kv_heads, group;
  int blocks;          // query (key) blocks per (batch, head)
  int causal;
  int64_t nfull;       // blocks run whole; the others run as ksplit parts of their steps
  int ksplit;
  float scale, scale_log2;
};

OGA_DEVICE int64_t key_count(const AttnGradArgs& a, int64_t b) {
  return a.k_lens ? min(max((int64_t)a.k_lens[b], (int64_t)0), a.nk) : a.nk;
}

// The eight XCDs receive workgroups round-robin: renumbered so that each
// one's are consecutive, the blocks of a head share an L2.
OGA_DEVICE int64_t xcd_order(uint32_t block, uint32_t grid) {
  const uint32_t xcd = block & 7, per = grid >> 3, extra = grid & 7;
  return (int64_t)xcd * per + min(xcd, extra) + (block >> 3);
}

// The block a workgroup works on, and its part (-1: whole). Either all blocks
// run in ksplit parts (nfull 0), or blocks 0 .. nfull - 1 whole and the rest,
// which would fill only part of a last round of the CUs, in parts; a join adds
// the parts up. Causal blocks differ in length: the blocks with the most steps
// (blk 0) of all of an XCD's heads go first, so that the short ones fill up
// the end (heads in turn, 4099 x 32 heads x 64: 143 against 157 us for dq).
struct GradUnit {
  int64_t bh;
  int blk, part;
  int64_t slot;  // of a part's place in the workspace
};
template <bool CAUSAL>
OGA_DEVICE GradUnit grad_unit(const AttnGradArgs& a, int64_t bhs) {
  const uint32_t id = blockIdx.x;
  const int64_t nfull = a.nfull;
  GradUnit u;
  u.slot = 0;
  if (nfull && id >= nfull) {
    const uint32_t i = id - (uint32_t)nfull;
    const int64_t wg = nfull + i / (uint32_t)a.ksplit;
    u = {wg / a.blocks, (int)(wg % a.blocks), (int)(i % (uint32_t)a.ksplit), i};
    return u;
  }
  const uint32_t kk = nfull ? 1 : a.ksplit, all = nfull ? (uint32_t)nfull : gridDim.x;
  if (CAUSAL && bhs % 8 == 0 && all == gridDim.x) {
    const uint32_t per = (uint32_t)(bhs / 8) * kk, w = id >> 3, r = w % per;
    u = {(int64_t)(id & 7) * (bhs / 8) + r / kk, (int)(w / per), (int)(r % kk), 0};
  } else {
    const uint32_t o = (uint32_t)xcd_order(id, all), wg = o / kk;
    u = {wg / (uint32_t)a.blocks, (int)(wg % (uint32_t)a.blocks), (int)(o % kk), 0};
  }
  u.slot = (u.bh * a.blocks + u.blk) * kk + u.part;
  if (nfull) u.part = -1;
  return u;
}

// ------------------------------------------------------------- LDS tiles
// Row r of a tile (2 D bytes, D / 8 chunks of 16) keeps chunk c at c ^ sw(r).
// Two orders, by how the kernel reads: 32-row fragments (32x32x16 MFMA) with
// transposing reads of 4 rows x 64 bytes, or 16-row fragments (16x16x32) with
// transposing reads of 8 rows x 32 bytes. A ds_read_b128 is served 16 lanes at
// a time, lanes 0-3, 12-15, 20-23, 24-27 together (and 4-11, 16-19, 28-31),
// which for a 16-row fragment are rows 0-3, 12-15 of one chunk and 4-11 of the
// next one: sw16 keeps the two chunks of a pair apart for those rows, and for
// the 8 rows of a transposing read (checked below).
template <int D>
constexpr int sw32(int r) {
  return D == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}
template <int D>
constexpr int sw16(int r) {
  return D == 128 ? (((r & 7) ^ ((r >> 1) & 4)) << 1) | ((r >> 3) & 1)
                  : ((((r >> 1) & 3) ^ ((r >> 2) & 2)) << 1) | ((r >> 3) & 1);
}

template <int D>
constexpr bool frag16_conflict_free() {
  for (int s = 0; s < D / 32; ++s)
    for (int half = 0; half < 2; ++half)
      for (int first = 0; first < 2; ++first) {
        unsigned seen = 0;  // 16-byte columns of the 256 bytes of all banks
        for (int l = 0; l < 32; ++l) {
          const bool in = l < 4 || (l >= 12 && l < 16) || (l >= 20 && l < 28);
          if (in != (first == 0)) continue;
          const int r = l & 15, c = 4 * s + 2 * half + (l >> 4);
          seen |= 1u << ((r * (D / 8) + (c ^ sw16<D>(r))) & 15);
        }
        if (seen != 0xFFFF) return false;
      }
  for (int d = 0; d < D / 16; ++d)
    for (int r0 = 0; r0 < 16; r0 += 8) {
      unsigned seen = 0;
      for (int r = r0; r < r0 + 8; ++r)
        for (int c = 2 * d; c < 2 * d + 2; ++c) seen |= 1u << ((r * (D / 8) + (c ^ sw16<D>(r))) & 15);
      if (seen != 0xFFFF) return false;
    }
  return true;
}
static_assert(frag16_conflict_free<64>() && frag16_conflict_free<128>(), "fragment reads would conflict");

template <int OFF>
OGA_DEVICE bf16x8 rd_b128(uint32_t addr) {
  static_assert(OFF >= 0 && OFF < 2 * 65536, "LDS offset");
  uint4 v;
  if constexpr (OFF >= 65536)
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr + 65536u), "i"(OFF - 65536));
  else
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFF));
  return __builtin_bit_cast(bf16x8, v);
}
template <int OFF>
OGA_DEVICE u32x2 rd_tr16(uint32_t addr) {
  static_assert(OFF >= 0 && OFF < 2 * 65536, "LDS offset");
  u32x2 v;
  if constexpr (OFF >= 65536)
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(addr + 65536u), "i"(OFF - 65536));
  else
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFF));
  return v;
}
// An LDS address made where it is used: the compiler would otherwise keep the
// dozens of addresses that differ in a few bits in registers over the loop.
OGA_DEVICE uint32_t here(uint32_t addr, uint32_t add) {
  addr += add;
  asm volatile("" : "+v"(addr));
  return addr;
}
#define GRAD_LGKM(N, ...) asm volatile("s_waitcnt lgkmcnt(" #N ")" : __VA_ARGS__)

OGA_DEVICE bf16x8 frag2(const u32x2& a, const u32x2& b) {
  const uint4 u = {a[0], a[1], b[0], b[1]};
  return __builtin_bit_cast(bf16x8, u);
}
OGA_DEVICE f32x16 mfma32(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
OGA_DEVICE f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// LDS-DMA of a 64-row tile by W waves: instruction i of wave w fills 1 KiB.
// Rows past the last one (`rows` of them exist) read the last one again.
// A source is a uniform base and a 32-bit offset per lane. HOLD 2 keeps the two
// operands' offsets over the loop (4 registers). k_attn_dkv at D 128 has none
// to spare and makes them anew for each tile from the lane number: HOLD 1 once
// where the operands' row strides are equal, 0 (causal) for each operand, as
// even that costs spills.
template <int D, int W, bool S16, int HOLD>
struct TileDma {
  static constexpr bool KEEP = HOLD == 2;
  static constexpr int kCh = D / 8, kRpi = 64 / kCh, kDI = kGT / kRpi / W;
  static_assert(kDI >= 1, "waves");
  struct Off {
    uint32_t o[kDI];
  };
  Off full[KEEP ? 2 : 1];
  static OGA_DEVICE void offsets(Off& f, uint32_t row_stride, int rows, int wv, int lane) {
#pragma unroll
    for (int i = 0; i < kDI; ++i) {
      int row = (wv * kDI + i) * kRpi + lane / kCh;
      const int chunk = (lane % kCh) ^ (S16 ? sw16<D>(row) : sw32<D>(row));
      if (HOLD == 0 || rows < kGT) row = min(row, rows - 1);
      f.o[i] = __umul24((uint32_t)row, row_stride) * 2 + chunk * 16;
    }
  }
  static OGA_DEVICE void send(const uint16_t* base, const Off& f, char* lds, int wv) {
#pragma unroll
    for (int i = 0; i < kDI; ++i)
      __builtin_amdgcn_global_load_lds((const void*)((const char*)base + f.o[i]),
                                       (lds_void*)(lds + (wv * kDI + i) * 1024), 16, 0, 0);
  }
  OGA_DEVICE void init(uint32_t s0, uint32_t s1, int wv, int lane) {
    if constexpr (KEEP) {
      offsets(full[0], s0, kGT, wv, lane);
      offsets(full[1], s1, kGT, wv, lane);
    }
  }
  // The same `rows` rows of both operands into the tile pair at lds.
  OGA_DEVICE void pair(const uint16_t* b0, uint32_t s0, const uint16_t* b1, uint32_t s1, int rows, char* lds, int wv,
                       int lane) const {
    constexpr int kTile = kGT * D * 2;
    if (KEEP && rows >= kGT) {
      send(b0, full[0], lds, wv);
      send(b1, full[KEEP ? 1 : 0], lds + kTile, wv);
      return;
    }
    asm volatile("" : "+v"(lane));
    Off f;
    offsets(f, s0, rows, wv, lane);
    send(b0, f, lds, wv);
    if (HOLD == 0) asm volatile("" : "+v"(lane));
    if (HOLD == 0 || s1 != s0) offsets(f, s1, rows, wv, lane);
    send(b1, f, lds + kTile, wv);
  }
};

// One step of a kernel's tile loop in ring slot SLOT: wait until this wave's
// DMA of the step has landed (that of the next step, AHEAD instructions, may
// be in flight), then for every wave. A bare barrier: a fence would drain the
// DMA sent ahead, and the LDS reads are inline assembly.
template <int AHEAD>
OGA_DEVICE void ring_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(AHEAD) : "memory");
  asm volatile("s_barrier" ::: "memory");
}

OGA_DEVICE float max_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
OGA_DEVICE float sum_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---------------------------------------------------------------- forward
// W waves of 32 queries. S^T = K Q^T in 32 x 32 blocks (lane l: query l % 32,
// keys 8g + 4 (l / 32) + r), online softmax in base 2 with the running max
// moved only when a score passes it by 8 (P stays below 2^8), O^T += V^T P^T.
// 9216 x 9216, 32 heads of 128: 1215 us, 1145 TFLOP/s of its two products; 4099
// x 4099 causal, 32 / 8 heads of 64: 98 us.
template <int D, int W, int BUFS, bool CAUSAL>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2))) void k_attn_lse(
    AttnGradArgs a) {
  constexpr int kTile = kGT * D * 2, kPair = 2 * kTile, NS = D / 16, ND = D / 32;
  typedef TileDma<D, W, false, 2> Dma;
  __shared__ uint4 smem[BUFS * kPair / 16];
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const GradUnit unit = grad_unit<CAUSAL>(a, a.batch * a.heads);
  const int qb = CAUSAL ? a.blocks - 1 - unit.blk : unit.blk;
  const int64_t bh = unit.bh;
  const int h = (int)(bh % a.heads);
  const int64_t b = bh / a.heads;
  const int hk = h / a.group;
  const int hl = lane >> 5, ql = lane & 31;
  const int64_t q0 = (int64_t)qb * 32 * W + wv * 32;
  const int64_t nkb = key_count(a, b);
  const int64_t shift = nkb - a.nq;  // causal: query i sees keys <= i + shift
  int64_t kend = nkb;
  if (CAUSAL) kend = min(nkb, max((int64_t)0, min((int64_t)(qb + 1) * 32 * W, a.nq) + shift));
  const int nsteps = (int)((kend + kGT - 1) / kGT);
  const int st0 = unit.part < 0 ? 0 : (int)((int64_t)nsteps * unit.part / a.ksplit);
  const int st1 = unit.part < 0 ? nsteps : (int)((int64_t)nsteps * (unit.part + 1) / a.ksplit);

  const uint16_t* kb = a.k + b * a.k_s[0] + (int64_t)hk * a.k_s[2];
  const uint16_t* vb = a.v + b * a.v_s[0] + (int64_t)hk * a.v_s[2];
  char* const lds = (char*)smem;
  Dma tiles;
  tiles.init((uint32_t)a.k_s[1], (uint32_t)a.v_s[1], wv, lane);
  auto dma = [&](int st, int slot) {
    const int64_t key0 = (int64_t)st * kGT;
    tiles.pair(kb + key0 * a.k_s[1], (uint32_t)a.k_s[1], vb + key0 * a.v_s[1], (uint32_t)a.v_s[1],
               (int)min((int64_t)kGT, nkb - key0), lds + slot * kPair, wv, lane);
  };
  if (st1 > st0) {  // (uniform over the workgroup) in flight under the loads below
    dma(st0, 0);
    if (BUFS == 3) dma(min(st0 + 1, st1 - 1), 1);
  }
  bf16x8 qf[NS];
  {
    const uint16_t* qr = a.q + b * a.q_s[0] + min(q0 + ql, a.nq - 1) * a.q_s[1] + (int64_t)h * a.q_s[2];
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = __builtin_bit_cast(bf16x8, *(const uint4*)(qr + 16 * s + 8 * hl));
  }
  f32x16 o[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;


  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)smem;
  const uint32_t ka = lds0 + ql * (2 * D) + ((hl ^ sw32<D>(ql)) << 4);
  const int a4 = lane & 3, j4 = (lane & 15) >> 2, g2 = (lane >> 4) & 1;
  const uint32_t va = lds0 + kTile + (4 * hl + j4) * (2 * D) +
                      (((2 * g2 + (a4 >> 1)) ^ sw32<D>(4 * hl + j4)) << 4) + (a4 & 1) * 8;

  auto step = [&](auto slot_c, int st) {
    constexpr int SLOT = decltype(slot_c)::value, BASE = SLOT * kPair;
    ring_wait<BUFS == 3 ? 2 * Dma::kDI : 0>();
    if (BUFS == 3 || st + 1 < st1) dma(min(st + BUFS - 1, st1 - 1), (SLOT + BUFS - 1) % BUFS);
    // a wave behind the last query, or whose queries see none of these keys
    if (q0 >= a.nq || (CAUSAL && (int64_t)st * kGT > q0 + 31 + shift)) return;
    f32x16 s[2];
    auto block = [&](auto j_c) {
      constexpr int OFF = BASE + 32 * 2 * D * decltype(j_c)::value;
      bf16x8 f[NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) f[i] = rd_b128<OFF>(ka ^ (i << 5));
      if constexpr (NS == 8)
        GRAD_LGKM(0, "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3]), "+v"(f[4]), "+v"(f[5]), "+v"(f[6]), "+v"(f[7]));
      else
        GRAD_LGKM(0, "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3]));
      f32x16 acc;
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < NS; ++i) acc = mfma32(f[i], qf[i], acc);
      return acc;
    };
    s[0] = block(IC<0>{});
    s[1] = block(IC<1>{});
    // V^T of 16-key chunk C: reads for each 32-wide d-block, both 8-key halves
    auto read_v = [&](auto c_c, u32x2(&vr)[2 * ND]) {
      constexpr int OFF = BASE + 16 * 2 * D * decltype(c_c)::value;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        vr[2 * d] = rd_tr16<OFF>(va ^ (d << 6));
        vr[2 * d + 1] = rd_tr16<OFF + 8 * 2 * D>(va ^ ((d << 6) | 32));
      }
    };
    u32x2 v0[2 * ND], v1[2 * ND];
    read_v(IC<0>{}, v0);
    const int64_t key0 = (int64_t)st * kGT;
    // keys at or past `limit` (relative to this lane's first) are hidden
    const int64_t lim64 = CAUSAL ? min(nkb, q0 + ql + shift + 1) - key0 : nkb - key0;
    if (CAUSAL ? key0 + kGT > min(nkb, q0 + shift + 1) : lim64 < kGT) {
      const int lim = (int)max(min(lim64, (int64_t)kGT), (int64_t)-kGT) - 4 * hl;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (32 * j + 8 * (e >> 2) + (e & 3) >= lim) s[j][e] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = (j == 0 ? 1 : 0); e < 16; ++e) mx = __builtin_fmaxf(mx, s[j][e]);
    const float ms = max_halves(mx) * a.scale_log2;
    if (__any(ms > m_run + 8.0f)) {
      const float m_new = __builtin_fmaxf(m_run, ms);
      // a row that has seen no key yet keeps O = l = 0 (and m = -inf)
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.0f : m_new));
      l_run *= alpha;
      m_run = m_new;
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
    }
    const float nm = m_run == -INFINITY ? 0.0f : -m_run;
    uint32_t pb[2][8];
    float ps0 = 0.0f, ps1 = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][e], a.scale_log2, nm));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][e + 1], a.scale_log2, nm));
        ps0 += p0;
        ps1 += p1;
        pb[j][e >> 1] = pack_bf16(p0, p1);
      }
    l_run += ps0 + ps1;
    auto pv = [&](auto c_c, u32x2(&cur)[2 * ND], u32x2(&nxt)[2 * ND]) {
      constexpr int C = decltype(c_c)::value;
      if constexpr (C < 3) read_v(IC<(C + 1) & 3>{}, nxt);
      if constexpr (ND == 4) {
        if constexpr (C < 3)
          GRAD_LGKM(8, "+v"(cur[0]), "+v"(cur[1]), "+v"(cur[2]), "+v"(cur[3]), "+v"(cur[4]), "+v"(cur[5]), "+v"(cur[6]),
                    "+v"(cur[7]));
        else
          GRAD_LGKM(0, "+v"(cur[0]), "+v"(cur[1]), "+v"(cur[2]), "+v"(cur[3]), "+v"(cur[4]), "+v"(cur[5]), "+v"(cur[6]),
                    "+v"(cur[7]));
      } else {
        if constexpr (C < 3)
          GRAD_LGKM(4, "+v"(cur[0]), "+v"(cur[1]), "+v"(cur[2]), "+v"(cur[3]));
        else
          GRAD_LGKM(0, "+v"(cur[0]), "+v"(cur[1]), "+v"(cur[2]), "+v"(cur[3]));
      }
      const uint32_t* pw = &pb[C >> 1][4 * (C & 1)];
      const uint4 pu = {pw[0], pw[1], pw[2], pw[3]};
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] = mfma32(frag2(cur[2 * d], cur[2 * d + 1]), __builtin_bit_cast(bf16x8, pu), o[d]);
    };
    pv(IC<0>{}, v0, v1);
    pv(IC<1>{}, v1, v0);
    pv(IC<2>{}, v0, v1);
    pv(IC<3>{}, v1, v0);
  };

  {
    for (int st = st0; st < st1; st += BUFS) {
      step(IC<0>{}, st);
      if (st + 1 < st1) step(IC<1>{}, st + 1);
      if constexpr (BUFS == 3)
        if (st + 2 < st1) step(IC<2 % BUFS>{}, st + 2);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  const float l = sum_halves(l_run);
  if (unit.part >= 0) {  // O^T unnormalized, with m and l (every wave takes this branch)
    const int64_t row = unit.slot * 32 * W + wv * 32 + ql;
    if (q0 + ql >= a.nq) return;
    float* po = a.part + row * D;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(float4*)(po + 32 * d + 8 * g + 4 * hl) =
            make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
    if (hl == 0) *(float2*)(a.part_ml + 2 * row) = make_float2(m_run, l);
    return;
  }
  const float inv = l > 0.0f ? 1.0f / l : l;  // no key: 0; NaN stays
  const int64_t qi = q0 + ql;
  if (hl == 0 && qi < a.nq)
    a.lse[bh * a.nq + qi] = l == 0.0f ? -INFINITY : m_run * kLn2 + logf(l);
  // Through the wave's own LDS (the tiles are done with), so that each store
  // writes whole rows: 16-byte chunk c of row r sits at c ^ (r % (D / 8)).
  __syncthreads();
  char* const ot = lds + wv * 32 * 2 * D;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint2 w;
      w.x = pack_bf16(o[d][4 * g] * inv, o[d][4 * g + 1] * inv);
      w.y = pack_bf16(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv);
      *(uint2*)(ot + ql * 2 * D + (((4 * d + g) ^ (ql % (D / 8))) << 4) + 8 * hl) = w;
    }
  __syncthreads();
  constexpr int kLpr = D / 8, kRows = 64 / kLpr;  // lanes a row, rows a store
  const int oc = lane % kLpr;
  uint16_t* ob = a.o + b * a.o_s[0] + (int64_t)h * a.o_s[2] + 8 * oc;
#pragma unroll
  for (int it = 0; it < 32 / kRows; ++it) {
    const int r = kRows * it + lane / kLpr;
    const uint4 w = *(const uint4*)(ot + r * 2 * D + ((oc ^ (r % kLpr)) << 4));
    if (q0 + r < a.nq) *(uint4*)(ob + (q0 + r) * a.o_s[1]) = w;
  }
}

// out and lse of the blocks that ran in parts: O = sum 2^(m_p - M) O_p / L,
// L = sum 2^(m_p - M) l_p. D / 8 lanes a row.
template <int D, int ROWS>
__global__ __launch_bounds__(256) void k_attn_lse_join(AttnGradArgs a) {
  constexpr int kLpr = D / 8;
  const int64_t r = (int64_t)blockIdx.x * (256 / kLpr) + threadIdx.x / kLpr;  // (split block, row)
  const int64_t blk = r / ROWS, wg = a.nfull + blk;
  if (wg >= a.batch * a.heads * a.blocks) return;
  int qb = (int)(wg % a.blocks);
  if (a.causal) qb = a.blocks - 1 - qb;
  const int64_t bh = wg / a.blocks, row = r - blk * ROWS, qi = (int64_t)qb * ROWS + row;
  if (qi >= a.nq) return;
  const int c = threadIdx.x % kLpr;
  const int64_t first = blk * a.ksplit * ROWS + row;
  float2 ml[kMaxParts];  // with the first parts' loads behind them, before any is used
#pragma unroll
  for (int p = 0; p < kMaxParts; ++p) ml[p] = *(const float2*)(a.part_ml + 2 * (first + min(p, a.ksplit - 1) * ROWS));
  float m = -INFINITY, nm = 0.0f, l = 0.0f, o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int p0 = 0; p0 < kMaxParts; p0 += 8) {
    if (p0 >= a.ksplit) break;
    float4 u[8], v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float* f = a.part + (first + min(p0 + e, a.ksplit - 1) * ROWS) * D + 8 * c;
      u[e] = *(const float4*)f, v[e] = *(const float4*)(f + 4);
    }
    if (p0 == 0) {
#pragma unroll
      for (int p = 0; p < kMaxParts; ++p) m = __builtin_fmaxf(m, ml[p].x);  // a part read twice changes nothing
      nm = m == -INFINITY ? 0.0f : -m;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (p0 + e >= a.ksplit) break;
      const float w = __builtin_amdgcn_exp2f(ml[p0 + e].x + nm);
      l = fmaf(w, ml[p0 + e].y, l);
      o[0] = fmaf(w, u[e].x, o[0]), o[1] = fmaf(w, u[e].y, o[1]), o[2] = fmaf(w, u[e].z, o[2]), o[3] = fmaf(w, u[e].w, o[3]);
      o[4] = fmaf(w, v[e].x, o[4]), o[5] = fmaf(w, v[e].y, o[5]), o[6] = fmaf(w, v[e].z, o[6]), o[7] = fmaf(w, v[e].w, o[7]);
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : l;  // no key: 0; NaN stays
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] *= inv;
  const int64_t b = bh / a.heads, h = bh - b * a.heads;
  *(uint4*)(a.o + b * a.o_s[0] + qi * a.o_s[1] + h * a.o_s[2] + 8 * c) = pack8(o);
  if (c == 0) a.lse[bh * a.nq + qi] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
}

// --------------------------------------------------------------------- dq
// W waves of 32 queries over tiles of 64 keys. S^T = K Q^T and dP^T = V dO^T
// in 16 x 16 blocks (lane l: query l % 16, keys 4 (l / 16) + r), so a lane's
// lse and Delta are two numbers; dq^T += K^T dS^T with K^T by transposing
// reads, whose 32 keys' order (4 (l / 16) + r of two 16-key blocks) is that of
// the blocks' accumulators. 16x16x32 MFMAs reach 2083 TFLOP/s where 32x32x16
// reach 1585 (registers only, random operands: power), and no row maximum, for
// which a query should stay in two lanes, is needed here. 9216 x 9216, 32 heads
// of 128: 1604 us, 1301 TFLOP/s of its three products; 4099 x 4099 causal, 32 /
// 8 heads of 64: 122 us.
template <int D, int W, int BUFS, bool CAUSAL>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2))) void k_attn_dq(
    AttnGradArgs a) {
  constexpr int kTile = kGT * D * 2, kPair = 2 * kTile, NS = D / 32, ND = D / 16;
  typedef TileDma<D, W, true, 2> Dma;
  __shared__ uint4 smem[BUFS * kPair / 16];
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const GradUnit unit = grad_unit<CAUSAL>(a, a.batch * a.heads);
  const int qb = CAUSAL ? a.blocks - 1 - unit.blk : unit.blk;
  const int64_t bh = unit.bh;
  const int h = (int)(bh % a.heads);
  const int64_t b = bh / a.heads;
  const int hk = h / a.group;
  const int c16 = lane & 15, kg = lane >> 4;
  const int64_t q0 = (int64_t)qb * 32 * W + wv * 32;
  const int64_t nkb = key_count(a, b);
  const int64_t shift = nkb - a.nq;
  int64_t kend = nkb;
  if (CAUSAL) kend = min(nkb, max((int64_t)0, min((int64_t)(qb + 1) * 32 * W, a.nq) + shift));
  const int nsteps = (int)((kend + kGT - 1) / kGT);
  const int st0 = unit.part < 0 ? 0 : (int)((int64_t)nsteps * unit.part / a.ksplit);
  const int st1 = unit.part < 0 ? nsteps : (int)((int64_t)nsteps * (unit.part + 1) / a.ksplit);

  const uint16_t* kb = a.k + b * a.k_s[0] + (int64_t)hk * a.k_s[2];
  const uint16_t* vb = a.v + b * a.v_s[0] + (int64_t)hk * a.v_s[2];
  char* const lds = (char*)smem;
  Dma tiles;
  tiles.init((uint32_t)a.k_s[1], (uint32_t)a.v_s[1], wv, lane);
  auto dma = [&](int st, int slot) {
    const int64_t key0 = (int64_t)st * kGT;
    tiles.pair(kb + key0 * a.k_s[1], (uint32_t)a.k_s[1], vb + key0 * a.v_s[1], (uint32_t)a.v_s[1],
               (int)min((int64_t)kGT, nkb - key0), lds + slot * kPair, wv, lane);
  };
  if (st1 > st0) {  // (uniform over the workgroup) in flight under the loads below
    dma(st0, 0);
    if (BUFS == 3) dma(min(st0 + 1, st1 - 1), 1);
  }
  bf16x8 qf[2][NS], gf[2][NS];  // Q and dO, B operands: query 16 i + c16, d = 32 s + 8 kg ..
  // Base-2 lse and Delta of the lane's queries, left in ld for k_attn_dkv: a
  // query that saw no key, and the rows behind the last query up to the
  // tile's 64, get lse2 = +inf, so that their P is 0.
  float lse2[2], delta[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t qi = min(q0 + 16 * i + c16, a.nq - 1);
    const uint16_t* qr = a.q + b * a.q_s[0] + qi * a.q_s[1] + (int64_t)h * a.q_s[2] + 8 * kg;
    const uint16_t* gr = a.dout + b * a.do_s[0] + qi * a.do_s[1] + (int64_t)h * a.do_s[2] + 8 * kg;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      qf[i][s] = __builtin_bit_cast(bf16x8, *(const uint4*)(qr + 32 * s));
      gf[i][s] = __builtin_bit_cast(bf16x8, *(const uint4*)(gr + 32 * s));
    }
    const uint16_t* orow = a.out + b * a.o_s[0] + qi * a.o_s[1] + (int64_t)h * a.o_s[2] + 8 * kg;
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      float x[8], y[8];
      unpack8(*(const uint4*)(orow + 32 * s), x);
      unpack8(__builtin_bit_cast(uint4, gf[i][s]), y);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(x[e], y[e], sum);
    }
    sum += __shfl_xor(sum, 16, 64);
    delta[i] = sum + __shfl_xor(sum, 32, 64);
    const float l = a.lse[bh * a.nq + qi];
    const int64_t row = q0 + 16 * i + c16;
    lse2[i] = l == -INFINITY || row >= a.nq ? INFINITY : l * kLog2e;
  }
  // out is rounded, and with it Delta, by up to 2^-9 |dO| |out|. Over many keys
  // |out| is small beside the values and that is lost in dS's own rounding; a
  // row of few keys sums P (dP - Delta) over them, which is 0 for the exact
  // Delta, first (9 x 9 causal: dq off by 0.30 % without, by 0.24 % with it; from
  // 49 keys on by less than 0.25 % without). Causal, these are a head's first
  // waves, else all of them: 2 x 2304 rows over 64 keys would take 61 us for 40,
  // over 128 85 for 48.
  constexpr int kFewKeys = CAUSAL ? 128 : 48;
  const int64_t seen = CAUSAL ? min(nkb, q0 + 32 + shift) : nkb;
  if (seen <= kFewKeys && q0 < a.nq) {
    float num[2] = {0.0f, 0.0f}, den[2] = {0.0f, 0.0f};
#pragma unroll 2
    for (int64_t key0 = 0; key0 < seen; key0 += 16) {
      const int64_t ki = min(key0 + c16, nkb - 1);
      f32x4 s[2], g[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        g[i] = f32x4{-delta[i], -delta[i], -delta[i], -delta[i]};
      }
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        const bf16x8 kf = __builtin_bit_cast(bf16x8, *(const uint4*)(kb + ki * a.k_s[1] + 32 * x + 8 * kg));
        const bf16x8 vf = __builtin_bit_cast(bf16x8, *(const uint4*)(vb + ki * a.v_s[1] + 32 * x + 8 * kg));
#pragma unroll
        for (int i = 0; i < 2; ++i) s[i] = mfma16(kf, qf[i][x], s[i]), g[i] = mfma16(vf, gf[i][x], g[i]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t lim = (CAUSAL ? min(nkb, q0 + 16 * i + c16 + shift + 1) : nkb) - key0 - 4 * kg;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][r], a.scale_log2, -lse2[i]));
          num[i] += r < lim ? p * g[i][r] : 0.0f;
          den[i] += r < lim ? p : 0.0f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      num[i] += __shfl_xor(num[i], 16, 64), den[i] += __shfl_xor(den[i], 16, 64);
      num[i] += __shfl_xor(num[i], 32, 64), den[i] += __shfl_xor(den[i], 32, 64);
      if (den[i] > 0.0f) delta[i] += num[i] / den[i];
    }
  }
  const int64_t nqt = (a.nq + kGT - 1) / kGT;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t row = q0 + 16 * i + c16;
    if (kg == 0 && row < nqt * kGT && unit.part <= 0) {
      float* t = a.ld + (bh * nqt + row / kGT) * 128 + row % kGT;
      t[0] = lse2[i];
      t[64] = row < a.nq ? -delta[i] : 0.0f;
    }
  }
  f32x4 acc[ND][2];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 2; ++i) acc[d][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)smem;
  const uint32_t ra = lds0 + c16 * (2 * D) + ((kg ^ sw16<D>(c16)) << 4);
  const int a4 = lane & 3, j4 = (lane & 15) >> 2;
  const uint32_t ta = lds0 + (4 * kg + j4) * (2 * D) + (((a4 >> 1) ^ sw16<D>(4 * kg + j4)) << 4) + (a4 & 1) * 8;

  uint32_t ra4[NS], ta8[ND];
#pragma unroll
  for (int x = 0; x < NS; ++x) ra4[x] = ra ^ (x << 6);
#pragma unroll
  for (int x = 0; x < ND; ++x) ta8[x] = ta ^ (x << 5);
  auto step = [&](uint32_t base, int slot2, int st) {
    uint32_t rs[NS], ts[ND];
    ring_wait<BUFS == 3 ? 2 * Dma::kDI : 0>();
    if (BUFS == 3 || st + 1 < st1) dma(min(st + BUFS - 1, st1 - 1), slot2);
    if (q0 >= a.nq || (CAUSAL && (int64_t)st * kGT > q0 + 31 + shift)) return;
#pragma unroll
    for (int x = 0; x < NS; ++x) rs[x] = ra4[x] + base;
#pragma unroll
    for (int x = 0; x < ND; ++x) ts[x] = ta8[x] + base;
    const int64_t key0 = (int64_t)st * kGT;
    const bool edge = CAUSAL ? key0 + kGT > min(nkb, q0 + shift + 1) : key0 + kGT > nkb;
    auto half = [&](auto j_c) {  // keys 32 j .. + 31 of the tile
      constexpr int OFF = 32 * 2 * D * decltype(j_c)::value;
      uint32_t ds[2][4];  // dS^T, B operand of dq: query block i
      auto block = [&](auto u_c) {  // keys 16 u .. + 15 of these
        constexpr int U = decltype(u_c)::value;
        f32x4 s[2], g[2];
        bf16x8 kf[NS], vf[NS];
#pragma unroll
        for (int x = 0; x < NS; ++x) kf[x] = rd_b128<OFF + 16 * 2 * D * U>(rs[x]);
#pragma unroll
        for (int x = 0; x < NS; ++x) vf[x] = rd_b128<OFF + 16 * 2 * D * U + kTile>(rs[x]);
        if constexpr (NS == 4)
          GRAD_LGKM(4, "+v"(kf[0]), "+v"(kf[1]), "+v"(kf[2]), "+v"(kf[3]));
        else
          GRAD_LGKM(2, "+v"(kf[0]), "+v"(kf[1]));
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // dP - Delta from the product's start value
          s[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          g[i] = f32x4{-delta[i], -delta[i], -delta[i], -delta[i]};
        }
#pragma unroll
        for (int x = 0; x < NS; ++x)
#pragma unroll
          for (int i = 0; i < 2; ++i) s[i] = mfma16(kf[x], qf[i][x], s[i]);
        if constexpr (NS == 4)
          GRAD_LGKM(0, "+v"(vf[0]), "+v"(vf[1]), "+v"(vf[2]), "+v"(vf[3]));
        else
          GRAD_LGKM(0, "+v"(vf[0]), "+v"(vf[1]));
#pragma unroll
        for (int x = 0; x < NS; ++x)
#pragma unroll
          for (int i = 0; i < 2; ++i) g[i] = mfma16(vf[x], gf[i][x], g[i]);
        if (edge) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int64_t lim64 = (CAUSAL ? min(nkb, q0 + 16 * i + c16 + shift + 1) : nkb) - key0;
            const int lim = (int)max(min(lim64, (int64_t)kGT), (int64_t)-kGT) - 4 * kg - 32 * decltype(j_c)::value - 16 * U;
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (r >= lim) s[i][r] = -INFINITY;
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float d[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][r], a.scale_log2, -lse2[i]));
            d[r] = p * g[i][r];
          }
          ds[i][2 * U] = pack_bf16(d[0], d[1]);
          ds[i][2 * U + 1] = pack_bf16(d[2], d[3]);
        }
      };
      block(IC<0>{});
      block(IC<1>{});
      bf16x8 df[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 u = {ds[i][0], ds[i][1], ds[i][2], ds[i][3]};
        df[i] = __builtin_bit_cast(bf16x8, u);
      }
#pragma unroll
      for (int d = 0; d < ND; d += 4) {
        u32x2 t[8];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          t[2 * x] = rd_tr16<OFF>(ts[d + x]);
          t[2 * x + 1] = rd_tr16<OFF + 16 * 2 * D>(ts[d + x]);
        }
        GRAD_LGKM(0, "+v"(t[0]), "+v"(t[1]), "+v"(t[2]), "+v"(t[3]), "+v"(t[4]), "+v"(t[5]), "+v"(t[6]), "+v"(t[7]));
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int i = 0; i < 2; ++i) acc[d + x][i] = mfma16(frag2(t[2 * x], t[2 * x + 1]), df[i], acc[d + x][i]);
      }
    };
    half(IC<0>{});
    half(IC<1>{});
  };
  {
    int slot = 0;
    for (int st = st0; st < st1; ++st) {
      step(slot * kPair, slot == 0 ? BUFS - 1 : slot - 1, st);
      slot = slot == BUFS - 1 ? 0 : slot + 1;
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  // lane: query 16 i + c16, d = 16 db + 4 kg .. + 3
  if (unit.part >= 0) {
    float* o = a.part + (unit.slot * 32 * W + wv * 32 + c16) * D + 4 * kg;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (q0 + 16 * i + c16 >= a.nq) continue;
#pragma unroll
      for (int d = 0; d < ND; ++d) *(f32x4*)(o + 16 * i * D + 16 * d) = acc[d][i] * a.scale;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t qi = q0 + 16 * i + c16;
    if (qi >= a.nq) continue;
    uint16_t* o = a.dq + b * a.dq_s[0] + qi * a.dq_s[1] + (int64_t)h * a.dq_s[2] + 4 * kg;
#pragma unroll
    for (int d = 0; d < ND; ++d)
      *(uint2*)(o + 16 * d) = make_uint2(pack_bf16(acc[d][i][0] * a.scale, acc[d][i][1] * a.scale),
                                         pack_bf16(acc[d][i][2] * a.scale, acc[d][i][3] * a.scale));
  }
}

// ------------------------------------------------------------- dk and dv
// W waves of 32 keys (K and V in registers as B operands) over tiles of 64
// queries of every query head of the group. S = Q K^T and dP = dO V^T in
// 16 x 16 blocks (lane l: key l % 16, queries 4 (l / 16) + r), whose lse and
// Delta come from LDS, four queries a read; dv^T += dO^T P and dk^T += Q^T dS
// with the transposed tiles by transposing reads. 9216 x 9216, 32 heads of 128:
// 2242 us, 1241 TFLOP/s of its four products; 4099 x 4099 causal, 32 / 8 heads of
// 64: 170 us.
template <int D, int W, int BUFS, bool CAUSAL>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2))) void k_attn_dkv(
    AttnGradArgs a) {
  constexpr int kTile = kGT * D * 2, kPair = 2 * kTile + 512, NS = D / 32, ND = D / 16;
  constexpr int KB = 2, kKeys = 32 * W;
  typedef TileDma<D, W, true, D == 64 ? 2 : CAUSAL ? 0 : 1> Dma;
  __shared__ uint4 smem[BUFS * kPair / 16];
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const GradUnit unit = grad_unit<CAUSAL>(a, a.batch * a.kv_heads);
  const int kblk = unit.blk;
  const int64_t bh = unit.bh;
  const int hk = (int)(bh % a.kv_heads);
  const int64_t b = bh / a.kv_heads;
  const int c16 = lane & 15, kg = lane >> 4;
  const int64_t kblk0 = (int64_t)kblk * kKeys, k0 = kblk0 + wv * 32;
  const int64_t nkb = key_count(a, b);
  const int64_t shift = nkb - a.nq;
  const int nqt = (int)((a.nq + kGT - 1) / kGT);
  // Query tiles t0 .. nqt - 1 of each head; this part takes steps s0 .. s1 - 1
  // of the group's.
  int t0 = 0;
  if (CAUSAL) t0 = (int)min((int64_t)nqt, max((int64_t)0, kblk0 - shift) / kGT);
  if (kblk0 >= nkb) t0 = nqt;
  const int per = nqt - t0;
  const int64_t all = (int64_t)per * a.group;
  const int s0 = unit.part < 0 ? 0 : (int)(all * unit.part / a.ksplit);
  const int s1 = unit.part < 0 ? (int)all : (int)(all * (unit.part + 1) / a.ksplit);

  bf16x8 kf[KB][NS], vf[KB][NS];
  f32x4 dk[ND][KB], dv[ND][KB];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < KB; ++i) dk[d][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f}, dv[d][i] = dk[d][i];

  if (s1 > s0) {
#pragma unroll
    for (int i = 0; i < KB; ++i) {
      const int64_t ki = min(k0 + 16 * i + c16, nkb - 1);
      const uint16_t* kr = a.k + b * a.k_s[0] + ki * a.k_s[1] + (int64_t)hk * a.k_s[2] + 8 * kg;
      const uint16_t* vr = a.v + b * a.v_s[0] + ki * a.v_s[1] + (int64_t)hk * a.v_s[2] + 8 * kg;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        kf[i][s] = __builtin_bit_cast(bf16x8, *(const uint4*)(kr + 32 * s));
        vf[i][s] = __builtin_bit_cast(bf16x8, *(const uint4*)(vr + 32 * s));
      }
    }
    const uint16_t* qbase = a.q + b * a.q_s[0] + (int64_t)hk * a.group * a.q_s[2];
    const uint16_t* gbase = a.dout + b * a.do_s[0] + (int64_t)hk * a.group * a.do_s[2];
    const float* lbase = a.ld + (b * a.heads + (int64_t)hk * a.group) * nqt * 128;
    char* const lds = (char*)smem;
    Dma tiles;
    tiles.init((uint32_t)a.q_s[1], (uint32_t)a.do_s[1], wv, lane);
    // The next step to send: its head of the group and query tile (the last
    // one again past the end).
    int send_s = s0, send_g = s0 / per, send_t = t0 + s0 % per;
    auto dma = [&](int slot) {
      const int g = send_g, t = send_t;
      if (send_s + 1 < s1) {
        ++send_s;
        if (++send_t == nqt) send_t = t0, ++send_g;
      }
      const int64_t q0 = (int64_t)t * kGT;
      const int rows = (int)min((int64_t)kGT, a.nq - q0);
      char* const at = lds + slot * kPair;
      tiles.pair(qbase + g * a.q_s[2] + q0 * a.q_s[1], (uint32_t)a.q_s[1], gbase + g * a.do_s[2] + q0 * a.do_s[1],
                 (uint32_t)a.do_s[1], rows, at, wv, lane);
      // lse2 and Delta, 256 bytes each: even waves the one, odd waves the other
      int l = lane;
      asm volatile("" : "+v"(l));
      const uint32_t off = 4 * l;
      __builtin_amdgcn_global_load_lds(
          (const void*)((const char*)(lbase + ((int64_t)g * nqt + t) * 128 + (wv & 1) * 64) + off),
          (lds_void*)(at + 2 * kTile + (wv & 1) * 256), 4, 0, 0);
    };
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)smem;
    const uint32_t ra = lds0 + c16 * (2 * D) + ((kg ^ sw16<D>(c16)) << 4);
    const int a4 = lane & 3, j4 = (lane & 15) >> 2;
    const uint32_t ta = lds0 + (4 * kg + j4) * (2 * D) + (((a4 >> 1) ^ sw16<D>(4 * kg + j4)) << 4) + (a4 & 1) * 8;

    auto step = [&](uint32_t base, int slot2, int first, bool last) {
      ring_wait<BUFS == 3 ? 2 * Dma::kDI + 1 : 0>();
      if (BUFS == 3 || !last) dma(slot2);
      if (k0 >= nkb || (CAUSAL && first >= kGT)) return;  // no key here, or none that the tile's queries see
      auto half = [&](auto j_c) {  // queries 32 j .. + 31 of the tile
        constexpr int J = decltype(j_c)::value, OFF = 32 * 2 * D * J;
        uint32_t pp[KB][4], ds[KB][4];  // P and dS, B operands: key block i
        auto block = [&](auto u_c) {  // queries 16 u .. + 15 of these
          constexpr int U = decltype(u_c)::value;
          const uint32_t r0 = here(ra, base);
          constexpr int OQ = OFF + 16 * 2 * D * U, OG = OQ + kTile, OL = (32 * J + 16 * U) * 4;
          f32x4 s[KB], g[KB];
#pragma unroll
          for (int i = 0; i < KB; ++i) s[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          // two pairs of fragments in flight, each read under the other's MFMAs
          bf16x8 x0, x1, y0, y1, dr;
          auto mul = [&](f32x4(&c)[KB], const bf16x8& u, const bf16x8& v, const bf16x8(&w)[KB][NS], auto n_c) {
            constexpr int N = decltype(n_c)::value;
#pragma unroll
            for (int i = 0; i < KB; ++i) c[i] = mfma16(u, w[i][N], c[i]);
#pragma unroll
            for (int i = 0; i < KB; ++i) c[i] = mfma16(v, w[i][N + 1], c[i]);
          };
          const uint32_t l0 = (here(lane, 0) & ~15u) + lds0 + 2 * kTile + base;  // 16 kg
          // dP - Delta from the product's start value (subtracted after it
          // where -Delta would be one register too many)
          constexpr bool kStart = D == 64 || !CAUSAL;
          auto start = [&] {
#pragma unroll
            for (int i = 0; i < KB; ++i) g[i] = kStart ? __builtin_bit_cast(f32x4, dr) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          };
          x0 = rd_b128<OQ>(r0);
          x1 = rd_b128<OQ>(r0 ^ 64);
          if constexpr (NS == 4) {
            y0 = rd_b128<OQ>(r0 ^ 128);
            y1 = rd_b128<OQ>(r0 ^ 192);
            GRAD_LGKM(2, "+v"(x0), "+v"(x1));
            mul(s, x0, x1, kf, IC<0>{});
            if constexpr (kStart) dr = rd_b128<OL + 256>(l0);
            x0 = rd_b128<OG>(r0);
            x1 = rd_b128<OG>(r0 ^ 64);
            if constexpr (kStart)
              GRAD_LGKM(3, "+v"(y0), "+v"(y1));
            else
              GRAD_LGKM(2, "+v"(y0), "+v"(y1));
            mul(s, y0, y1, kf, IC<2 % NS>{});
            y0 = rd_b128<OG>(r0 ^ 128);
            y1 = rd_b128<OG>(r0 ^ 192);
            if constexpr (kStart)
              GRAD_LGKM(2, "+v"(x0), "+v"(x1), "+v"(dr));
            else
              GRAD_LGKM(2, "+v"(x0), "+v"(x1));
            start();
            mul(g, x0, x1, vf, IC<0>{});
            x0 = rd_b128<OL>(l0);
            if constexpr (!kStart) dr = rd_b128<OL + 256>(l0);
            if constexpr (kStart)
              GRAD_LGKM(1, "+v"(y0), "+v"(y1));
            else
              GRAD_LGKM(2, "+v"(y0), "+v"(y1));
            mul(g, y0, y1, vf, IC<2 % NS>{});
          } else {
            dr = rd_b128<OL + 256>(l0);
            y0 = rd_b128<OG>(r0);
            y1 = rd_b128<OG>(r0 ^ 64);
            GRAD_LGKM(3, "+v"(x0), "+v"(x1));
            mul(s, x0, x1, kf, IC<0>{});
            x0 = rd_b128<OL>(l0);
            GRAD_LGKM(1, "+v"(y0), "+v"(y1), "+v"(dr));
            start();
            mul(g, y0, y1, vf, IC<0>{});
          }
          if constexpr (kStart)
            GRAD_LGKM(0, "+v"(x0));
          else
            GRAD_LGKM(0, "+v"(x0), "+v"(dr));
          const f32x4 lse2 = __builtin_bit_cast(f32x4, x0);
          // (D 128 compares in every tile: behind a uniform branch the scores
          // cost more registers than there are)
          if (CAUSAL && (D == 128 || first + 16 * KB - 1 > 0)) {
#pragma unroll
            for (int i = 0; i < KB; ++i) {
              const int l = (int)here(lane, 0);
              const int low = first + 16 * i + (l & 15) - 4 * (l >> 4) - 32 * J - 16 * U;
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (r < low) s[i][r] = -INFINITY;
            }
          }
#pragma unroll
          for (int i = 0; i < KB; ++i) {
            float p[4], d[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][r], a.scale_log2, -lse2[r]));
              d[r] = p[r] * (kStart ? g[i][r] : g[i][r] + __builtin_bit_cast(f32x4, dr)[r]);
            }
            pp[i][2 * U] = pack_bf16(p[0], p[1]);
            pp[i][2 * U + 1] = pack_bf16(p[2], p[3]);
            ds[i][2 * U] = pack_bf16(d[0], d[1]);
            ds[i][2 * U + 1] = pack_bf16(d[2], d[3]);
          }
        };
        __builtin_amdgcn_sched_barrier(0);
        block(IC<0>{});
        __builtin_amdgcn_sched_barrier(0);
        block(IC<1>{});
        __builtin_amdgcn_sched_barrier(0);
        bf16x8 pf[KB], df[KB];
#pragma unroll
        for (int i = 0; i < KB; ++i) {
          const uint4 u = {pp[i][0], pp[i][1], pp[i][2], pp[i][3]}, w = {ds[i][0], ds[i][1], ds[i][2], ds[i][3]};
          pf[i] = __builtin_bit_cast(bf16x8, u);
          df[i] = __builtin_bit_cast(bf16x8, w);
        }
#pragma unroll
        for (int d = 0; d < ND; d += 2) {
          const uint32_t w0 = here(ta, base);
          u32x2 x[4], y[4];  // dO^T and Q^T of two 16-wide d-blocks
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            x[2 * z] = rd_tr16<OFF + kTile>(w0 ^ ((d + z) << 5));
            x[2 * z + 1] = rd_tr16<OFF + kTile + 16 * 2 * D>(w0 ^ ((d + z) << 5));
          }
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            y[2 * z] = rd_tr16<OFF>(w0 ^ ((d + z) << 5));
            y[2 * z + 1] = rd_tr16<OFF + 16 * 2 * D>(w0 ^ ((d + z) << 5));
          }
          GRAD_LGKM(4, "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
#pragma unroll
          for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int i = 0; i < KB; ++i) dv[d + z][i] = mfma16(frag2(x[2 * z], x[2 * z + 1]), pf[i], dv[d + z][i]);
          GRAD_LGKM(0, "+v"(y[0]), "+v"(y[1]), "+v"(y[2]), "+v"(y[3]));
#pragma unroll
          for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int i = 0; i < KB; ++i) dk[d + z][i] = mfma16(frag2(y[2 * z], y[2 * z + 1]), df[i], dk[d + z][i]);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      half(IC<0>{});
      half(IC<1>{});
    };
    int t = t0 + s0 % per;  // this step's query tile
    dma(0);
    if (BUFS == 3) dma(1);
    int slot = 0;
    for (int st = s0; st < s1; ++st) {
      // causal: key k is hidden from query q where k - shift > q; `first` is
      // that of this wave's first key against the tile's first query
      const int64_t first = k0 - shift - (int64_t)t * kGT;
      step(slot * kPair, slot == 0 ? BUFS - 1 : slot - 1, (int)max(min(first, (int64_t)2 * kGT), (int64_t)-2 * kGT),
           st + 1 == s1);
      if (++t == nqt) t = t0;
      slot = slot == BUFS - 1 ? 0 : slot + 1;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  // lane: key 16 i + c16, d = 16 db + 4 kg .. + 3; keys behind the sequence: 0
#pragma unroll
  for (int i = 0; i < KB; ++i) {
    const int64_t ki = k0 + 16 * i + c16;
    if (ki >= a.nk) continue;
    const bool live = ki < nkb;
    if (unit.part >= 0) {
      float* o = a.part + (unit.slot * kKeys + wv * 32 + 16 * i + c16) * 2 * D + 4 * kg;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        *(f32x4*)(o + 16 * d) = live ? dk[d][i] * a.scale : zero;
        *(f32x4*)(o + D + 16 * d) = live ? dv[d][i] : zero;
      }
      continue;
    }
    uint16_t* ok = a.dk + b * a.dk_s[0] + ki * a.dk_s[1] + (int64_t)hk * a.dk_s[2] + 4 * kg;
    uint16_t* ov = a.dv + b * a.dv_s[0] + ki * a.dv_s[1] + (int64_t)hk * a.dv_s[2] + 4 * kg;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const f32x4 x = dk[d][i] * a.scale, y = dv[d][i];
      const uint2 none = make_uint2(0, 0);
      *(uint2*)(ok + 16 * d) = live ? make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])) : none;
      *(uint2*)(ov + 16 * d) = live ? make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])) : none;
    }
  }
}

// The gradients of the blocks that ran in parts, added in part order; 8 values
// a thread (2 x 2304 x 256: 75 MB in 12.7 us). Side 0: dq (rows of D), side 1: dk and dv (rows of 2 D).
struct GradJoin {
  const float* part;
  uint16_t *o, *o2;
  int64_t s[3], s2[3];
  int64_t nfull, n;  // blocks run whole, rows of the tensor
  int ksplit, blocks, rows, heads, causal;
  int64_t units;     // threads
};
struct GradJoins {
  GradJoin side[2];
  int64_t blocks0;   // workgroups of side 0
};
template <int D>
__global__ __launch_bounds__(256) void k_attn_grad_join(GradJoins a) {
  const bool second = (int64_t)blockIdx.x >= a.blocks0;
  const GradJoin& j = second ? a.side[1] : a.side[0];
  const int64_t i = ((int64_t)blockIdx.x - (second ? a.blocks0 : 0)) * 256 + threadIdx.x;
  if (i >= j.units) return;
  const int width = second ? 2 * D : D;
  const int64_t r = i / (width / 8);
  int c = 8 * (int)(i - r * (width / 8));
  const int64_t blk = r / j.rows, wg = j.nfull + blk, row = r - blk * j.rows;
  int b8 = (int)(wg % j.blocks);
  if (j.causal) b8 = j.blocks - 1 - b8;
  const int64_t at = (int64_t)b8 * j.rows + row;
  if (at >= j.n) return;
  const int64_t bh = wg / j.blocks, b = bh / j.heads, h = bh - b * j.heads;
  const float* f = j.part + (blk * j.ksplit * j.rows + row) * width + c;
  float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  const int64_t step = (int64_t)j.rows * width;
  for (int p0 = 0; p0 < j.ksplit; p0 += 8) {  // eight parts' loads in flight
    float4 u[8], v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float* g = f + min(p0 + e, j.ksplit - 1) * step;
      u[e] = *(const float4*)g, v[e] = *(const float4*)(g + 4);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (p0 + e >= j.ksplit) break;
      s[0] += u[e].x, s[1] += u[e].y, s[2] += u[e].z, s[3] += u[e].w;
      s[4] += v[e].x, s[5] += v[e].y, s[6] += v[e].z, s[7] += v[e].w;
    }
  }
  const bool two = c >= D;
  if (two) c -= D;
  uint16_t* o = two ? j.o2 + b * j.s2[0] + at * j.s2[1] + h * j.s2[2] : j.o + b * j.s[0] + at * j.s[1] + h * j.s[2];
  *(uint4*)(o + c) = pack8(s);
}

// -------------------------------------------------------------------- host
static int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

// Which of a kernel's blocks run whole, and the parts of the others.
struct GradPlan {
  int64_t blocks, nfull;
  int ksplit;
  int64_t units() const { return nfull + (blocks - nfull) * ksplit; }
  int64_t parts() const { return units() - nfull; }
};
// `blocks` blocks of `steps` steps each (step_us) run `slots` at a time; with
// `fill` < 1 (causal) a block has any number of steps up to that, this share of
// them on average. Candidates: all whole; all in k parts; with equal blocks
// the last, partial round in k parts. A part costs its own start (fixed_us; a
// whole block of an only round has it too) and part_bytes written and read back
// by a join, whose chain of loads grows with k (4 x 8 heads of 128, one query
// each, 577 keys: lse and join 15.1 us whole, 13.1 in 2 parts, 10.6 in 5, 11.6
// in 10).
static GradPlan grad_plan(int64_t blocks, int64_t steps, int64_t slots, double step_us, double part_bytes,
                          double fill) {
  const double fixed_us = 4.0, join_us = 3.0, join_part_us = 0.35, bytes_per_us = 4e6;
  GradPlan best = {blocks, blocks, 1};
  const bool equal = fill >= 1.0;
  const int64_t whole = equal ? blocks / slots * slots : 0, rest = blocks - whole;
  if (!rest || steps < 2) return best;
  double least = 1e30;
  for (int k = 1; k <= kMaxParts && k <= steps; ++k) {
    const double part = (double)((steps + k - 1) / k) * step_us + (k > 1 || !whole ? fixed_us : 0.0);
    double us = equal ? (double)((rest * k + slots - 1) / slots) * part
                      : max(part, (double)(rest * k) / slots * (fill * part) + 0.5 * part);
    if (k > 1) us += join_us + k * join_part_us + 2.0 * rest * k * part_bytes / bytes_per_us;
    if (us < least) least = us, best = {blocks, k == 1 ? blocks : whole, k};
  }
  return best;
}
// The share of the scores that a causal mask leaves.
static double causal_fill(const AttnGradArgs& a) {
  if (!a.causal) return 1.0;
  return a.nk >= a.nq ? 1.0 - 0.5 * a.nq / a.nk : 0.5 * a.nk / a.nq;
}

// The forms of the three kernels: many steps run 8 waves and three tile pairs
// in one workgroup per CU (D 128); few, or few rows, 4 waves and two pairs in
// two, one's loads and stores under the other's products. lse / dq / dkv with
// joins, 32 heads of 128, us, few against many: 1024 x 1024 27 / 40 / 51 against
// 35 / 38 / 78, 2048 x 2048 causal 54 / 76 / 122 against 62 / 90 / 134, 2304 x
// 2304 111 / 143 / 202 against 111 / 149 / 214, 4096 x 4096 286 / 384 / 513
// against 265 / 370 / 516, 128 x 4096 30 / 29 / 49 against 30 / 29 / 57; two
// sequences of 2304 x 256 39 / 62 / 73 against 46 / 74 / 65.
static bool few_steps(int64_t own_rows, int64_t other_rows) { return other_rows <= 32 * kGT || own_rows <= 128; }
static int grad_waves(int64_t head_dim, bool few) { return head_dim == 64 || few ? 4 : 8; }
static int64_t grad_slots(int64_t head_dim, bool few, int per_cu64) {
  return (int64_t)cu_count() * (head_dim == 64 ? per_cu64 : few ? 2 : 1);
}

static GradPlan rows_plan(const AttnGradArgs& a, int64_t d, bool dq) {
  const bool few = few_steps(a.nq, a.nk);
  const int rows = 32 * grad_waves(d, few);
  const int64_t blocks = a.batch * a.heads * ((a.nq + rows - 1) / rows);
  const double step = (dq ? 2.6 : 1.8) * (d == 64 || few ? 0.6 : 1.0);
  return grad_plan(blocks, (a.nk + kGT - 1) / kGT, grad_slots(d, few, 3), step,
                   min((int64_t)rows, a.nq) * (d + (dq ? 0 : 2)) * 4.0, causal_fill(a));
}
static bool few_query_steps(const AttnGradArgs& a) { return few_steps(a.nk, a.nq * a.group); }
static GradPlan keys_plan(const AttnGradArgs& a, int64_t d) {
  const bool few = few_query_steps(a);
  const int rows = 32 * grad_waves(d, few);
  const int64_t blocks = a.batch * a.kv_heads * ((a.nk + rows - 1) / rows);
  return grad_plan(blocks, (a.nq + kGT - 1) / kGT * a.group, grad_slots(d, few, 3),
                   3.5 * (d == 64 || few ? 0.6 : 1.0), min((int64_t)rows, a.nk) * d * 8.0, causal_fill(a));
}

// The offsets of a tile's rows are 32-bit; with one query a sequence, the
// heads are its rows.
static bool grad_strides(const void* p, const int64_t* s, int64_t tokens, bool heads_are_rows = false) {
  if (!p || !aligned(p, 16)) return false;
  for (int i = 0; i < 3; ++i)
    if (s[i] % 8) return false;
  if (heads_are_rows && (s[2] < 0 || s[2] >= (1 << 24))) return false;
  return tokens <= 1 || (s[1] >= 0 && s[1] < (1 << 24));
}

static void gset3(int64_t* d, const int64_t* s) { d[0] = s[0], d[1] = s[1], d[2] = s[2]; }

// Shape checks; a single query per sequence sees every valid key, causal or
// not, so the query heads of a key head become the queries of one.
static int grad_shape(AttnGradArgs& a, int64_t batch, int64_t nq, int64_t nk, int64_t heads, int64_t kv_heads,
                      int64_t head_dim, float scale, int causal, const int32_t* k_lens) {
  if (head_dim != 64 && head_dim != 128) return unsupported("head_dim %lld", (long long)head_dim);
  if (batch < 1 || nq < 1 || nk < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads)
    return fail("shape (%lld, %lld, %lld, %lld, %lld)", (long long)batch, (long long)nq, (long long)nk,
                (long long)heads, (long long)kv_heads);
  if (nq > (1 << 30) || nk > (1 << 30) || heads > (1 << 20) || batch > (1 << 20))
    return unsupported("shape (%lld, %lld, %lld, %lld)", (long long)batch, (long long)nq, (long long)nk, (long long)heads);
  // a grid holds less than 2^32 threads: 256 for 128 rows
  if (batch * heads * ((nq + 127) / 128) >= 1 << 24 || batch * kv_heads * ((nk + 127) / 128) >= 1 << 24)
    return unsupported("more than 2^24 blocks of 128 rows");
  if ((nq + kGT - 1) / kGT * (heads / kv_heads) > INT32_MAX / 64) return unsupported("too many queries per key head");
  if (!(scale > 0.0f) || scale > 1e30f) return fail("softmax scale");
  if (!aligned(k_lens, 4)) return fail("k_lens alignment");
  a.batch = batch, a.nq = nq, a.nk = nk;
  a.heads = (int)heads, a.kv_heads = (int)kv_heads, a.group = (int)(heads / kv_heads);
  a.scale = scale, a.scale_log2 = scale * kLog2e;
  a.causal = causal ? 1 : 0;
  a.k_lens = k_lens;
  if (nq == 1) {
    a.nq = a.group, a.heads = a.kv_heads, a.group = 1;
    a.causal = 0;
  }
  return OGA_OK;
}
// Strides of q, o, dout or dq under that view.
static void query_strides(const AttnGradArgs& a, bool one_query, int64_t* d, const int64_t* s) {
  gset3(d, s);
  if (one_query) d[1] = s[2], d[2] = s[2] * a.nq;  // (a.nq: the group)
}

// Workspaces: forward [parts of O | m, l]; backward [lse2 and Delta | parts of
// dq | parts of dk and dv].
struct GradSpace {
  GradPlan rows, keys;
  int64_t ml, dq, dkv, total;
};
static GradSpace fwd_space(const AttnGradArgs& a, int64_t d) {
  GradSpace w = {};
  w.rows = rows_plan(a, d, false);
  const int64_t rows = w.rows.parts() * 32 * grad_waves(d, few_steps(a.nq, a.nk));
  w.ml = align256(rows * d * 4);
  w.total = rows ? w.ml + align256(rows * 8) : 0;
  return w;
}
static GradSpace bwd_space(const AttnGradArgs& a, int64_t d) {
  GradSpace w = {};
  w.rows = rows_plan(a, d, true);
  w.keys = keys_plan(a, d);
  w.dq = align256(a.batch * a.heads * ((a.nq + kGT - 1) / kGT) * 128 * 4);
  w.dkv = w.dq + align256(w.rows.parts() * 32 * grad_waves(d, few_steps(a.nq, a.nk)) * d * 4);
  w.total = w.dkv + align256(w.keys.parts() * 32 * grad_waves(d, few_query_steps(a)) * d * 8);
  return w;
}

template <int D, int W, int BUFS>
static void lse_launch(AttnGradArgs& a, const GradPlan& p, hipStream_t s) {
  a.blocks = (int)((a.nq + 32 * W - 1) / (32 * W));
  a.nfull = p.nfull, a.ksplit = p.ksplit;
  const dim3 grid((unsigned)p.units()), block(64 * W);
  if (a.causal)
    k_attn_lse<D, W, BUFS, true><<<grid, block, 0, s>>>(a);
  else
    k_attn_lse<D, W, BUFS, false><<<grid, block, 0, s>>>(a);
  if (p.parts()) {
    const int64_t rows = (p.blocks - p.nfull) * 32 * W, per = 256 / (D / 8);
    k_attn_lse_join<D, 32 * W><<<dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, s>>>(a);
  }
}

template <int D, int W, int BUFS>
static GradJoin dq_launch(AttnGradArgs a, const GradPlan& p, hipStream_t s) {
  a.blocks = (int)((a.nq + 32 * W - 1) / (32 * W));
  a.nfull = p.nfull, a.ksplit = p.ksplit;
  const dim3 grid((unsigned)p.units()), block(64 * W);
  if (a.causal)
    k_attn_dq<D, W, BUFS, true><<<grid, block, 0, s>>>(a);
  else
    k_attn_dq<D, W, BUFS, false><<<grid, block, 0, s>>>(a);
  GradJoin j = {a.part, a.dq, nullptr, {}, {}, p.nfull, a.nq, p.ksplit, a.blocks, 32 * W, a.heads, a.causal,
                (p.blocks - p.nfull) * 32 * W * (D / 8)};
  gset3(j.s, a.dq_s);
  return j;
}

template <int D, int W, int BUFS>
static GradJoin dkv_launch(AttnGradArgs a, const GradPlan& p, hipStream_t s) {
  a.blocks = (int)((a.nk + 32 * W - 1) / (32 * W));
  a.nfull = p.nfull, a.ksplit = p.ksplit;
  const dim3 grid((unsigned)p.units()), block(64 * W);
  if (a.causal)
    k_attn_dkv<D, W, BUFS, true><<<grid, block, 0, s>>>(a);
  else
    k_attn_dkv<D, W, BUFS, false><<<grid, block, 0, s>>>(a);
  GradJoin j = {a.part, a.dk, a.dv, {}, {}, p.nfull, a.nk, p.ksplit, a.blocks, 32 * W, a.kv_heads, 0,
                (p.blocks - p.nfull) * 32 * W * (2 * D / 8)};
  gset3(j.s, a.dk_s), gset3(j.s2, a.dv_s);
  return j;
}

template <int D>
static void bwd_launch(AttnGradArgs& a, const GradSpace& w, char* ws, hipStream_t s) {
  a.ld = (float*)ws;
  const bool few_q = few_steps(a.nq, a.nk), few_k = few_query_steps(a);
  GradJoins j = {};
  a.part = (float*)(ws + w.dq);
  if constexpr (D == 64) {
    j.side[0] = dq_launch<D, 4, 3>(a, w.rows, s);
  } else {
    j.side[0] = few_q ? dq_launch<D, 4, 2>(a, w.rows, s) : dq_launch<D, 8, 3>(a, w.rows, s);
  }
  a.part = (float*)(ws + w.dkv);
  if constexpr (D == 64) {
    j.side[1] = dkv_launch<D, 4, 3>(a, w.keys, s);
  } else {
    j.side[1] = few_k ? dkv_launch<D, 4, 2>(a, w.keys, s) : dkv_launch<D, 8, 3>(a, w.keys, s);
  }
  j.blocks0 = (j.side[0].units + 255) / 256;
  const int64_t grid = j.blocks0 + (j.side[1].units + 255) / 256;
  if (grid) k_attn_grad_join<D><<<dim3((unsigned)grid), dim3(256), 0, s>>>(j);
}

}  // namespace oga

using namespace oga;

extern "C" int64_t oga_attention_lse_workspace_bytes(int64_t batch, int64_t nq, int64_t nk, int64_t heads,
                                                     int64_t kv_heads, int64_t head_dim, int causal) {
  AttnGradArgs a = {};
  if (grad_shape(a, batch, nq, nk, heads, kv_heads, head_dim, 1.0f, causal, nullptr)) return 0;
  return fwd_space(a, head_dim).total;
}

extern "C" int oga_attention_lse(const void* q, const int64_t q_strides[3], const void* k, const int64_t k_strides[3],
                                 const void* v, const int64_t v_strides[3], void* o, const int64_t o_strides[3],
                                 float* lse, int64_t batch, int64_t nq, int64_t nk, int64_t heads, int64_t kv_heads,
                                 int64_t head_dim, float softmax_scale, int causal, const int32_t* k_lens,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  AttnGradArgs a = {};
  if (int rc = grad_shape(a, batch, nq, nk, heads, kv_heads, head_dim, softmax_scale, causal, k_lens)) return rc;
  if (!grad_strides(q, q_strides, nq, nq == 1) || !grad_strides(k, k_strides, nk) || !grad_strides(v, v_strides, nk) ||
      !grad_strides(o, o_strides, nq, nq == 1) || !lse || !aligned(lse, 4))
    return fail("operand layout");
  const GradSpace w = fwd_space(a, head_dim);
  if (w.total && (!workspace || !aligned(workspace, 256) || workspace_bytes < w.total))
    return fail("workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)w.total);
  a.q = (const uint16_t*)q, a.k = (const uint16_t*)k, a.v = (const uint16_t*)v, a.o = (uint16_t*)o, a.lse = lse;
  query_strides(a, nq == 1, a.q_s, q_strides), query_strides(a, nq == 1, a.o_s, o_strides);
  gset3(a.k_s, k_strides), gset3(a.v_s, v_strides);
  a.part = (float*)workspace, a.part_ml = (float*)((char*)workspace + w.ml);
  const hipStream_t s = (hipStream_t)stream;
  if (head_dim == 64)
    lse_launch<64, 4, 3>(a, w.rows, s);
  else if (few_steps(a.nq, a.nk))
    lse_launch<128, 4, 2>(a, w.rows, s);
  else
    lse_launch<128, 8, 3>(a, w.rows, s);
  return launch_status();
}

extern "C" int64_t oga_attention_bwd_workspace_bytes(int64_t batch, int64_t nq, int64_t nk, int64_t heads,
                                                     int64_t kv_heads, int64_t head_dim, int causal) {
  AttnGradArgs a = {};
  if (grad_shape(a, batch, nq, nk, heads, kv_heads, head_dim, 1.0f, causal, nullptr)) return 0;
  return bwd_space(a, head_dim).total;
}

extern "C" int oga_attention_bwd(const void* dout, const int64_t do_strides[3], const void* q,
                                 const int64_t q_strides[3], const void* k, const int64_t k_strides[3], const void* v,
                                 const int64_t v_strides[3], const void* out, const int64_t o_strides[3],
                                 const float* lse, void* dq, const int64_t dq_strides[3], void* dk,
                                 const int64_t dk_strides[3], void* dv, const int64_t dv_strides[3], int64_t batch,
                                 int64_t nq, int64_t nk, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                 float softmax_scale, int causal, const int32_t* k_lens, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  AttnGradArgs a = {};
  if (int rc = grad_shape(a, batch, nq, nk, heads, kv_heads, head_dim, softmax_scale, causal, k_lens)) return rc;
  if (!grad_strides(dout, do_strides, nq, nq == 1) || !grad_strides(q, q_strides, nq, nq == 1) || !grad_strides(k, k_strides, nk) ||
      !grad_strides(v, v_strides, nk) || !grad_strides(out, o_strides, nq, nq == 1) || !grad_strides(dq, dq_strides, nq, nq == 1) ||
      !grad_strides(dk, dk_strides, nk) || !grad_strides(dv, dv_strides, nk) || !lse || !aligned(lse, 4))
    return fail("operand layout");
  const GradSpace w = bwd_space(a, head_dim);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < w.total)
    return fail("workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)w.total);
  a.dout = (const uint16_t*)dout, a.q = (const uint16_t*)q, a.k = (const uint16_t*)k, a.v = (const uint16_t*)v;
  a.out = (const uint16_t*)out, a.lse = const_cast<float*>(lse);
  a.dq = (uint16_t*)dq, a.dk = (uint16_t*)dk, a.dv = (uint16_t*)dv;
  query_strides(a, nq == 1, a.do_s, do_strides), query_strides(a, nq == 1, a.q_s, q_strides);
  query_strides(a, nq == 1, a.o_s, o_strides), query_strides(a, nq == 1, a.dq_s, dq_strides);
  gset3(a.k_s, k_strides), gset3(a.v_s, v_strides), gset3(a.dk_s, dk_strides), gset3(a.dv_s, dv_strides);
  if (head_dim == 128)
    bwd_launch<128>(a, w, (char*)workspace, (hipStream_t)stream);
  else
    bwd_launch<64>(a, w, (char*)workspace, (hipStream_t)stream);
  return launch_status();
}
