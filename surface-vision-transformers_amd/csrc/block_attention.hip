// sitk attention over key blocks that a cheap score selects for each query (heads of 64 features, dense attention: attention.hip).
//   pool, select: block_select.hip;   attend: softmax(scale q K^T) V over the valid keys of the row's blocks; forward, dQ, dK / dV
// A row is one (token, head of the group): the G = H / Hk query heads that share a key head are R = Nq G rows beside each other, so
// shared heads fill the matrix tiles and their gradients add up inside one kernel.  The selection travels as bits, 64 rows to a word.
//   query side (forward, dQ): 64 rows visit the blocks that any of them selected -- neighbouring patches select alike -- and mask the
//     rest by their own bit; a wave whose 16 rows all skip a block skips its products.
//   key side (dK, dV): the rows that selected the block are gathered, so the products run on full tiles whatever the selection.
// Masked keys (key_mask, the tail of the last tile) never enter: their K and V rows are staged as zeros and their scores replaced, so
// whatever they hold (NaN, infinities) stays out.  Nor does a row see what K and V hold in a block that it did not select.
//
// 16-bit kernels: K / V (key side: Q / dO) tiles of 64 rows through an LDS-DMA ring, fragments and products as in attention.hip.  The
// waits, not one unit, bound them (matrix pipe busy 38 % and vector issue 30 % of dQ's time, half of a wave's time spent waiting), so
// the ring is as short as lets another workgroup onto the CU: forward two stages (four workgroups a CU), dQ three (three), key
// side two (two: 203 registers).  Where one workgroup per 64 rows leaves the card empty (single queries), the forward pass splits a
// row tile's keys over up to 16 workgroups and joins them in order.
// What 64 rows visit over what one row selects: 1.3 at 32 x 1281 tokens, top 8 of 21 blocks; 2.3 at 5121, 12 of 81; 3.6 at 20481, 16 of 321 (a
// wave's 16 rows 1.2, 1.8, 2.5) -- the price of tiles, paid on the query side only.  Smaller tiles would read K and V more often from L2;
// 32 rows a wave, 128 a workgroup, leave two workgroups a CU (forward at 32 x 1281 tokens 107 us where this took 84).
// Measured, bf16, 6 heads (means of 150 calls): 32 x 1281 forward 80 us, dQ 110, dK / dV 128 (useful work 400, 440 and 500 TFLOP/s); 2 x 20481 forward
// 297, dQ 424, dK / dV 241 (215, 230, 530).  16 single queries over 20481 keys, 12 heads on 3, top 16 of 161 blocks of 128: 14 us + join 5.
// Scores, maxima, sums and accumulators are 32 bits.  P and dS are rounded to the operands' 16 bits once, for the second product (it has no
// 32-bit operands); the row sum l adds P before that rounding, so lse stays a 32-bit value.
// f32 (the verification mode): one plain tiled kernel per direction.
#include <type_traits>

#include "block_common.h"

namespace sitk {

// Where few rows meet a key, a few of them make up its gradient, and errors of single entries do not average out (dK of 2 to 200 rows 1.5 to
// 2.2 times as far off as by its own rounding).  Up to this many query rows per key head dQ's kernel therefore also sums dS before its
// rounding, which is rowsum(dO o) of the exact o less that of the rounded one, and hands the exact one on; and dK and dV are taken
// from P and dS as sums of two 16-bit values: both then as exact as their own rounding, and dK of a row with one key is zero.
// Backward of 32 x 321 tokens, 6 heads, bf16: 63 us without, 70 with; with 1000 rows the gradients are 1.4 times as far off without it.
// The rule asks for the rows of the key head, not of a block: dQ's kernel hands delta on before anyone has counted who selected a block, and the exact
// delta for any number of rows costs more than it gives (2 x 20481 tokens: backward 656 us, 821 with it, 877 with P and dS of two values
// too).  So a block that few of more than 512 rows select has its gradients off like any other of that call: r.m.s. error over that of their own
// rounding dk 1.5 to 1.6, dv 1.3 to 1.7 for 2 to 2000 rows of 2048 (a single row: up to 2.3), 1.0 within the rule.
constexpr int BLK_FINE_ROWS = 512;
constexpr int BLK_LIST = 384;        // key tiles of the short list: with it three workgroups' LDS fit a CU

struct BlkAttn {
  const void *q, *k, *v, *o, *d_o;
  void *out, *dk, *dv;               // out: o (forward), dq; contiguous (B, N, heads, 64)
  Rows qs, ks, vs, os, dos;
  const uint64_t* mask;              // [bh][rt][j]; behind it [bh][j][rt]
  const uint64_t* kbits;
  float* lse;                        // (B, H, Nq)
  float *stat, *delta;               // backward, (B Hk, Rp): lse / scale, rowsum(dO o)
  float* part;                       // forward over parts of the tiles: per (part, row) 64 sums, then maximum, then sum
  int parts;
  float scale;
  BlkShape s;
};

__device__ u32x4 g_blk_zero[8];      // 128 bytes of zeros: rows that must not enter come from here
__device__ float g_blk_inf[64] = {
#define SITK_INF8 INFINITY, INFINITY, INFINITY, INFINITY, INFINITY, INFINITY, INFINITY, INFINITY
    SITK_INF8, SITK_INF8, SITK_INF8, SITK_INF8, SITK_INF8, SITK_INF8, SITK_INF8, SITK_INF8
#undef SITK_INF8
};

// ------------------------------------------------------------------------------------------
// the key tiles that any of 64 rows selected, ascending, with the rows' bits and the valid-key bits; tiles without a valid key are out
// ------------------------------------------------------------------------------------------
template <int CAP>
struct TileList {
  uint64_t rows[CAP];
  uint16_t tile[CAP];
  int found[4];
};
template <int CAP>
SITK_DEV int build_list(TileList<CAP>& l, const uint64_t* __restrict__ sel, const uint64_t* __restrict__ kbits, const BlkShape& s, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
  int n = 0;
  for (int t0 = 0; t0 < s.nt; t0 += 256) {
    const int t = t0 + tid;
    const uint64_t rows = t < s.nt ? sel[s.c == 1 ? t : t / s.c] : 0;
    const bool in = rows && kbits[t] != 0;
    const uint64_t hit = __ballot(in);
    __syncthreads();                                          // found[] of the last round has been read
    if (lane == 0) l.found[wave] = __popcll(hit);
    __syncthreads();
    int at = n;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) at += l.found[w];
      n += l.found[w];
    }
    if (in) {
      at += __popcll(hit & ((1ull << lane) - 1));
      l.rows[at] = rows;
      l.tile[at] = (uint16_t)t;
    }
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(n);
}
SITK_DEV uint64_t uniform64(uint64_t v) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
}
SITK_DEV bool bit64(uint64_t v, int i) { return v >> i & 1; }

struct RowTile {
  int rt, bh, hk, b;
};
SITK_DEV RowTile row_tile(const BlkShape& s, int L) {
  const int rt = L % s.nrt, bh = L / s.nrt;
  return RowTile{rt, bh, bh % s.Hk, bh / s.Hk};
}

// a row's unnormalised sums over one part of its tiles; begun == false (l == 0): the part holds no block of the row
SITK_DEV void store_part(const BlkAttn& a, int part, int bh, int r, int fq, const f32x4 (&o)[4], float m, float l) {
  const int64_t rows = (int64_t)a.s.B * a.s.Hk * a.s.Rp, row = (int64_t)part * rows + (int64_t)bh * a.s.Rp + r;
  float* p = a.part + row * 64;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) store4(p + 16 * dt + 4 * fq, o[dt]);
  if (fq == 0) {
    float* ml = a.part + (int64_t)a.parts * rows * 64;
    ml[row] = m;
    ml[(int64_t)a.parts * rows + row] = l;
  }
}

// ------------------------------------------------------------------------------------------
// plain tiles of 64 rows x 64 keys: f32, and 16-bit row tiles in which an infinity or a NaN has shown
// ------------------------------------------------------------------------------------------
// 64 rows of K or V from row t * 64: rows whose bit is clear are zero
template <typename T>
SITK_DEV void stage_keys(char* tile, const T* __restrict__ src, int64_t ld, int t, uint64_t bits, int tid) {
  using G = AttnGeom<T>;
#pragma unroll
  for (int i = 0; i < G::CH; ++i) {
    const int c = tid + 256 * i, row = c / G::CPR, cc = c % G::CPR;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (bit64(bits, row)) v = *reinterpret_cast<const u32x4*>(src + (int64_t)(64 * t + row) * ld + cc * G::EPV);
    *reinterpret_cast<u32x4*>(tile + ((cc * 16) / 128) * (64 * 128) + tile_off<T>(row, (cc * 16) % 128)) = v;
  }
}
template <typename T>
SITK_DEV void stage_rows(char* tile, const T* __restrict__ src, const Rows& st, const BlkShape& s, int hk, int r0, uint64_t bits, int tid) {
  using G = AttnGeom<T>;
#pragma unroll
  for (int i = 0; i < G::CH; ++i) {
    const int c = tid + 256 * i, row = c / G::CPR, cc = c % G::CPR;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (bit64(bits, row)) v = *reinterpret_cast<const u32x4*>(src + q_row(st, s, hk, r0 + row) + cc * G::EPV);
    *reinterpret_cast<u32x4*>(tile + ((cc * 16) / 128) * (64 * 128) + tile_off<T>(row, (cc * 16) % 128)) = v;
  }
}

// A 64-row tile over entries i0 .. n - 1 of its list: rows that skipped a tile keep their accumulators whatever K and V hold.
// part < 0: writes o and lse; else the part's sums.
template <typename T, class List>
SITK_DEV void fwd_rows(const BlkAttn& a, char* smem, const List& list, int i0, int n, const RowTile& w, int part) {
  using Gm = AttnGeom<T>;
  const BlkShape& s = a.s;
  char *sK = smem, *sV = smem + Gm::TILE_BYTES;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fq = lane >> 4, hk = w.hk, b = w.b, bh = w.bh;
  const int r = w.rt * 64 + 16 * wave + fr, rc = min(r, s.R - 1);
  const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)b * a.qs.b + q_row(a.qs, s, hk, rc);
  const T* kp = reinterpret_cast<const T*>(a.k) + (int64_t)b * a.ks.b + (int64_t)hk * a.ks.h;
  const T* vp = reinterpret_cast<const T*>(a.v) + (int64_t)b * a.vs.b + (int64_t)hk * a.vs.h;
  u32x4 qf[Gm::KS];
#pragma unroll
  for (int ks = 0; ks < Gm::KS; ++ks) qf[ks] = *reinterpret_cast<const u32x4*>(qp + (ks * 64 + fq * 16) / (int)sizeof(T));
  float m = -INFINITY, l = 0.f;                             // in units of q . k
  const float c = a.scale * kLog2e;
  f32x4 oacc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) oacc[dt] = splat4(0.f);
  for (int i = i0; i < n; ++i) {
    const uint64_t rows = uniform64(list.rows[i]);
    const int t0 = __builtin_amdgcn_readfirstlane((int)list.tile[i]);
    const uint64_t kb = a.kbits[(int64_t)b * s.nt + t0];
    __syncthreads();
    stage_keys<T>(sK, kp, a.ks.n, t0, kb, tid);
    stage_keys<T>(sV, vp, a.vs.n, t0, kb, tid);
    __syncthreads();
    const bool mine = bit64(rows, 16 * wave + fr);
    if (!__any(mine)) continue;
    f32x4 sc[4], old[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) sc[t] = splat4(0.f);
    row_mma<T>(sc, sK, qf, lane);
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        sc[t][jj] = mine && bit64(kb, 16 * t + 4 * fq + jj) ? sc[t][jj] : -INFINITY;
        mx = fmaxf(mx, sc[t][jj]);
      }
    mx = xor_max4(mx);
    const float mn = fmaxf(m, mx), ms = mn == -INFINITY ? 0.f : mn;
    const float alpha = fast_exp2(c * (m - ms));
    float ps = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        const float pv = fast_exp2(c * (sc[t][jj] - ms));
        sc[t][jj] = pv;
        ps += pv;
      }
    if (mine) { l = l * alpha + ps; m = mn; }
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) { old[dt] = oacc[dt]; oacc[dt] *= alpha; }
    TrMma<T>::run(oacc, sc, sV, lane);
    if (!mine) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) oacc[dt] = old[dt];
    }
  }
  const float lt = xor_sum4(l);
  if (r >= s.R) return;
  if (part >= 0) {
    store_part(a, part, bh, r, fq, oacc, m, lt);
    return;
  }
  const float inv = lt == 0.f ? 0.f : 1.0f / lt;
  T* orow = reinterpret_cast<T*>(a.out) + (int64_t)b * a.os.b + q_row(a.os, s, hk, r);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) store4(orow + 16 * dt + 4 * fq, oacc[dt] * inv);
  if (fq == 0) a.lse[q_flat(s, b, hk, r)] = lt == 0.f ? -INFINITY : m * a.scale + __log2f(lt) * kLn2;
}

template <typename T, int CAP>
__global__ __launch_bounds__(256) void block_attn_fwd_kernel(BlkAttn a) {
  __shared__ __attribute__((aligned(256))) char smem[2 * AttnGeom<T>::TILE_BYTES];
  __shared__ TileList<CAP> list;
  const RowTile w = row_tile(a.s, xcd_remap(blockIdx.x, gridDim.x));
  const int n = build_list<CAP>(list, a.mask + ((int64_t)w.bh * a.s.nrt + w.rt) * a.s.nb, a.kbits + (int64_t)w.b * a.s.nt, a.s, threadIdx.x);
  fwd_rows<T>(a, smem, list, 0, n, w, -1);
}

// dQ of a 64-row tile; delta and lse / scale of its rows come from the caller
template <typename T, class List>
SITK_DEV void dq_rows(const BlkAttn& a, char* smem, const List& list, int n, const RowTile& w) {
  using Gm = AttnGeom<T>;
  const BlkShape& s = a.s;
  char *sK = smem, *sV = smem + Gm::TILE_BYTES;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fq = lane >> 4, hk = w.hk, b = w.b, bh = w.bh;
  const int r = w.rt * 64 + 16 * wave + fr, rc = min(r, s.R - 1);
  const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)b * a.qs.b + q_row(a.qs, s, hk, rc);
  const T* op = reinterpret_cast<const T*>(a.o) + (int64_t)b * a.os.b + q_row(a.os, s, hk, rc);
  const T* dop = reinterpret_cast<const T*>(a.d_o) + (int64_t)b * a.dos.b + q_row(a.dos, s, hk, rc);
  const T* kp = reinterpret_cast<const T*>(a.k) + (int64_t)b * a.ks.b + (int64_t)hk * a.ks.h;
  const T* vp = reinterpret_cast<const T*>(a.v) + (int64_t)b * a.vs.b + (int64_t)hk * a.vs.h;
  u32x4 qf[Gm::KS], dof[Gm::KS];
  float dpart = 0.f;
#pragma unroll
  for (int ks = 0; ks < Gm::KS; ++ks) {
    const int eo = (ks * 64 + fq * 16) / (int)sizeof(T);
    qf[ks] = *reinterpret_cast<const u32x4*>(qp + eo);
    dof[ks] = *reinterpret_cast<const u32x4*>(dop + eo);
#pragma unroll
    for (int e = 0; e < Gm::EPV; ++e) dpart += to_f32(dop[eo + e]) * to_f32(op[eo + e]);
  }
  const float dl = xor_sum4(dpart), Lr = a.lse[q_flat(s, b, hk, rc)] / a.scale;
  if (fq == 0 && r < s.R) {
    a.delta[(int64_t)bh * s.Rp + r] = dl;
    a.stat[(int64_t)bh * s.Rp + r] = Lr;
  }
  const float c = a.scale * kLog2e;
  f32x4 dq[4], pk[4];
  float sd = 0.f;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) dq[dt] = pk[dt] = splat4(0.f);
  for (int i = 0; i < n; ++i) {
    const uint64_t rows = uniform64(list.rows[i]);
    const int t0 = __builtin_amdgcn_readfirstlane((int)list.tile[i]);
    const uint64_t kb = a.kbits[(int64_t)b * s.nt + t0];
    __syncthreads();
    stage_keys<T>(sK, kp, a.ks.n, t0, kb, tid);
    stage_keys<T>(sV, vp, a.vs.n, t0, kb, tid);
    __syncthreads();
    const bool mine = bit64(rows, 16 * wave + fr);
    if (!__any(mine)) continue;
    f32x4 sc[4], dp[4], old[4], old2[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) { sc[t] = splat4(0.f); dp[t] = splat4(0.f); }
    row_mma<T>(sc, sK, qf, lane);
    row_mma<T>(dp, sV, dof, lane);
    float sn = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        const bool ok = mine && bit64(kb, 16 * t + 4 * fq + jj);
        sc[t][jj] = ok ? fast_exp2(c * (sc[t][jj] - Lr)) : 0.f;
        dp[t][jj] = ok ? sc[t][jj] * (dp[t][jj] - dl) : 0.f;
        sn += to_f32(from_f32<T>(dp[t][jj]));
      }
    if (mine) sd += sn;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) { old[dt] = dq[dt]; old2[dt] = pk[dt]; }
    TrMma<T>::run(dq, dp, sK, lane);
    if constexpr (sizeof(T) == 2) TrMma<T>::run(pk, sc, sK, lane);
    if (!mine) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) { dq[dt] = old[dt]; pk[dt] = old2[dt]; }
    }
  }
  sd = sizeof(T) == 2 ? xor_sum4(sd) : 0.f;
  if (r >= s.R) return;
  T* row = reinterpret_cast<T*>(a.out) + (int64_t)b * a.os.b + q_row(a.os, s, hk, r);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) store4(row + 16 * dt + 4 * fq, (sizeof(T) == 2 ? dq[dt] - pk[dt] * sd : dq[dt]) * a.scale);
}

template <typename T, int CAP>
__global__ __launch_bounds__(256) void block_attn_bwd_dq_kernel(BlkAttn a) {
  __shared__ __attribute__((aligned(256))) char smem[2 * AttnGeom<T>::TILE_BYTES];
  __shared__ TileList<CAP> list;
  const RowTile w = row_tile(a.s, xcd_remap(blockIdx.x, gridDim.x));
  const int n = build_list<CAP>(list, a.mask + ((int64_t)w.bh * a.s.nrt + w.rt) * a.s.nb, a.kbits + (int64_t)w.b * a.s.nt, a.s, threadIdx.x);
  dq_rows<T>(a, smem, list, n, w);
}

// one workgroup per (sample, key head, 64-key tile): wave w owns keys 16 w .. + 15 and sweeps the row tiles that selected the block
template <typename T>
__global__ __launch_bounds__(256) void block_attn_bwd_dkv_kernel(BlkAttn a) {
  using Gm = AttnGeom<T>;
  __shared__ __attribute__((aligned(256))) char smem[2 * Gm::TILE_BYTES + 2 * 64 * 4];
  const BlkShape& s = a.s;
  char *sQ = smem, *sDO = smem + Gm::TILE_BYTES;
  float *sL = reinterpret_cast<float*>(smem + 2 * Gm::TILE_BYTES), *sD = sL + 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fq = lane >> 4;
  const int L = xcd_remap(blockIdx.x, gridDim.x), t0 = L % s.nt, bh = L / s.nt, hk = bh % s.Hk, b = bh / s.Hk;
  const uint64_t kb = a.kbits[(int64_t)b * s.nt + t0];
  const int key = 64 * t0 + 16 * wave + fr;
  const bool live = bit64(kb, 16 * wave + fr);
  const int64_t kc = min(key, s.Nk - 1);
  const T* kp = reinterpret_cast<const T*>(a.k) + (int64_t)b * a.ks.b + (int64_t)hk * a.ks.h + kc * a.ks.n;
  const T* vp = reinterpret_cast<const T*>(a.v) + (int64_t)b * a.vs.b + (int64_t)hk * a.vs.h + kc * a.vs.n;
  const T* qb = reinterpret_cast<const T*>(a.q) + (int64_t)b * a.qs.b;
  const T* dob = reinterpret_cast<const T*>(a.d_o) + (int64_t)b * a.dos.b;
  u32x4 kf[Gm::KS], vf[Gm::KS];
#pragma unroll
  for (int ks = 0; ks < Gm::KS; ++ks) {
    const int eo = (ks * 64 + fq * 16) / (int)sizeof(T);
    const u32x4 zero = {0u, 0u, 0u, 0u};
    kf[ks] = live ? *reinterpret_cast<const u32x4*>(kp + eo) : zero;
    vf[ks] = live ? *reinterpret_cast<const u32x4*>(vp + eo) : zero;
  }
  const float c = a.scale * kLog2e;
  f32x4 dk[4], dv[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) { dk[dt] = splat4(0.f); dv[dt] = splat4(0.f); }
  const uint64_t* sel = a.mask + (int64_t)s.B * s.Hk * s.nrt * s.nb + ((int64_t)bh * s.nb + t0 / s.c) * s.nrt;
  for (int rt = 0; kb && rt < s.nrt; ++rt) {
    const uint64_t bits = uniform64(sel[rt]);
    if (bits == 0) continue;
    __syncthreads();
    stage_rows<T>(sQ, qb, a.qs, s, hk, 64 * rt, bits, tid);
    stage_rows<T>(sDO, dob, a.dos, s, hk, 64 * rt, bits, tid);
    if (tid < 64) {
      const bool in = bit64(bits, tid);
      sL[tid] = in ? a.stat[(int64_t)bh * s.Rp + 64 * rt + tid] : INFINITY;
      sD[tid] = in ? a.delta[(int64_t)bh * s.Rp + 64 * rt + tid] : 0.f;
    }
    __syncthreads();
    f32x4 sc[4], dp[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) { sc[t] = splat4(0.f); dp[t] = splat4(0.f); }
    row_mma<T>(sc, sQ, kf, lane);
    row_mma<T>(dp, sDO, vf, lane);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const f32x4 Lr = *reinterpret_cast<const f32x4*>(sL + 16 * t + 4 * fq);
      const f32x4 Dr = *reinterpret_cast<const f32x4*>(sD + 16 * t + 4 * fq);
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        const float pv = fast_exp2((sc[t][jj] - Lr[jj]) * c);
        sc[t][jj] = pv;
        dp[t][jj] = pv * (dp[t][jj] - Dr[jj]) * a.scale;
      }
    }
    TrMma<T>::run(dv, sc, sDO, lane);
    TrMma<T>::run(dk, dp, sQ, lane);
  }
  if (key < s.Nk) {
    const int64_t row = (((int64_t)b * s.Nk + key) * s.Hk + hk) * 64;
    const f32x4 zero = splat4(0.f);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      store4(reinterpret_cast<T*>(a.dk) + row + 16 * dt + 4 * fq, live ? dk[dt] : zero);
      store4(reinterpret_cast<T*>(a.dv) + row + 16 * dt + 4 * fq, live ? dv[dt] : zero);
    }
  }
}

// ------------------------------------------------------------------------------------------
// 16-bit, query side
// ------------------------------------------------------------------------------------------
constexpr int BLK_STAGE = 16384;                    // a stage: 64 rows of two tensors, 128 bytes each
constexpr int FWD_STAGES = 2, DQ_STAGES = 3, DKV_STAGES = 2;
constexpr float kBlkRescale = 8.0f;                 // probabilities may reach 2^8 before the running maximum moves

// LDS reads of the last stage are done, every wave is here; a fence for the compiler too
SITK_DEV void blk_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
SITK_DEV void blk_dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// all but the last LOADS loads (of this wave) have landed
template <int LOADS>
SITK_DEV void blk_dma_wait_but() {
  static_assert(LOADS == 4 || LOADS == 5);
  if constexpr (LOADS == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(5)" ::: "memory");
}

// the four transposed fragments (column blocks of 16) of rows 32 s2 .. + 31 of the tile at LDS address `tile`; written out because the
// compiler puts a wait for every LDS-DMA in flight in front of an LDS read that it sees
#define SITK_BLK_TR4(F, TILE, S2)                                                                                             \
  do {                                                                                                                        \
    u32x2 _f[8];                                                                                                              \
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:" #S2 "*4096\n\tds_read_b64_tr_b16 %1, %8 offset:" #S2 "*4096+2048\n\t"    \
                 "ds_read_b64_tr_b16 %2, %9 offset:" #S2 "*4096\n\tds_read_b64_tr_b16 %3, %9 offset:" #S2 "*4096+2048\n\t"    \
                 "ds_read_b64_tr_b16 %4, %10 offset:" #S2 "*4096\n\tds_read_b64_tr_b16 %5, %10 offset:" #S2 "*4096+2048\n\t"  \
                 "ds_read_b64_tr_b16 %6, %11 offset:" #S2 "*4096\n\tds_read_b64_tr_b16 %7, %11 offset:" #S2 "*4096+2048\n\t"  \
                 "s_waitcnt lgkmcnt(0)"                                                                                       \
                 : "=&v"(_f[0]), "=&v"(_f[1]), "=&v"(_f[2]), "=&v"(_f[3]), "=&v"(_f[4]), "=&v"(_f[5]), "=&v"(_f[6]), "=&v"(_f[7]) \
                 : "v"((TILE) + lo.tr[0]), "v"((TILE) + lo.tr[1]), "v"((TILE) + lo.tr[2]), "v"((TILE) + lo.tr[3])             \
                 : "memory");                                                                                                 \
    for (int _d = 0; _d < 4; ++_d) F[_d] = u32x4{_f[2 * _d][0], _f[2 * _d][1], _f[2 * _d + 1][0], _f[2 * _d + 1][1]};         \
  } while (0)

// K and V tile -> stage: pieces of 8 rows x 128 bytes, waves 0 and 1 move K, 2 and 3 V, four pieces each
struct KeyDma {
  static constexpr int PIECES = 4;
  const char* base;
  int64_t step;          // bytes per tile
  uint32_t off[PIECES];       // lane offset of piece i
  int row0, dst0;        // row of piece 0 of this lane, piece 0's place in the stage
  SITK_DEV void init(const h16* k, int64_t kn, const h16* v, int64_t vn, int wave, int lane) {
    const bool is_v = wave >= 2;
    base = reinterpret_cast<const char*>(is_v ? v : k);
    const int64_t ld = is_v ? vn : kn;
    step = 128 * ld;
    row0 = (wave & 1) * 32 + (lane >> 3);
    dst0 = (is_v ? 8192 : 0) + (wave & 1) * 4096;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int row = row0 + 8 * i;
      off[i] = (uint32_t)(row * (int)ld * 2 + ((lane & 7) ^ (attn_res_key(row) << 1)) * 16);
    }
  }
  SITK_DEV void issue(char* stage, int t, uint64_t keys) const {
    const char* g = base + (int64_t)t * step;
    if (keys == ~0ull) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(g + off[i]),
                                         (__attribute__((address_space(3))) void*)(stage + dst0 + i * 1024), 16, 0, 0);
    } else {
      asm volatile("" ::: "memory");                        // (keeps the two ways apart: this one is rare)
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const char* src = bit64(keys, row0 + 8 * i) ? g + off[i] : reinterpret_cast<const char*>(g_blk_zero) + (off[i] & 127);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                         (__attribute__((address_space(3))) void*)(stage + dst0 + i * 1024), 16, 0, 0);
      }
    }
  }
};
// valid-key bits of a tile by a scalar load (the bits are final before the kernel starts)
SITK_DEV uint64_t tile_keys(const uint64_t* kbits, int t) {
  return *(const __attribute__((address_space(4))) uint64_t*)(uintptr_t)(kbits + t);
}
// The pipeline over a tile list: (tile, keys) of the tile to fetch next sit in scalar registers an iteration ahead, so that an
// iteration waits for no list read
template <int STAGES, class List>
struct TileFeed {
  const List& list;
  const uint64_t* kbits;
  const KeyDma& dma;
  char* smem;
  int n, fetched, stage;                                    // entries, entries fetched so far, stage of the next one
  int t_next;
  uint64_t k_next, keys[STAGES];                            // keys of the tile to fetch; of the tiles i, i + 1, ..
  SITK_DEV void look(int i) {
    t_next = __builtin_amdgcn_readfirstlane((int)list.tile[i < n ? i : n - 1]);
    k_next = tile_keys(kbits, t_next);
  }
  SITK_DEV void fetch(int slot) {
    if (fetched >= n) return;
    dma.issue(smem + stage * BLK_STAGE, t_next, k_next);
    keys[slot] = k_next;
    stage = stage == STAGES - 1 ? 0 : stage + 1;
    ++fetched;
    look(fetched);
  }
  SITK_DEV void start(int i0, int end) {
    n = end; fetched = i0; stage = 0;
    if (i0 >= end) return;
    look(i0);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(i);
  }
  // top of iteration i: tile i has landed for every wave, none reads tile i - 1 any more, and its stage takes tile i + STAGES - 1
  SITK_DEV void step(int i) {
    if (STAGES == 3 && i + 1 < n) blk_dma_wait_but<KeyDma::PIECES>();
    else blk_dma_wait();
    blk_barrier();
    fetch(STAGES - 1);
  }
  SITK_DEV void advance() {
#pragma unroll
    for (int i = 0; i + 1 < STAGES; ++i) keys[i] = keys[i + 1];
  }
};
// scores of keys whose bit is clear -> -infinity (rare: the last tile, masked keys)
SITK_DEV void mask_keys(f32x4 (&sc)[4], uint64_t keys, int fq) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint32_t nib = (uint32_t)(keys >> (16 * t + 4 * fq));
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) sc[t][jj] = nib >> jj & 1 ? sc[t][jj] : -INFINITY;
  }
}

// forward.  Scores start from minus the running maximum (the accumulators' initial value), in units of q . k; rows that did not select
// the block start from -infinity, so their probabilities are zero.  The maximum moves only when a score exceeds it by 2^8 in the
// exponent, or a row meets its first block.
// The sweep lets a zero probability meet every value of the tile, which is right unless K or V holds an infinity or a NaN there: then a
// NaN shows in the row, and the workgroup takes its rows again the plain way.
template <int CAP, bool PARTS>
__global__ __launch_bounds__(256, 4) void block_attn_fwd_ring_kernel(BlkAttn a) {
  typedef TileList<CAP> List;
  __shared__ __attribute__((aligned(256))) char smem[FWD_STAGES * BLK_STAGE];
  __shared__ List list;
  const BlkShape& s = a.s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
  const int L = xcd_remap(blockIdx.x, gridDim.x);
  const int part = PARTS ? L % a.parts : 0;
  const RowTile w = row_tile(s, PARTS ? L / a.parts : L);
  const int r = w.rt * 64 + 16 * wave + fr;
  const h16* qp = reinterpret_cast<const h16*>(a.q) + (int64_t)w.b * a.qs.b + q_row(a.qs, s, w.hk, min(r, s.R - 1));
  u32x4 qf[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) qf[ks] = *reinterpret_cast<const u32x4*>(qp + ks * 32 + fq * 8);
  KeyDma dma;
  dma.init(reinterpret_cast<const h16*>(a.k) + (int64_t)w.b * a.ks.b + (int64_t)w.hk * a.ks.h, a.ks.n,
           reinterpret_cast<const h16*>(a.v) + (int64_t)w.b * a.vs.b + (int64_t)w.hk * a.vs.h, a.vs.n, wave, lane);
  const uint64_t* kbits = a.kbits + (int64_t)w.b * s.nt;
  const int all = build_list<CAP>(list, a.mask + ((int64_t)w.bh * s.nrt + w.rt) * s.nb, kbits, s, tid);
  const int i0 = PARTS ? (int)((int64_t)all * part / a.parts) : 0, n = PARTS ? (int)((int64_t)all * (part + 1) / a.parts) : all;
  const float c = a.scale * kLog2e, thr = kBlkRescale / c;
  const LaneOffs lo = lane_offs_h16(lane);
  const uint32_t lbase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  float m = 0.f, l = 0.f;                                   // l: this lane's 16 keys of every tile, before the rounding of P
  bool begun = false;                                       // the row has met a block: m is its running maximum
  f32x4 oacc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) oacc[dt] = splat4(0.f);
  TileFeed<FWD_STAGES, List> feed{list, kbits, dma, smem};
  feed.start(i0, n);
  int at = 0;
  for (int i = i0; i < n; ++i, at = at == (FWD_STAGES - 1) * BLK_STAGE ? 0 : at + BLK_STAGE, feed.advance()) {
    feed.step(i);
    const uint32_t bits = (uint32_t)(uniform64(list.rows[i]) >> (16 * wave)) & 0xFFFFu;
    const uint64_t keys = feed.keys[0];
    if (bits == 0) continue;
    const bool mine = bits >> fr & 1;
    f32x4 sc[4];
    {
      u32x4 kf[4][2];
      SITK_RING_ROWS8(kf, lbase + at + lo.row[0], lbase + at + lo.row[1], 0);
      const f32x4 init = splat4(mine ? -m : -INFINITY);
#pragma unroll
      for (int t = 0; t < 4; ++t) sc[t] = Mma<h16>::mma(kf[t][0], qf[0], init);
#pragma unroll
      for (int t = 0; t < 4; ++t) sc[t] = Mma<h16>::mma(kf[t][1], qf[1], sc[t]);
    }
    if (keys != ~0ull) {
      asm volatile("" ::: "memory");
      mask_keys(sc, keys, fq);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) mx = fmaxf(mx, sc[t][jj]);
    if (__any(mx > thr || (mine && !begun))) {
      asm volatile("" ::: "memory");
      mx = xor_max4(mx);
      float d = begun ? fmaxf(mx, 0.f) : fmaxf(mx, -3e38f);
      if (!mine) d = 0.f;
      const float alpha = begun ? fast_exp2(-c * d) : 1.f;  // (nothing summed yet: any finite factor)
      m += d;
      begun |= mine;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) oacc[dt] *= alpha;
#pragma unroll
      for (int t = 0; t < 4; ++t) sc[t] -= d;
    }
    float ps = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        sc[t][jj] = fast_exp2(c * sc[t][jj]);
        ps += sc[t][jj];
      }
    l += ps;
    const u32x4 pf[2] = {pack_pair(sc[0], sc[1]), pack_pair(sc[2], sc[3])};
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {                        // 32 keys at a time
      u32x4 vf[4];
      if (s2 == 0) SITK_BLK_TR4(vf, lbase + at + 8192, 0);
      else SITK_BLK_TR4(vf, lbase + at + 8192, 1);
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) oacc[dt] = Mma<h16>::mma(vf[dt], pf[s2], oacc[dt]);
    }
  }
  float bad = l * 0.f;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) bad += oacc[dt][jj] * 0.f;
  if (__syncthreads_or(bad != bad)) {
    fwd_rows<h16>(a, smem, list, i0, n, w, PARTS ? part : -1);
    return;
  }
  const float lt = xor_sum4(l);
  if (r >= s.R) return;
  if constexpr (PARTS) {
    store_part(a, part, w.bh, r, fq, oacc, m, begun ? lt : 0.f);
  } else {
    const float inv = lt == 0.f ? 0.f : 1.0f / lt;
    h16* orow = reinterpret_cast<h16*>(a.out) + (int64_t)w.b * a.os.b + q_row(a.os, s, w.hk, r);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) store4(orow + 16 * dt + 4 * fq, oacc[dt] * inv);
    if (fq == 0) a.lse[q_flat(s, w.b, w.hk, r)] = lt == 0.f ? -INFINITY : m * a.scale + __log2f(lt) * kLn2;
  }
}

// parts of a row -> o, lse; one wave per row, a lane per feature
__global__ __launch_bounds__(256) void block_attn_join_kernel(BlkAttn a) {
  const BlkShape& s = a.s;
  const int lane = threadIdx.x & 63;
  const int64_t rows = (int64_t)s.B * s.Hk * s.Rp, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int bh = (int)(row / s.Rp), r = (int)(row - (int64_t)bh * s.Rp), hk = bh % s.Hk, b = bh / s.Hk;
  if (r >= s.R) return;
  // lane z holds part z's maximum and sum (at most 16 parts); a part without a block of the row has the sum 0 and weighs nothing
  const float* pm = a.part + (int64_t)a.parts * rows * 64;
  const bool part = lane < a.parts;
  const float mz = part ? pm[(int64_t)lane * rows + row] : 0.f, lz = part ? pm[(int64_t)(a.parts + lane) * rows + row] : 0.f;
  const float m = wave_max(lz != 0.f ? mz : -INFINITY);
  const float f = lz != 0.f ? fast_exp2(a.scale * kLog2e * (mz - m)) : 0.f;
  const float l = wave_sum(f * lz);
  float o = 0.f;
#pragma unroll 4
  for (int z = 0; z < a.parts; ++z) {
    const float v = a.part[((int64_t)z * rows + row) * 64 + lane], fz = __shfl(f, z, 64);
    o += fz != 0.f ? fz * v : 0.f;
  }
  h16* orow = reinterpret_cast<h16*>(a.out) + (int64_t)b * a.os.b + q_row(a.os, s, hk, r);
  orow[lane] = (h16)(l == 0.f ? 0.f : o / l);
  if (lane == 0) a.lse[q_flat(s, b, hk, r)] = l == 0.f ? -INFINITY : m * a.scale + __log2f(l) * kLn2;
}

// dQ, and the rows' statistics for the key side.  Sum over the keys of dS is zero by definition, but not once dS is rounded to 16 bits and
// delta comes from the rounded o; that remainder times the keys' common part is what dQ would lose most to (twice the rounding of dQ
// itself where keys are smooth).  So the kernel also sums the rounded dS and P K, and subtracts (sum dS) (P K): what is left sees only
// how far a key is from the row's mean key.
template <int CAP, bool FINE>
__global__ __launch_bounds__(256, FINE ? 2 : 3) void block_attn_bwd_dq_ring_kernel(BlkAttn a) {
  typedef TileList<CAP> List;
  __shared__ __attribute__((aligned(256))) char smem[DQ_STAGES * BLK_STAGE];
  __shared__ List list;
  const BlkShape& s = a.s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
  const RowTile w = row_tile(s, xcd_remap(blockIdx.x, gridDim.x));
  const int r = w.rt * 64 + 16 * wave + fr, rc = min(r, s.R - 1);
  const h16* qp = reinterpret_cast<const h16*>(a.q) + (int64_t)w.b * a.qs.b + q_row(a.qs, s, w.hk, rc);
  const h16* op = reinterpret_cast<const h16*>(a.o) + (int64_t)w.b * a.os.b + q_row(a.os, s, w.hk, rc);
  const h16* dop = reinterpret_cast<const h16*>(a.d_o) + (int64_t)w.b * a.dos.b + q_row(a.dos, s, w.hk, rc);
  u32x4 qf[2], dof[2];
  float dpart = 0.f;
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    qf[ks] = *reinterpret_cast<const u32x4*>(qp + ks * 32 + fq * 8);
    dof[ks] = *reinterpret_cast<const u32x4*>(dop + ks * 32 + fq * 8);
    const h16x8 d8 = __builtin_bit_cast(h16x8, dof[ks]), o8 = *reinterpret_cast<const h16x8*>(op + ks * 32 + fq * 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) dpart += (float)d8[e] * (float)o8[e];
  }
  const float dl = xor_sum4(dpart), Lr = a.lse[q_flat(s, w.b, w.hk, rc)] / a.scale;
  if (fq == 0 && r < s.R) {
    a.delta[(int64_t)w.bh * s.Rp + r] = dl;
    a.stat[(int64_t)w.bh * s.Rp + r] = Lr;
  }
  KeyDma dma;
  dma.init(reinterpret_cast<const h16*>(a.k) + (int64_t)w.b * a.ks.b + (int64_t)w.hk * a.ks.h, a.ks.n,
           reinterpret_cast<const h16*>(a.v) + (int64_t)w.b * a.vs.b + (int64_t)w.hk * a.vs.h, a.vs.n, wave, lane);
  const uint64_t* kbits = a.kbits + (int64_t)w.b * s.nt;
  const int n = build_list<CAP>(list, a.mask + ((int64_t)w.bh * s.nrt + w.rt) * s.nb, kbits, s, tid);
  const float c = a.scale * kLog2e;
  const LaneOffs lo = lane_offs_h16(lane);
  const uint32_t lbase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  const u32x4 ones = {kOnesH16x2, kOnesH16x2, kOnesH16x2, kOnesH16x2};
  f32x4 dq[4], pk[4], sd = splat4(0.f);
  float rest = 0.f;                                         // this lane's part of the sum of dS, before its rounding
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) dq[dt] = pk[dt] = splat4(0.f);
  TileFeed<DQ_STAGES, List> feed{list, kbits, dma, smem};
  feed.start(0, n);
  int at = 0;
  for (int i = 0; i < n; ++i, at = at == (DQ_STAGES - 1) * BLK_STAGE ? 0 : at + BLK_STAGE, feed.advance()) {
    feed.step(i);
    const uint32_t bits = (uint32_t)(uniform64(list.rows[i]) >> (16 * wave)) & 0xFFFFu;
    const uint64_t keys = feed.keys[0];
    if (bits == 0) continue;
    const bool mine = bits >> fr & 1;
    f32x4 sc[4], dp[4];
    {
      u32x4 kf[4][2];
      SITK_RING_ROWS8(kf, lbase + at + lo.row[0], lbase + at + lo.row[1], 0);
      const f32x4 init = splat4(mine ? -Lr : -INFINITY);
#pragma unroll
      for (int t = 0; t < 4; ++t) sc[t] = Mma<h16>::mma(kf[t][0], qf[0], init);
#pragma unroll
      for (int t = 0; t < 4; ++t) sc[t] = Mma<h16>::mma(kf[t][1], qf[1], sc[t]);
    }
    {
      u32x4 vf[4][2];
      SITK_RING_ROWS8(vf, lbase + at + lo.row[0], lbase + at + lo.row[1], 8192);
      const f32x4 init = splat4(FINE ? 0.f : -dl);
#pragma unroll
      for (int t = 0; t < 4; ++t) dp[t] = Mma<h16>::mma(vf[t][0], dof[0], init);
#pragma unroll
      for (int t = 0; t < 4; ++t) dp[t] = Mma<h16>::mma(vf[t][1], dof[1], dp[t]);
    }
    if (keys != ~0ull) {
      asm volatile("" ::: "memory");
      mask_keys(sc, keys, fq);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        sc[t][jj] = fast_exp2(c * sc[t][jj]);
        dp[t][jj] = (FINE ? dp[t][jj] - dl : dp[t][jj]) * sc[t][jj];
      }
    if constexpr (FINE) {
      const f32x4 four = (dp[0] + dp[1]) + (dp[2] + dp[3]);
      rest += (four[0] + four[1]) + (four[2] + four[3]);
    }
    const u32x4 pf[2] = {pack_pair(sc[0], sc[1]), pack_pair(sc[2], sc[3])}, df[2] = {pack_pair(dp[0], dp[1]), pack_pair(dp[2], dp[3])};
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      u32x4 kt[4];
      if (s2 == 0) SITK_BLK_TR4(kt, lbase + at, 0);
      else SITK_BLK_TR4(kt, lbase + at, 1);
      sd = Mma<h16>::mma(ones, df[s2], sd);
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        dq[dt] = Mma<h16>::mma(kt[dt], df[s2], dq[dt]);
        pk[dt] = Mma<h16>::mma(kt[dt], pf[s2], pk[dt]);
      }
    }
  }
  float bad = sd[0] * 0.f;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) bad += dq[dt][jj] * 0.f + pk[dt][jj] * 0.f;
  if (__syncthreads_or(bad != bad)) {
    dq_rows<h16>(a, smem, list, n, w);
    return;
  }
  if constexpr (FINE) rest = xor_sum4(rest);
  if (r >= s.R) return;
  if (FINE && fq == 0) a.delta[(int64_t)w.bh * s.Rp + r] = dl + rest;
  h16* row = reinterpret_cast<h16*>(a.out) + (int64_t)w.b * a.os.b + q_row(a.os, s, w.hk, r);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) store4(row + 16 * dt + 4 * fq, (dq[dt] - pk[dt] * sd[0]) * a.scale);
}

// ------------------------------------------------------------------------------------------
// 16-bit, key side: one workgroup per (sample, key head, 64-key tile).  The rows that selected the block are listed in LDS (ascending)
// and gathered 64 at a time: Q and dO rows, lse / scale and delta by LDS-DMA.  Wave (kh, rh) = (wave & 1, wave >> 1) owns 32 keys and
// 32 of the 64 gathered rows (half the LDS reads of 16 keys x 64 rows); the two row halves are added at the end.
// ------------------------------------------------------------------------------------------
constexpr int DKV_WAIT = 512, DKV_LIST = DKV_WAIT + 4096;   // rows listed at once: up to 64 words are appended while at most DKV_WAIT wait
constexpr int DKV_STAGE = BLK_STAGE + 512;  // Q tile, dO tile, 64 x lse / scale, 64 x delta

// what is left of a, b behind their rounding to `packed`
SITK_DEV u32x4 pack_rest(f32x4 a, f32x4 b, u32x4 packed) {
  const h16x8 h = __builtin_bit_cast(h16x8, packed);
#pragma unroll
  for (int i = 0; i < 4; ++i) { a[i] -= (float)h[i]; b[i] -= (float)h[4 + i]; }
  return pack_pair(a, b);
}
// FINE: P and dS enter as the sum of two 16-bit values.
template <bool FINE>
__global__ __launch_bounds__(256, 2) void block_attn_bwd_dkv_ring_kernel(BlkAttn a) {
  __shared__ __attribute__((aligned(256))) char smem[DKV_STAGES * DKV_STAGE];
  __shared__ int list[DKV_LIST];
  const BlkShape& s = a.s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
  const int kh = wave & 1, rh = wave >> 1;
  const int L = xcd_remap(blockIdx.x, gridDim.x), t0 = L % s.nt, bh = L / s.nt, hk = bh % s.Hk, b = bh / s.Hk;
  const uint64_t kb = a.kbits[(int64_t)b * s.nt + t0];
  const h16* kp = reinterpret_cast<const h16*>(a.k) + (int64_t)b * a.ks.b + (int64_t)hk * a.ks.h;
  const h16* vp = reinterpret_cast<const h16*>(a.v) + (int64_t)b * a.vs.b + (int64_t)hk * a.vs.h;
  u32x4 kf[2][2], vf[2][2];
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const int in = 32 * kh + 16 * kt + fr;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      kf[kt][ks] = vf[kt][ks] = u32x4{0u, 0u, 0u, 0u};
      if (bit64(kb, in)) {
        kf[kt][ks] = *reinterpret_cast<const u32x4*>(kp + (int64_t)(64 * t0 + in) * a.ks.n + ks * 32 + fq * 8);
        vf[kt][ks] = *reinterpret_cast<const u32x4*>(vp + (int64_t)(64 * t0 + in) * a.vs.n + ks * 32 + fq * 8);
      }
    }
  }
  // this wave's pieces of a stage: waves 0 and 1 move Q, 2 and 3 dO, four pieces of 8 rows; wave 0 also lse / scale, wave 1 delta
  const Rows& st = wave >= 2 ? a.dos : a.qs;
  const h16* src = wave >= 2 ? reinterpret_cast<const h16*>(a.d_o) + (int64_t)b * a.dos.b : reinterpret_cast<const h16*>(a.q) + (int64_t)b * a.qs.b;
  const float* stat = (wave == 0 ? a.stat : a.delta) + (int64_t)bh * s.Rp;
  auto issue = [&](int n, int total) {                       // rows list[64 n ..] -> stage n
    if (64 * n >= total) return;
    char* dst = smem + n % DKV_STAGES * DKV_STAGE;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = (wave & 1) * 4 + i, row = p * 8 + (lane >> 3), ch = ((lane & 7) ^ (attn_res_key(row) << 1)) * 16;
      const int at = 64 * n + row;
      const char* g = reinterpret_cast<const char*>(g_blk_zero) + ch;
      if (at < total) g = reinterpret_cast<const char*>(src + q_row(st, s, hk, list[at])) + ch;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                       (__attribute__((address_space(3))) void*)(dst + (wave >= 2 ? 8192 : 0) + p * 1024), 16, 0, 0);
    }
    if (wave < 2) {
      const int at = 64 * n + lane;
      const float* g = wave == 0 ? g_blk_inf + lane : reinterpret_cast<const float*>(g_blk_zero) + (lane & 31);
      if (at < total) g = stat + list[at];
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                       (__attribute__((address_space(3))) void*)(dst + BLK_STAGE + wave * 256), 4, 0, 0);
    }
  };
  const float c = a.scale * kLog2e;
  const LaneOffs lo = lane_offs_h16(lane);
  const uint32_t lbase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  f32x4 dk[2][4], dv[2][4];
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) { dk[kt][dt] = splat4(0.f); dv[kt][dt] = splat4(0.f); }

  const uint64_t* sel = a.mask + (int64_t)s.B * s.Hk * s.nrt * s.nb + ((int64_t)bh * s.nb + t0 / s.c) * s.nrt;
  int have = 0;                                              // rows listed and not yet used
  uint64_t word = kb && lane < s.nrt ? sel[lane] : 0;
  for (int rt0 = 0; kb && rt0 < s.nrt;) {
    // append words until more than DKV_WAIT rows wait or none are left
    do {
      const uint64_t cur = word;
      word = rt0 + 64 + lane < s.nrt ? sel[rt0 + 64 + lane] : 0;       // the next 64, in flight meanwhile
      int upto = __popcll(cur);
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(upto, o, 64);
        if (lane >= o) upto += t;
      }
      const int total = __builtin_amdgcn_readlane(upto, 63), before = upto - __popcll(cur);
      uint64_t todo = __ballot(cur != 0);
      for (int i = 0; todo; ++i) {                           // wave i of four lists the i-th word that has rows
        const int l = __ffsll((unsigned long long)todo) - 1;
        todo &= todo - 1;
        if ((i & 3) != wave) continue;
        const uint64_t v = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(cur >> 32), l) << 32 |
                           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)cur, l);
        const int at = have + __builtin_amdgcn_readlane(before, l);
        if (bit64(v, lane)) list[at + __popcll(v & ((1ull << lane) - 1))] = 64 * (rt0 + l) + lane;
      }
      have += total;
      rt0 += 64;
    } while (rt0 < s.nrt && have <= DKV_WAIT);
    const bool last = rt0 >= s.nrt;
    const int total = last ? have : have & ~63, tiles = (total + 63) / 64;
    __syncthreads();                                         // the list is whole
    blk_dma_wait();                                          // (nothing but tiles of rows counts below)
#pragma unroll
    for (int i = 0; i + 1 < DKV_STAGES; ++i) issue(i, total);
    int at = 0;
    for (int n = 0; n < tiles; ++n, at = at == (DKV_STAGES - 1) * DKV_STAGE ? 0 : at + DKV_STAGE) {
      if (DKV_STAGES == 2 || n + 1 >= tiles) blk_dma_wait();
      else if (wave < 2) blk_dma_wait_but<5>();
      else blk_dma_wait_but<4>();
      blk_barrier();
      issue(n + DKV_STAGES - 1, total);
      f32x4 sc[2][2], dp[2][2];                              // [16-row tile][16-key tile]: rows on the registers, keys on the lanes
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        u32x4 qf[2], of[2];
        f32x4 Lr, Dr;
        const uint32_t o0 = lbase + at + lo.row[0] + (2 * rh + t) * 2048, o1 = lbase + at + lo.row[1] + (2 * rh + t) * 2048;
        asm volatile("ds_read_b128 %0, %6\n\tds_read_b128 %1, %7\n\tds_read_b128 %2, %6 offset:8192\n\tds_read_b128 %3, %7 offset:8192\n\t"
                     "ds_read_b128 %4, %8\n\tds_read_b128 %5, %8 offset:256\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(qf[0]), "=&v"(qf[1]), "=&v"(of[0]), "=&v"(of[1]), "=&v"(Lr), "=&v"(Dr)
                     : "v"(o0), "v"(o1), "v"(lbase + at + BLK_STAGE + (32 * rh + 16 * t + 4 * fq) * 4)
                     : "memory");
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          sc[t][kt] = Mma<h16>::mma(qf[0], kf[kt][0], -Lr);
          dp[t][kt] = Mma<h16>::mma(of[0], vf[kt][0], FINE ? splat4(0.f) : -Dr);
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          sc[t][kt] = Mma<h16>::mma(qf[1], kf[kt][1], sc[t][kt]);
          dp[t][kt] = Mma<h16>::mma(of[1], vf[kt][1], dp[t][kt]);
          if constexpr (FINE) dp[t][kt] -= Dr;
        }
      }
      u32x4 pf[2], df[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            sc[t][kt][jj] = fast_exp2(c * sc[t][kt][jj]);
            dp[t][kt][jj] *= sc[t][kt][jj];
          }
        pf[kt] = pack_pair(sc[0][kt], sc[1][kt]);
        df[kt] = pack_pair(dp[0][kt], dp[1][kt]);
      }
      u32x4 qt[4], ot[4];
      SITK_BLK_TR4(ot, lbase + at + 8192 + rh * 4096, 0);
      SITK_BLK_TR4(qt, lbase + at + rh * 4096, 0);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
          dv[kt][dt] = Mma<h16>::mma(ot[dt], pf[kt], dv[kt][dt]);
          dk[kt][dt] = Mma<h16>::mma(qt[dt], df[kt], dk[kt][dt]);
        }
      if constexpr (FINE) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          const u32x4 pr = pack_rest(sc[0][kt], sc[1][kt], pf[kt]), dr = pack_rest(dp[0][kt], dp[1][kt], df[kt]);
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) {
            dv[kt][dt] = Mma<h16>::mma(ot[dt], pr, dv[kt][dt]);
            dk[kt][dt] = Mma<h16>::mma(qt[dt], dr, dk[kt][dt]);
          }
        }
      }
    }
    __syncthreads();                                         // every wave is done with the list
    if (!last) {
      int keep = 0;
      if (tid < have - total) keep = list[total + tid];
      __syncthreads();
      if (tid < have - total) list[tid] = keep;
      have -= total;
      __syncthreads();
    }
  }
  // rows 32 .. 63's half joins rows 0 .. 31's; stages are free
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);              // [kh][dk, dv][2][4][64 lanes][4] = 32 KB
  if (rh == 1) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        *reinterpret_cast<f32x4*>(red + (((kh * 2 + 0) * 8 + kt * 4 + dt) * 64 + lane) * 4) = dk[kt][dt];
        *reinterpret_cast<f32x4*>(red + (((kh * 2 + 1) * 8 + kt * 4 + dt) * 64 + lane) * 4) = dv[kt][dt];
      }
  }
  __syncthreads();
  if (rh == 1) return;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const int in = 32 * kh + 16 * kt + fr, key = 64 * t0 + in;
    if (key >= s.Nk) continue;
    const bool live = bit64(kb, in);
    const int64_t row = (((int64_t)b * s.Nk + key) * s.Hk + hk) * 64;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      const f32x4 k2 = dk[kt][dt] + *reinterpret_cast<const f32x4*>(red + (((kh * 2 + 0) * 8 + kt * 4 + dt) * 64 + lane) * 4);
      const f32x4 v2 = dv[kt][dt] + *reinterpret_cast<const f32x4*>(red + (((kh * 2 + 1) * 8 + kt * 4 + dt) * 64 + lane) * 4);
      store4(reinterpret_cast<h16*>(a.dk) + row + 16 * dt + 4 * fq, live ? k2 * a.scale : splat4(0.f));
      store4(reinterpret_cast<h16*>(a.dv) + row + 16 * dt + 4 * fq, live ? v2 : splat4(0.f));
    }
  }
}

// Parts of a row tile's key tiles: enough workgroups for two per CU, at least four tiles of the sequence each (321 tokens, 3 heads: a call of
// 14 us in one part, 18 in three and a join; 1 x 321 queries over 1281 keys: 13.4 us in five parts, 17 in two), at most 16.
static int blk_parts(const BlkShape& s, int dtype) {
  if (dtype == SITK_F32) return 1;
  const int64_t wgs = (int64_t)s.B * s.Hk * s.nrt;
  int64_t p = 512 / wgs;
  if (p > s.nt / 4) p = s.nt / 4;
  return (int)(p < 1 ? 1 : p > 16 ? 16 : p);
}

}  // namespace sitk

static int blk_attn_args(const char* who, const sitk_block_attn* p, int dtype, sitk::BlkAttn& a) {
  SITK_REQUIRE(p, "%s: null pointer", who);
  SITK_TRY(sitk::blk_check(who, p->B, p->Nq, p->Nk, p->H, p->Hk, p->block, dtype));
  SITK_REQUIRE(p->mask && p->pool && p->lse && (uintptr_t)p->pool % 16 == 0, "%s: null or unaligned pointer", who);
  // lse / scale has to be a number (below 1e-37 it was not, and the gradients were zero)
  SITK_REQUIRE(p->scale >= 0x1p-100f && p->scale <= 0x1p100f, "%s: scale = %g (2^-100 to 2^100)", who, (double)p->scale);
  SITK_TRY(sitk::blk_rows(who, "q", p->q, p->qs, dtype));
  SITK_TRY(sitk::blk_rows(who, "k", p->k, p->ks, dtype));
  SITK_TRY(sitk::blk_rows(who, "v", p->v, p->vs, dtype));
  const sitk_block_rows rows = {(int64_t)p->Nq * p->H * 64, (int64_t)p->H * 64, 64};
  SITK_TRY(sitk::blk_rows(who, "o", p->o, rows, dtype));
  a.q = p->q; a.k = p->k; a.v = p->v; a.o = p->o;
  a.qs = sitk::to_rows(p->qs); a.ks = sitk::to_rows(p->ks); a.vs = sitk::to_rows(p->vs); a.os = sitk::to_rows(rows);
  a.s = sitk::blk_shape(p->B, p->Nq, p->Nk, p->H, p->Hk, p->block);
  a.mask = p->mask; a.lse = p->lse; a.scale = p->scale;
  a.kbits = sitk::blk_pool_at(const_cast<void*>(p->pool), a.s, dtype).kbits;
  return SITK_OK;
}

extern "C" size_t sitk_block_attention_fwd_ws_bytes(int B, int Nq, int Nk, int H, int Hk, int block, int dtype) {
  if (B < 1 || Nq < 1 || Nk < 1 || Hk < 1 || H < Hk || H % Hk || block < 64) return 0;
  const sitk::BlkShape s = sitk::blk_shape(B, Nq, Nk, H, Hk, block);
  const int parts = sitk::blk_parts(s, dtype);
  return parts > 1 ? (size_t)parts * B * Hk * s.Rp * 66 * 4 : 0;
}

SITK_F16_TWIN(sitk_block_attention_fwd)
extern "C" int sitk_block_attention_fwd(const sitk_block_attn* p, void* ws, size_t ws_bytes, int dtype, sitk_stream_t stream) {
  sitk::BlkAttn a{};
  SITK_TRY(blk_attn_args("block_attention_fwd", p, dtype, a));
  const size_t need = sitk_block_attention_fwd_ws_bytes(p->B, p->Nq, p->Nk, p->H, p->Hk, p->block, dtype);
  SITK_REQUIRE(ws_bytes >= need && (need == 0 || (ws && (uintptr_t)ws % 16 == 0)), "block_attention_fwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  SITK_FORWARD_F16(dtype, sitk_block_attention_fwd, p, ws, ws_bytes, dtype, stream);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  a.out = p->o;
  a.part = reinterpret_cast<float*>(ws);
  a.parts = sitk::blk_parts(a.s, dtype);
  const dim3 grid((unsigned)(a.s.B * a.s.Hk * a.s.nrt * a.parts));
  const bool small = a.s.nt <= sitk::BLK_LIST;
  if (dtype == SITK_F32) {
    if (small) hipLaunchKernelGGL((sitk::block_attn_fwd_kernel<float, sitk::BLK_LIST>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((sitk::block_attn_fwd_kernel<float, sitk::BLK_MAX_TILES>), grid, dim3(256), 0, st, a);
  } else if (a.parts > 1) {
    if (small) hipLaunchKernelGGL((sitk::block_attn_fwd_ring_kernel<sitk::BLK_LIST, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((sitk::block_attn_fwd_ring_kernel<sitk::BLK_MAX_TILES, true>), grid, dim3(256), 0, st, a);
    SITK_LAUNCH_CHECK("block_attention_fwd");
    hipLaunchKernelGGL(sitk::block_attn_join_kernel, dim3((unsigned)cdiv64((int64_t)a.s.B * a.s.Hk * a.s.Rp, 4)), dim3(256), 0, st, a);
  } else {
    if (small) hipLaunchKernelGGL((sitk::block_attn_fwd_ring_kernel<sitk::BLK_LIST, false>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((sitk::block_attn_fwd_ring_kernel<sitk::BLK_MAX_TILES, false>), grid, dim3(256), 0, st, a);
  }
  SITK_LAUNCH_CHECK("block_attention_fwd");
  return SITK_OK;
}

extern "C" size_t sitk_block_attention_bwd_ws_bytes(int B, int Nq, int Nk, int H, int Hk, int block) {
  if (B < 1 || Nq < 1 || Nk < 1 || Hk < 1 || H < Hk || H % Hk || block < 64) return 0;
  const sitk::BlkShape s = sitk::blk_shape(B, Nq, Nk, H, Hk, block);
  return (size_t)B * Hk * s.Rp * 8;
}

SITK_F16_TWIN(sitk_block_attention_bwd)
extern "C" int sitk_block_attention_bwd(const sitk_block_attn* p, const void* d_o, const sitk_block_rows* dos, void* dq, void* dk, void* dv,
                                        void* ws, size_t ws_bytes, int dtype, sitk_stream_t stream) {
  sitk::BlkAttn a{};
  SITK_TRY(blk_attn_args("block_attention_bwd", p, dtype, a));
  SITK_REQUIRE(dos && dq && dk && dv, "block_attention_bwd: null pointer");
  SITK_REQUIRE(((uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16 == 0, "block_attention_bwd: gradients are not 16-byte aligned");
  SITK_TRY(sitk::blk_rows("block_attention_bwd", "d_o", d_o, *dos, dtype));
  const size_t need = sitk_block_attention_bwd_ws_bytes(p->B, p->Nq, p->Nk, p->H, p->Hk, p->block);
  SITK_REQUIRE(ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need, "block_attention_bwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  SITK_FORWARD_F16(dtype, sitk_block_attention_bwd, p, d_o, dos, dq, dk, dv, ws, ws_bytes, dtype, stream);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  a.d_o = d_o; a.dos = sitk::to_rows(*dos); a.out = dq; a.dk = dk; a.dv = dv;
  a.stat = reinterpret_cast<float*>(ws);
  a.delta = a.stat + (size_t)a.s.B * a.s.Hk * a.s.Rp;
  const dim3 gq((unsigned)(a.s.B * a.s.Hk * a.s.nrt)), gk((unsigned)(a.s.B * a.s.Hk * a.s.nt));
  const bool small = a.s.nt <= sitk::BLK_LIST;
  if (dtype == SITK_F32) {
    if (small) hipLaunchKernelGGL((sitk::block_attn_bwd_dq_kernel<float, sitk::BLK_LIST>), gq, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((sitk::block_attn_bwd_dq_kernel<float, sitk::BLK_MAX_TILES>), gq, dim3(256), 0, st, a);
    SITK_LAUNCH_CHECK("block_attention_bwd dq");
    hipLaunchKernelGGL((sitk::block_attn_bwd_dkv_kernel<float>), gk, dim3(256), 0, st, a);
  } else {
    const bool fine = a.s.R <= sitk::BLK_FINE_ROWS;
#define SITK_DQ(CAP, FINE) hipLaunchKernelGGL((sitk::block_attn_bwd_dq_ring_kernel<CAP, FINE>), gq, dim3(256), 0, st, a)
    if (small && fine) SITK_DQ(sitk::BLK_LIST, true);
    else if (small) SITK_DQ(sitk::BLK_LIST, false);
    else if (fine) SITK_DQ(sitk::BLK_MAX_TILES, true);
    else SITK_DQ(sitk::BLK_MAX_TILES, false);
#undef SITK_DQ
    SITK_LAUNCH_CHECK("block_attention_bwd dq");
    if (fine) hipLaunchKernelGGL((sitk::block_attn_bwd_dkv_ring_kernel<true>), gk, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((sitk::block_attn_bwd_dkv_ring_kernel<false>), gk, dim3(256), 0, st, a);
  }
  SITK_LAUNCH_CHECK("block_attention_bwd dkv");
  return SITK_OK;
}
