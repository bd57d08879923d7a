// sitk attention over selected key blocks: the shapes and host checks that the selection (block_select.hip) and the attention
// (block_attention.hip) share.
#pragma once
#include "attn_tile.h"

namespace sitk {

constexpr int BLK_MAX_NB = 2048;       // blocks of one sequence (select: 16 rows' scores in a wave's registers up to 640, above them row by row in 64 bits)
constexpr int BLK_MAX_TILES = 4096;    // 64-key tiles of one sequence (the attention kernels list a row tile's key tiles in LDS)

struct BlkShape {
  int B, Nq, Nk, H, Hk, G, R, Rp, nrt; // R = Nq G rows per key head, Rp: rounded up to 64, nrt: 64-row tiles
  int nt, c, nb, nbp;                  // 64-key tiles, tiles per block, blocks, blocks rounded up to 64
};
static inline BlkShape blk_shape(int B, int Nq, int Nk, int H, int Hk, int block) {
  BlkShape s{};
  s.B = B; s.Nq = Nq; s.Nk = Nk; s.H = H; s.Hk = Hk; s.G = H / Hk; s.R = Nq * s.G; s.nrt = cdiv(s.R, 64); s.Rp = s.nrt * 64;
  s.nt = cdiv(Nk, 64); s.c = block / 64; s.nb = cdiv(Nk, block); s.nbp = cdiv(s.nb, 64) * 64;
  return s;
}

// The pool: one allocation, every part 256-byte aligned.
struct BlkPool {
  float* pooled;      // (B, Hk, nbp, 64) means, rows behind nb zero
  float* norm;        // (B, Hk, nbp) their 2-norms, rounded up
  int* count;         // (B, nbp) valid keys
  uint64_t* kbits;    // (B, nt) valid-key bits
  h16* planes;        // (3, B Hk, nbp, 64) pooled as a sum of three 16-bit values (16-bit types only)
  size_t bytes;
};
static inline BlkPool blk_pool_at(void* base, const BlkShape& s, int dtype) {
  BlkPool p{};
  char* at = reinterpret_cast<char*>(base);
  size_t o = 0;
  const size_t bh = (size_t)s.B * s.Hk;
  auto take = [&](size_t n) { char* r = at + o; o += align_up(n, 256); return r; };
  p.pooled = reinterpret_cast<float*>(take(bh * s.nbp * 64 * 4));
  p.norm = reinterpret_cast<float*>(take(bh * s.nbp * 4));
  p.count = reinterpret_cast<int*>(take((size_t)s.B * s.nbp * 4));
  p.kbits = reinterpret_cast<uint64_t*>(take((size_t)s.B * s.nt * 8));
  p.planes = reinterpret_cast<h16*>(take(dtype == SITK_F32 ? 0 : 3 * bh * s.nbp * 64 * 2));
  p.bytes = o;
  return p;
}

// The selection as bits: bit i of [bh][rt][j] = row 64 rt + i selected block j; behind it the same as [bh][j][rt].
static inline size_t blk_mask_words(const BlkShape& s) { return (size_t)s.B * s.Hk * s.nrt * s.nb; }

struct Rows {                       // (sample, token, head) strides in elements; the 64 features are contiguous
  int64_t b, n, h;
};
// row r of key head hk in a tensor of query rows
SITK_DEV int64_t q_row(const Rows& st, const BlkShape& s, int hk, int r) {
  if (s.G == 1) return (int64_t)r * st.n + (int64_t)hk * st.h;
  const int n = (int)((uint32_t)r / (uint32_t)s.G), g = r - n * s.G;
  return (int64_t)n * st.n + (int64_t)(hk * s.G + g) * st.h;
}
// flat index of row r in the contiguous (B, H, Nq) arrays (lse, index)
SITK_DEV int64_t q_flat(const BlkShape& s, int b, int hk, int r) {
  const int n = s.G == 1 ? r : (int)((uint32_t)r / (uint32_t)s.G), g = s.G == 1 ? 0 : r - n * s.G;
  return ((int64_t)b * s.H + hk * s.G + g) * s.Nq + n;
}

static int blk_check(const char* who, int B, int Nq, int Nk, int H, int Hk, int block, int dtype) {
  SITK_REQUIRE(B >= 1 && Nq >= 1 && Nk >= 1 && H >= 1 && Hk >= 1, "%s: bad sizes B=%d Nq=%d Nk=%d H=%d Hk=%d", who, B, Nq, Nk, H, Hk);
  SITK_REQUIRE(H % Hk == 0, "%s: %d query heads do not share %d key heads", who, H, Hk);
  SITK_REQUIRE(block >= 64 && block % 64 == 0 && block <= 1024, "%s: block of %d keys (a multiple of 64, at most 1024)", who, block);
  SITK_REQUIRE(cdiv(Nk, block) <= BLK_MAX_NB, "%s: %d blocks (at most %d: take a larger block)", who, cdiv(Nk, block), BLK_MAX_NB);
  SITK_REQUIRE(cdiv(Nk, 64) <= BLK_MAX_TILES, "%s: %d keys (at most %d)", who, Nk, 64 * BLK_MAX_TILES);
  const int64_t R = (int64_t)Nq * (H / Hk), nrt = cdiv64(R, 64);
  SITK_REQUIRE(R < ((int64_t)1 << 30), "%s: %lld query rows per key head: too many", who, (long long)R);
  SITK_REQUIRE((int64_t)B * H < (1 << 24) && (int64_t)B * Hk * nrt < ((int64_t)1 << 30) && (int64_t)B * Hk * cdiv(Nk, 64) < ((int64_t)1 << 30),
               "%s: B * heads * tiles too large for one call", who);
  SITK_REQUIRE(dtype == SITK_F32 || dtype == SITK_BF16 || dtype == SITK_F16, "%s: unknown dtype %d", who, dtype);
  return SITK_OK;
}
static int blk_rows(const char* who, const char* what, const void* p, const sitk_block_rows& st, int dtype) {
  const int v = 16 / (dtype == SITK_F32 ? 4 : 2);
  SITK_REQUIRE(p && (uintptr_t)p % 16 == 0, "%s: %s is null or not 16-byte aligned", who, what);
  SITK_REQUIRE(st.n >= 0 && st.n < (1 << 23), "%s: token stride %lld of %s (at most 2^23 elements)", who, (long long)st.n, what);
  SITK_REQUIRE(st.b % v == 0 && st.n % v == 0 && st.h % v == 0, "%s: strides of %s are not multiples of 16 bytes", who, what);
  return SITK_OK;
}
static inline Rows to_rows(const sitk_block_rows& r) { return Rows{r.b, r.n, r.h}; }

}  // namespace sitk
