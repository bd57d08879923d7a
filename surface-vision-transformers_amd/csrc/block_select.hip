// sitk selection of key blocks by a cheap score (what it is for: block_attention.hip).
//   pool    kbar[j] = mean of the valid keys of block j, summed in 64 bits and kept in 32
//   select  the top_k blocks of every query row by q . kbar[j], ties to the lower block, blocks without a valid key left out
//
// The selection is exact: a row's blocks are those that scores in 64 bits would give, so nothing depends on how a product is summed.
// Scores in 32 bits come from the matrix instructions (kbar = hi + mid + lo in three 16-bit planes, the hi products summed apart, so
// that only their 64 terms round at the size of the score: |error| <= 2^-17 |q| |kbar|); a row whose border -- the gap between its
// top_k-th and its next score -- lies inside twice that bound is scored again in 64 bits by its wave.  With random scores that is one row
// in a few hundred; equal scores (copied blocks, a query of zeros) always take that way.  Only the blocks inside the bound of the border
// are scored there (with all of the row's blocks: 183 instead of 167 us at 2 x 20481 rows, 6 heads).
//
// Layout: a wave owns 16 rows; matrix tile i gives lane l the scores of row l & 15 with blocks 16 i + 4 (l >> 4) + 0..3, so a row is spread
// over four lanes and the whole search for its threshold (count the scores at or above a guess, move the guess between the two
// nearest known counts by their logarithms) runs in registers for 16 rows at once.  The planes pass through LDS, 64 blocks at a time, for
// the four waves of a workgroup.  Above 640 blocks (BLK_MAX_NB are allowed) the registers do not hold the scores and every row goes in 64 bits:
// 81921 rows, 6 heads, 18.3 ms with 1281 blocks of 64 keys, 0.28 ms with 321 of 256 -- long sequences want larger blocks.
// Bound: vector issue (search and bits; the products are 20 us of the 156 at 2 x 20481 rows, 6 heads, 321 blocks, bf16); 32 x 1281 rows, 21 blocks:
// 39 us.  pool: HBM; 32 x 1281 keys, 6 heads 12 us (2.5 TB/s: a workgroup has one 8 KB block to load and join), 16 x 20481 keys, 3 heads 25 us (5.0 TB/s).
#include "block_common.h"

namespace sitk {

// sum over the lanes that share lane % WIDTH (8 or 16), without LDS: with shuffles through it pool of 32 x 1281 keys, 6 heads took 16 us instead of 13
template <int WIDTH>
SITK_DEV double stride_sum(double v) {
  auto halves = [](double d, float& lo, float& hi) {
    const uint64_t u = __builtin_bit_cast(uint64_t, d);
    lo = __builtin_bit_cast(float, (uint32_t)u);
    hi = __builtin_bit_cast(float, (uint32_t)(u >> 32));
  };
  auto whole = [](float lo, float hi) {
    return __builtin_bit_cast(double, (uint64_t)__builtin_bit_cast(uint32_t, lo) | (uint64_t)__builtin_bit_cast(uint32_t, hi) << 32);
  };
  float lo, hi, lo2, hi2;
  if constexpr (WIDTH == 8) {
    halves(v, lo, hi);
#define SITK_ROR8(x) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, false))
    v += whole(SITK_ROR8(lo), SITK_ROR8(hi));
#undef SITK_ROR8
  }
  halves(v, lo, hi);
  lo2 = lo; hi2 = hi;
  permlane16_swap(lo, lo2);
  permlane16_swap(hi, hi2);
  v = whole(lo, hi) + whole(lo2, hi2);
  halves(v, lo, hi);
  lo2 = lo; hi2 = hi;
  permlane32_swap(lo, lo2);
  permlane32_swap(hi, hi2);
  return whole(lo, hi) + whole(lo2, hi2);
}

// one workgroup per (sample, key head, block): a lane sums 16 bytes of features over every (rows per load)-th key
template <typename T>
__global__ __launch_bounds__(256) void block_pool_kernel(const T* __restrict__ k, Rows ks, const uint8_t* __restrict__ key_mask,
                                                         int64_t mask_b, BlkPool p, BlkShape s) {
  constexpr int EPV = 16 / (int)sizeof(T), CPR = 64 / EPV, RPL = 64 / CPR;   // features per load, lanes per key, keys per wave and load
  __shared__ double part[4][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, ch = lane % CPR, kr = lane / CPR;
  const int L = xcd_remap(blockIdx.x, gridDim.x), hk = L % s.Hk, j = L / s.Hk % s.nb, b = L / (s.nb * s.Hk);   // heads of a token lie together
  const int k0 = j * s.c * 64;
  const T* kb = k + (int64_t)b * ks.b + (int64_t)hk * ks.h + ch * EPV;
  int n = 0;
  double sum[EPV];
#pragma unroll
  for (int e = 0; e < EPV; ++e) sum[e] = 0.0;
  constexpr int LOADS = 64 / (4 * RPL);
  typedef __attribute__((ext_vector_type(EPV))) T vec;
#pragma unroll 2
  for (int t = 0; t < s.c && k0 + 64 * t < s.Nk; ++t) {
    const int kt = k0 + 64 * t;
    vec v[LOADS];                                            // all loads first, of a row in range whether it is valid or not
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      v[i] = *reinterpret_cast<const vec*>(kb + (int64_t)min(kt + (i * 4 + wave) * RPL + kr, s.Nk - 1) * ks.n);
    const bool ok = kt + lane < s.Nk && (!key_mask || key_mask[(int64_t)b * mask_b + kt + lane]);
    const uint64_t bits = __ballot(ok);
    n += __popcll(bits);
    if (hk == 0 && tid == 0) p.kbits[(int64_t)b * s.nt + j * s.c + t] = bits;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const bool in = bits >> ((i * 4 + wave) * RPL + kr) & 1;
#pragma unroll
      for (int e = 0; e < EPV; ++e) sum[e] += in ? (double)to_f32(v[i][e]) : 0.0;
    }
  }
#pragma unroll
  for (int e = 0; e < EPV; ++e) {
    sum[e] = stride_sum<CPR>(sum[e]);
    if (kr == 0) part[wave][ch * EPV + e] = sum[e];
  }
  const int64_t bh = (int64_t)b * s.Hk + hk, plane = (int64_t)s.B * s.Hk * s.nbp * 64;
  auto write = [&](int jj, float m, float norm, int count) {
    const int64_t o = (bh * s.nbp + jj) * 64 + lane;
    p.pooled[o] = m;
    if constexpr (sizeof(T) == 2) {
      const h16 hi = (h16)m, mid = (h16)(m - (float)hi);
      p.planes[o] = hi;
      p.planes[o + plane] = mid;
      p.planes[o + 2 * plane] = (h16)(m - (float)hi - (float)mid);
    }
    if (lane == 0) p.norm[bh * s.nbp + jj] = norm;
    if (hk == 0 && lane == 0) p.count[(int64_t)b * s.nbp + jj] = count;
  };
  if (j == s.nb - 1)                                         // the last block also clears the rows behind it
    for (int jj = s.nb + wave; jj < s.nbp; jj += 4) write(jj, 0.f, 0.f, 0);
  __syncthreads();
  if (wave) return;
  const double t = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
  const float m = n ? (float)(t / n) : 0.f;
  const float nn = wave_sum(m * m);
  write(j, m, sqrtf(nn) * 1.00001f, n);
}

// the four lanes that share lane & 15
SITK_DEV uint32_t or4(uint32_t v) {
  float a = __builtin_bit_cast(float, v), b = a;
  permlane16_swap(a, b);
  a = b = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, a) | __builtin_bit_cast(uint32_t, b));
  permlane32_swap(a, b);
  return __builtin_bit_cast(uint32_t, a) | __builtin_bit_cast(uint32_t, b);
}
SITK_DEV int add4(int v) {
  float a = __builtin_bit_cast(float, v), b = a;
  permlane16_swap(a, b);
  a = b = __builtin_bit_cast(float, __builtin_bit_cast(int, a) + __builtin_bit_cast(int, b));
  permlane32_swap(a, b);
  return __builtin_bit_cast(int, a) + __builtin_bit_cast(int, b);
}
// the two largest of four lanes' two largest (a >= b in each)
SITK_DEV void top2(float& a, float& b) {
  float a2 = a, b2 = b;
  permlane16_swap(a, a2);
  permlane16_swap(b, b2);
  b = fmaxf(fminf(a, a2), fmaxf(b, b2));
  a = fmaxf(a, a2);
  a2 = a; b2 = b;
  permlane32_swap(a, a2);
  permlane32_swap(b, b2);
  b = fmaxf(fminf(a, a2), fmaxf(b, b2));
  a = fmaxf(a, a2);
}
SITK_DEV float uniform_lane(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }
SITK_DEV void lds_fence() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// words[64 rows][pitch] (LDS, one bit per block) -> both layouts of the selection bits
SITK_DEV void emit_bits(const uint32_t* words, int pitch, uint64_t* __restrict__ mask, const BlkShape& s, int bh, int rt, int wave, int lane) {
  const size_t half = (size_t)s.B * s.Hk * s.nrt * s.nb;
  for (int w = wave; 32 * w < s.nb; w += 4) {
    const uint32_t v = words[lane * pitch + w];
    uint64_t out = 0;
#pragma unroll
    for (int b = 0; b < 32; ++b) {
      const uint64_t bal = __ballot(v >> b & 1);
      if (lane == b) out = bal;
    }
    const int j = 32 * w + lane;
    if (lane < 32 && j < s.nb) {
      mask[((size_t)bh * s.nrt + rt) * s.nb + j] = out;
      mask[half + ((size_t)bh * s.nb + j) * s.nrt + rt] = out;
    }
  }
}

// Scores in 64 bits as integers of the same order (0: no candidate); the `want` largest of a wave's 64 NV are found by halving a range
// with wave-wide counts: the range around `thr`, which the scores in 32 bits know to within `near`, or all of it (near < 0, or the border is
// not inside).  What is left at the end of the range are equal scores, of which the first are taken.  bits[i]: taken of v[i].
SITK_DEV uint64_t order64(double x) {
  if (x != x) x = INFINITY;                                  // a NaN score is the largest: the output then shows it
  x = x > -1.7e308 ? x + 0.0 : -1.7e308;                     // a live block is never -inf, and never -0
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return u ^ ((uint64_t)((int64_t)u >> 63) | (1ull << 63));
}
template <int NV>
SITK_DEV void pick64(const uint64_t (&v)[NV], uint64_t (&bits)[NV], int groups, int want, float thr, float near) {
  auto reach = [&](uint64_t at) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i < groups) n += __popcll(__ballot(v[i] >= at));
    return n;
  };
  uint64_t lo = 1, hi = ~0ull;                               // reached by more than wanted; by fewer
  if (reach(lo) > want) {
    if (near >= 0.f) {
      const uint64_t a = order64((double)thr - near), b = order64((double)thr + near);
      if (reach(a) > want && reach(b) < want) { lo = a; hi = b; }
    }
    while (hi - lo > 1) {
      const uint64_t mid = lo + (hi - lo) / 2;
      const int n = reach(mid);
      if (n >= want) lo = mid;
      if (n <= want) hi = mid;                               // as many as wanted: both, and nothing is left between
    }
  } else {
    hi = lo;
  }
  int left = hi == lo ? 0 : want - reach(hi);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    bits[i] = 0;
    if (i >= groups) continue;
    bits[i] = __ballot(v[i] >= hi);
    for (uint64_t equal = hi == lo ? 0 : __ballot(v[i] == lo); equal && left > 0; equal &= equal - 1, --left) bits[i] |= equal & (~equal + 1);
  }
}
template <int UNROLL>
SITK_DEV double dot64(const float* qv, const float* __restrict__ key) {
  const f32x4* kb = reinterpret_cast<const f32x4*>(key);
  double t[2] = {0.0, 0.0};
#pragma unroll(UNROLL)
  for (int d = 0; d < 16; ++d) {
    const f32x4 kk = kb[d];
#pragma unroll
    for (int e = 0; e < 4; ++e) t[d & 1] += (double)qv[4 * d + e] * (double)kk[e];
  }
  return t[0] + t[1];
}
// a row with all its blocks in 64 bits: bits of blocks 32 l .. + 31 in lane l.  NV: blocks per lane
template <int NV>
SITK_DEV uint32_t select_row64(const float* qv, const float* __restrict__ pooled, const int* __restrict__ count, int nb, int top_k, int lane) {
  uint64_t v[NV], bits[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    v[i] = 0;
    if (64 * i >= nb) continue;
    const int j = lane + 64 * i;                             // rows behind nb are there, and zero
    const uint64_t x = order64(dot64<4>(qv, pooled + (int64_t)j * 64));
    if (count[j]) v[i] = x;
  }
  pick64<NV>(v, bits, (nb + 63) / 64, top_k, 0.f, -1.f);
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (lane >> 1 == i) word = (uint32_t)(bits[i] >> (32 * (lane & 1)));
  return word;
}

constexpr int SEL_STAGE = 3 * 8192;      // 64 blocks of three planes, rows of 128 bytes
// NG: groups of 64 blocks whose scores are held in registers (0: every row in 64 bits, up to 2048 blocks)
template <typename T, int NG>
__global__ __launch_bounds__(256, NG > 6 ? 2 : 3) void block_select_kernel(const T* __restrict__ q, Rows qs, BlkPool p, int* __restrict__ index,
                                                                         uint64_t* __restrict__ mask, int top_k, BlkShape s) {
  using Gm = AttnGeom<T>;
  constexpr int WMAX = NG ? NG * 2 : BLK_MAX_NB / 32, PITCH = WMAX | 1, NV = NG ? NG : BLK_MAX_NB / 64, NT = 4 * NG;
  __shared__ uint32_t words[64 * PITCH];
  // the scores' stages; after them the waves' own parts
  constexpr int SEL_WAVE = 256 + 128 + 16 * PITCH * 4;       // of a wave: a query row, the list and the bits of its candidates
  __shared__ __attribute__((aligned(256))) char stage[NG > 0 && sizeof(T) == 2 ? (NG > 1 ? 2 : 1) * SEL_STAGE : 4 * SEL_WAVE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
  const int L = xcd_remap(blockIdx.x, gridDim.x), rt = L % s.nrt, bh = L / s.nrt, hk = bh % s.Hk, b = bh / s.Hk;
  const int r = rt * 64 + 16 * wave + fr, rc = min(r, s.R - 1), W = (s.nb + 31) / 32;
  const T* qb = q + (int64_t)b * qs.b;
  const float* pooled = p.pooled + (int64_t)bh * s.nbp * 64;
  const int* count = p.count + (int64_t)b * s.nbp;
  bool again = r < s.R;                                      // this row goes the 64-bit way
  bool few = false;                                          // .. with the blocks whose scores are near its border
  float thr = 0.f, near = -1.f;                              // the border lies within near of thr (near < 0: anywhere)
  char* own = stage + wave * SEL_WAVE;
  float* qrow = reinterpret_cast<float*>(own);
  uint16_t* list = reinterpret_cast<uint16_t*>(own + 256);
  uint32_t* cand = reinterpret_cast<uint32_t*>(own + 384);   // [16 rows][PITCH]
  if constexpr (NG > 0) {
    const int64_t plane = (int64_t)s.B * s.Hk * s.nbp * 64;
    auto issue = [&](int g) {                                // group g -> its stage: 24 pieces of 8 rows, six a wave
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 6; ++i) {
          const int pc = wave * 6 + i, row = (pc & 7) * 8 + (lane >> 3);
          const h16* src = p.planes + (pc >> 3) * plane + ((int64_t)bh * s.nbp + 64 * g + row) * 64 + ((lane & 7) ^ (attn_res_key(row) << 1)) * 8;
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                           (__attribute__((address_space(3))) void*)(stage + (g & 1) * SEL_STAGE + pc * 1024), 16, 0, 0);
        }
      }
    };
    issue(0);
    const T* qp = qb + q_row(qs, s, hk, rc);
    u32x4 qf[Gm::KS];
    float qq = 0.f, kn = 0.f;
    uint64_t live[NG];                                       // blocks with a valid key
    int alive = 0;
#pragma unroll
    for (int ks = 0; ks < Gm::KS; ++ks) {
      qf[ks] = *reinterpret_cast<const u32x4*>(qp + (ks * 64 + fq * 16) / (int)sizeof(T));
      typedef __attribute__((ext_vector_type(Gm::EPV))) T vec;
      const vec v = __builtin_bit_cast(vec, qf[ks]);
#pragma unroll
      for (int e = 0; e < Gm::EPV; ++e) qq += to_f32(v[e]) * to_f32(v[e]);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      live[g] = 0;
      if (64 * g >= s.nb) continue;
      live[g] = __ballot(count[64 * g + lane] > 0);
      kn = fmaxf(kn, p.norm[(int64_t)bh * s.nbp + 64 * g + lane]);
      alive += __popcll(live[g]);
    }
    kn = wave_max(kn);
    const float qn = sqrtf(xor_sum4(qq));
    const LaneOffs lo_ = lane_offs_h16(lane);
    const uint32_t lbase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)stage;
    f32x4 sc[NT];
    float lo = INFINITY, hi = -INFINITY, sum = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int t = 0; t < 4; ++t) sc[4 * g + t] = splat4(-INFINITY);
      if (64 * g >= s.nb) continue;
      f32x4 a0[4], a1[4];
      if constexpr (sizeof(T) == 2) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");   // group g has landed, group g - 1 is read
        if (64 * (g + 1) < s.nb) issue(g + 1);
        const uint32_t at = lbase + (g & 1) * SEL_STAGE;
        u32x4 kf[4][2];
        SITK_RING_ROWS8(kf, at + lo_.row[0], at + lo_.row[1], 16384);
#pragma unroll
        for (int t = 0; t < 4; ++t) a1[t] = Mma<T>::mma(kf[t][0], qf[0], splat4(0.f));
#pragma unroll
        for (int t = 0; t < 4; ++t) a1[t] = Mma<T>::mma(kf[t][1], qf[1], a1[t]);
        SITK_RING_ROWS8(kf, at + lo_.row[0], at + lo_.row[1], 8192);
#pragma unroll
        for (int t = 0; t < 4; ++t) a1[t] = Mma<T>::mma(kf[t][0], qf[0], a1[t]);
#pragma unroll
        for (int t = 0; t < 4; ++t) a1[t] = Mma<T>::mma(kf[t][1], qf[1], a1[t]);
        SITK_RING_ROWS8(kf, at + lo_.row[0], at + lo_.row[1], 0);
#pragma unroll
        for (int t = 0; t < 4; ++t) a0[t] = Mma<T>::mma(kf[t][0], qf[0], splat4(0.f));
#pragma unroll
        for (int t = 0; t < 4; ++t) a0[t] = Mma<T>::mma(kf[t][1], qf[1], a0[t]);
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          a0[t] = a1[t] = splat4(0.f);
#pragma unroll
          for (int ks = 0; ks < Gm::KS; ++ks)
            a0[t] = Mma<T>::mma(*reinterpret_cast<const u32x4*>(pooled + (int64_t)(64 * g + 16 * t + fr) * 64 + ks * 16 + fq * 4), qf[ks], a0[t]);
        }
      }
      if (live[g] == ~0ull) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const f32x4 v = a0[t] + a1[t];
          sc[4 * g + t] = v;
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) { lo = fminf(lo, v[jj]); hi = fmaxf(hi, v[jj]); sum += v[jj]; }
        }
      } else {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const f32x4 v = a0[t] + a1[t];
          const uint32_t nib = (uint32_t)(live[g] >> (16 * t + 4 * fq));
#pragma unroll
          for (int jj = 0; jj < 4; ++jj)
            if (nib >> jj & 1) { sc[4 * g + t][jj] = v[jj]; lo = fminf(lo, v[jj]); hi = fmaxf(hi, v[jj]); sum += v[jj]; }
        }
      }
    }
    lo = -xor_max4(-lo);
    hi = xor_max4(hi);
    sum = xor_sum4(sum);
    // 2^-17 |q| |kbar| per score; half planes end at 2^-24 (subnormal): 2^-25 sum |q| <= 2^-22 |q| more
    const float bound = qn * (kn * 0x1p-17f + (SITK_H16 == SITK_F16 ? 0x1p-22f : 0.f));
    // A NaN or an infinity among the scores, or no bound for them: all blocks again.  The bound needs squares and products inside the range of
    // 32 bits.  Squares of finite |q| or |kbar| above 1.8e19 are not; below 1e37 it keeps `below` above the -infinity of blocks without a
    // valid key, which are no candidates then.  Small ones underflow: from norms of 2^-60 and a bound of 2^-100 on, what flushed planes (2^-126
    // each), products and squares lose is far inside the bound.  So near > 0 wherever a score is not, and no more than top_k are sure.
    const bool odd = !(fabsf(sum) < 1e38f) || !(hi < 3e38f) || !(lo > -3e38f) || !(bound < 1e37f) || !(bound > 0x1p-100f) ||
                     !(fminf(qn, kn) > 0x1p-60f);
    bool found = alive <= top_k, done = found || odd || r >= s.R;
    thr = -INFINITY;
    int reached = top_k;                                     // scores at or above thr
    float clo = (float)alive, chi = 0.f;    // scores at or above lo; above hi
    const float want = __log2f((float)top_k);
    for (int it = 0; it < 48 && __any(!done); ++it) {
      // between the two known counts by their logarithms (a tail of scores falls off like that), late ones in the middle
      const float a = __log2f(clo), c = __log2f(fmaxf(chi, 0.5f)), mid = 0.5f * lo + 0.5f * hi;
      float next = it < 10 ? lo + (hi - lo) * fminf(fmaxf((a - want) / (a - c), 0.1f), 0.9f) : mid;
      if (!(next > lo) || !(next < hi)) next = mid;
      if (!done) {
        thr = next;
        done = !(next > lo) || !(next < hi);                 // equal scores at the border
      }
      int n = 0;
#pragma unroll
      for (int i = 0; i < NT; ++i)
        if (16 * i < s.nb)
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) n += sc[i][jj] >= thr;
      n = add4(n);
      if (!done) {
        reached = n;
        if ((uint32_t)(n - top_k + 1) <= 2u) done = found = true;       // top_k, or one off: settled below
        else if (n > top_k) { lo = thr; clo = (float)n; }
        else { hi = thr; chi = (float)n; }
      }
    }
    // the two lowest scores at or above thr and the two highest below: the border, also where thr reaches one too many or too few (on average
    // half as many rounds as until it reaches top_k: a wave waits for the slowest of its 16 rows)
    float in = INFINITY, in2 = INFINITY, out = -INFINITY, out2 = -INFINITY;
#pragma unroll
    for (int i = 0; i < NT; ++i)
      if (16 * i < s.nb)
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          const bool t = sc[i][jj] >= thr;
          const float x = t ? sc[i][jj] : INFINITY, y = t ? -INFINITY : sc[i][jj];
          in2 = __builtin_amdgcn_fmed3f(x, in, in2);
          in = fminf(in, x);
          out2 = __builtin_amdgcn_fmed3f(y, out, out2);
          out = fmaxf(out, y);
        }
    float lo1 = -in, lo2 = -in2;
    top2(lo1, lo2);
    top2(out, out2);
    in = -lo1; in2 = -lo2;
    float gap = in - out;
    if (alive > top_k) {
      thr = in;                                              // now the score of rank top_k
      if (reached > top_k) { gap = in2 - in; thr = in2; }
      if (reached < top_k) { gap = out - out2; thr = out; }
    }
    again = r < s.R && (odd || !found || (alive > top_k && !(gap > 2.0f * bound)));
    const bool take = r < s.R && found && !again;
    // The score of rank top_k is thr (not found: from lo up to hi), in 64 bits at most `bound` away.  So a block more than 2 bound above is
    // taken, one as far below is not, and only those between are scored again.
    few = again && !odd;
    near = 2.25f * bound;
    const float above = (found ? thr : hi) + near, below = (found ? thr : lo) - near;
    if (found) near = fmaxf(near, 1e-30f);
    else near = -1.f;
    // blocks without a valid key have the score -infinity
    const float from = take ? fmaxf(thr, -3.4e38f) : few ? above : NAN;
    __syncthreads();                                         // every wave is done with the stages
    const bool any = __any(few);
#pragma unroll
    for (int w = 0; w < WMAX; ++w) {
      uint32_t v = 0, u = 0;
#pragma unroll
      for (int ii = 0; ii < 2; ++ii)
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) v |= sc[2 * w + ii][jj] >= from ? 1u << (16 * ii + jj) : 0u;
      v = or4(v << (4 * fq));
      if (fq == 0) words[(16 * wave + fr) * PITCH + w] = v;
      if (any) {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int ii = 0; ii < 2; ++ii)
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) u |= few && sc[2 * w + ii][jj] >= below && sc[2 * w + ii][jj] < from ? 1u << (16 * ii + jj) : 0u;
        u = or4(u << (4 * fq));
        if (fq == 0) cand[fr * PITCH + w] = u;
      }
    }
  } else {
    for (int w = fq; w < W; w += 4) words[(16 * wave + fr) * PITCH + w] = 0;
  }
  lds_fence();
  for (uint32_t todo = (uint32_t)(__ballot(again) & 0xFFFF); todo; todo &= todo - 1) {
    const int i = __ffs((int)todo) - 1, rr = rt * 64 + 16 * wave + i;
    uint32_t* row = words + (16 * wave + i) * PITCH;
    qrow[lane] = to_f32(qb[q_row(qs, s, hk, rr) + lane]);
    int n = 0, sure = 0;
    if (__builtin_amdgcn_readlane(few, i)) {
      for (int w = 0; w < W; ++w) {                          // the candidates in order
        const uint32_t v = __builtin_amdgcn_readfirstlane(cand[i * PITCH + w]);
        sure += __popc(__builtin_amdgcn_readfirstlane(row[w]));
        const int at = n + __popc(v & ((1u << (lane & 31)) - 1));
        if (lane < 32 && v >> lane & 1 && at < 64) list[at] = (uint16_t)(32 * w + lane);
        n += __popc(v);
      }
    }
    lds_fence();
    if (n > 0 && n <= 64) {
      const int j = list[min(lane, n - 1)];
      uint64_t v[1] = {order64(dot64<16>(qrow, pooled + (int64_t)j * 64))}, bits[1];
      if (lane >= n) v[0] = 0;
      pick64<1>(v, bits, 1, top_k - sure, uniform_lane(thr, i), uniform_lane(near, i));
      if (bits[0] >> lane & 1) atomicOr(row + (j >> 5), 1u << (j & 31));
    } else {
      const uint32_t w = select_row64<NV>(qrow, pooled, count, s.nb, top_k, lane);
      if (lane < W) row[lane] = w;
    }
    lds_fence();
  }
  lds_fence();
  if (r < s.R) {                                             // four lanes write a row's index, word by word in turn
    int* dst = index + q_flat(s, b, hk, r) * top_k;
    const uint32_t* row = words + (16 * wave + fr) * PITCH;
    int at = 0;
    for (int w = 0; w < W; ++w) {
      uint32_t v = row[w];
      if ((w & 3) == fq)
        for (int o = at; v; v &= v - 1) dst[o++] = 32 * w + __ffs((int)v) - 1;
      at += __popc(row[w]);
    }
    for (int o = at + fq; o < top_k; o += 4) dst[o] = -1;
  }
  __syncthreads();
  emit_bits(words, PITCH, mask, s, bh, rt, wave, lane);
}

// bits of a selection that the caller made: entries outside [0, nb) select nothing, an entry twice counts once
__global__ __launch_bounds__(256) void block_mask_kernel(const int* __restrict__ index, uint64_t* __restrict__ mask, int top_k, BlkShape s) {
  constexpr int PITCH = (BLK_MAX_NB / 32) | 1;
  __shared__ uint32_t words[64 * PITCH];
  const int tid = threadIdx.x, rt = blockIdx.x % s.nrt, bh = blockIdx.x / s.nrt, hk = bh % s.Hk, b = bh / s.Hk;
  for (int i = tid; i < 64 * PITCH; i += 256) words[i] = 0;
  __syncthreads();
  const int r = rt * 64 + tid;
  if (tid < 64 && r < s.R) {
    const int* src = index + q_flat(s, b, hk, r) * top_k;
    for (int i = 0; i < top_k; ++i) {
      const int j = src[i];
      if (j >= 0 && j < s.nb) words[tid * PITCH + (j >> 5)] |= 1u << (j & 31);
    }
  }
  __syncthreads();
  emit_bits(words, PITCH, mask, s, bh, rt, tid >> 6, tid & 63);
}

template <typename T>
static int select_launch(const void* q, const Rows& qs, const BlkPool& p, int* index, uint64_t* mask, int top_k, const BlkShape& s, hipStream_t st) {
  const dim3 grid((unsigned)(s.B * s.Hk * s.nrt)), block(256);
  const T* qp = reinterpret_cast<const T*>(q);
  const int ng = s.nbp / 64;
#define SITK_SELECT(NG) hipLaunchKernelGGL((block_select_kernel<T, NG>), grid, block, 0, st, qp, qs, p, index, mask, top_k, s)
  if (ng <= 1) SITK_SELECT(1);
  else if (ng <= 2) SITK_SELECT(2);
  else if (ng <= 6) SITK_SELECT(6);
  else if (ng <= 10) SITK_SELECT(10);
  else SITK_SELECT(0);
#undef SITK_SELECT
  SITK_LAUNCH_CHECK("block_select");
  return SITK_OK;
}

}  // namespace sitk

extern "C" size_t sitk_block_pool_bytes(int B, int Nk, int Hk, int block, int dtype) {
  if (B < 1 || Nk < 1 || Hk < 1 || block < 64) return 0;
  return sitk::blk_pool_at(nullptr, sitk::blk_shape(B, 1, Nk, Hk, Hk, block), dtype).bytes;
}
extern "C" size_t sitk_block_mask_words(int B, int Nq, int Nk, int H, int Hk, int block) {
  if (B < 1 || Nq < 1 || Nk < 1 || Hk < 1 || H < Hk || H % Hk || block < 64) return 0;
  return 2 * sitk::blk_mask_words(sitk::blk_shape(B, Nq, Nk, H, Hk, block));
}

SITK_F16_TWIN(sitk_block_pool)
extern "C" int sitk_block_pool(const void* k, const sitk_block_rows* ks, const uint8_t* key_mask, int64_t mask_b, void* pool, int B,
                               int Nk, int Hk, int block, int dtype, sitk_stream_t stream) {
  SITK_TRY(sitk::blk_check("block_pool", B, 1, Nk, Hk, Hk, block, dtype));
  SITK_REQUIRE(ks && pool && (uintptr_t)pool % 16 == 0, "block_pool: null or unaligned pointer");
  SITK_TRY(sitk::blk_rows("block_pool", "k", k, *ks, dtype));
  SITK_FORWARD_F16(dtype, sitk_block_pool, k, ks, key_mask, mask_b, pool, B, Nk, Hk, block, dtype, stream);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const sitk::BlkShape s = sitk::blk_shape(B, 1, Nk, Hk, Hk, block);
  const sitk::BlkPool p = sitk::blk_pool_at(pool, s, dtype);
  const dim3 grid((unsigned)(B * Hk * s.nb));
  if (dtype == SITK_F32)
    hipLaunchKernelGGL((sitk::block_pool_kernel<float>), grid, dim3(256), 0, st, reinterpret_cast<const float*>(k), sitk::to_rows(*ks), key_mask, mask_b, p, s);
  else
    hipLaunchKernelGGL((sitk::block_pool_kernel<h16>), grid, dim3(256), 0, st, reinterpret_cast<const h16*>(k), sitk::to_rows(*ks), key_mask, mask_b, p, s);
  SITK_LAUNCH_CHECK("block_pool");
  return SITK_OK;
}

SITK_F16_TWIN(sitk_block_select)
extern "C" int sitk_block_select(const void* q, const sitk_block_rows* qs, const void* pool, int* index, uint64_t* mask, int B, int Nq,
                                 int Nk, int H, int Hk, int block, int top_k, int dtype, sitk_stream_t stream) {
  SITK_TRY(sitk::blk_check("block_select", B, Nq, Nk, H, Hk, block, dtype));
  SITK_REQUIRE(top_k >= 1, "block_select: top_k = %d", top_k);
  SITK_REQUIRE(qs && pool && index && mask && (uintptr_t)pool % 16 == 0, "block_select: null or unaligned pointer");
  SITK_TRY(sitk::blk_rows("block_select", "q", q, *qs, dtype));
  SITK_FORWARD_F16(dtype, sitk_block_select, q, qs, pool, index, mask, B, Nq, Nk, H, Hk, block, top_k, dtype, stream);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const sitk::BlkShape s = sitk::blk_shape(B, Nq, Nk, H, Hk, block);
  const sitk::BlkPool p = sitk::blk_pool_at(const_cast<void*>(pool), s, dtype);
  if (dtype == SITK_F32) return sitk::select_launch<float>(q, sitk::to_rows(*qs), p, index, mask, top_k, s, st);
  return sitk::select_launch<h16>(q, sitk::to_rows(*qs), p, index, mask, top_k, s, st);
}

extern "C" int sitk_block_mask(const int* index, uint64_t* mask, int B, int Nq, int Nk, int H, int Hk, int block, int top_k,
                               sitk_stream_t stream) {
  SITK_TRY(sitk::blk_check("block_mask", B, Nq, Nk, H, Hk, block, SITK_F32));
  SITK_REQUIRE(top_k >= 1 && index && mask, "block_mask: null pointer or top_k = %d", top_k);
  const sitk::BlkShape s = sitk::blk_shape(B, Nq, Nk, H, Hk, block);
  hipLaunchKernelGGL(sitk::block_mask_kernel, dim3((unsigned)(B * Hk * s.nrt)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), index,
                     mask, top_k, s);
  SITK_LAUNCH_CHECK("block_mask");
  return SITK_OK;
}
