// sitk activations in 8 bits: what a layer keeps for its backward pass, one byte per element and one per group of 32.
// Group of 32 consecutive features of a row: step 2^k with the smallest k such that rint(amax / 2^k) <= 127 (k >= -126; >= -24 when
// the source is IEEE half: half's own step), code = rint(x / 2^k), ties to even.  No code saturates but above 127.5 2^121 = 3.39e38
// (half: 127.5 2^9 = 65280), where k stays 121 (9) -- a larger step would read back as infinity -- and codes end at 127.  In memory a code
// is a signed byte, a step the byte k + 127; a group with an infinity or a NaN has the step byte 255 and reads back as NaN.
// Why a power of two: code * 2^k is exact in bf16, half and f32 (7 bits and a sign), so the weight-gradient product below runs on
// the 16-bit matrix instructions without a second rounding; a byte is decoded by one conversion and one product.
// pack, unpack and the two GELU kernels are bound by HBM: a lane takes 8 elements, a quad a group, nothing else is shared.  Measured: pack of
// 40992 x 768 bf16 20 us (4.7 TB/s); 20544 x 768 half: GELU + pack 22 us (3.6 TB/s; erff's two branches), GELU backward 16 us (4.9 TB/s).
#include "attn_tile.h"

namespace sitk {

constexpr int A8_GROUP = 32;

template <typename T>
struct A8Range { static constexpr int min = 127 - 126, max = 127 + 121; };   // step bytes
#ifdef SITK_TU_F16
template <>
struct A8Range<h16> { static constexpr int min = 127 - 24, max = 127 + 9; };
#endif

SITK_DEV int a8_pad(int cols) { return (cols + A8_GROUP - 1) / A8_GROUP * A8_GROUP; }

// step byte of a group from its largest magnitude: amax = m 2^e, m in [1, 2): k = e - 6, one more when m 2^6 rounds to 128
template <typename T>
SITK_DEV uint32_t a8_step_byte(float amax) {
  const uint32_t u = __builtin_bit_cast(uint32_t, amax);
  if (u >= 0x7F800000u) return 255u;
  const int e = (int)(u >> 23) - 6 + ((u & 0x7FFFFFu) >= 0x7F0000u);  // 0x7F0000: m = 255/128, m 2^6 = 127.5 (tie to even: 128)
  return (uint32_t)min(max(e, A8Range<T>::min), A8Range<T>::max);
}
SITK_DEV float a8_step(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }          // byte 255: infinity
SITK_DEV float a8_inv_step(uint32_t byte) { return __builtin_bit_cast(float, (254u - byte) << 23); }

SITK_DEV float quad_max(float v) {
#define SITK_QP(ctrl) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, 0xf, 0xf, false))
  v = fmaxf(v, SITK_QP(0xB1));   // lanes 1 0 3 2
  v = fmaxf(v, SITK_QP(0x4E));   // lanes 2 3 0 1
#undef SITK_QP
  return v;
}

// 8 elements of a row from column c0; columns >= cols read as zero
template <typename T>
SITK_DEV void a8_load(float (&v)[8], const T* __restrict__ row, int c0, int cols, bool vec) {
  if (vec && c0 + 8 <= cols) {
    const f32x4 a = load4(row + c0), b = load4(row + c0 + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[i + 4] = b[i]; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i < cols ? to_f32(row[c0 + i]) : 0.f;
  }
}
template <typename T>
SITK_DEV void a8_store(T* __restrict__ row, const float (&v)[8], int c0, int cols, bool vec) {
  if (vec && c0 + 8 <= cols) {
    store4(row + c0, f32x4{v[0], v[1], v[2], v[3]});
    store4(row + c0 + 4, f32x4{v[4], v[5], v[6], v[7]});
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + i < cols) row[c0 + i] = from_f32<T>(v[i]);
  }
}

// the 8 codes of a lane; the four lanes of a quad hold one group and agree on its step
template <typename T>
SITK_DEV u32x2 a8_encode(const float (&v)[8], uint32_t& step) {
  float m = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m = fmaxf(m, fabsf(v[i]));
    bad |= v[i] != v[i];                                      // fmaxf drops NaN
  }
  if (bad) m = INFINITY;
  step = a8_step_byte<T>(quad_max(m));
  const float inv = a8_inv_step(min(step, 254u));
  u32x2 o = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float q = step == 255u ? 0.f : __builtin_rintf(v[i] * inv);
    if (step == (uint32_t)A8Range<T>::max) q = fminf(fmaxf(q, -127.f), 127.f);
    o[i >> 2] |= ((uint32_t)(int)q & 255u) << (8 * (i & 3));
  }
  return o;
}
SITK_DEV float a8_code(uint32_t word, int byte) { return (float)(int)(int8_t)(word >> (8 * byte)); }
SITK_DEV void a8_decode(float (&v)[8], u32x2 codes, uint32_t step) {
  const float s = a8_step(step);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = a8_code(codes[i >> 2], i & 3) * s;
}

// Standard normal tail Q(a) = P(X > a), a >= 0, and the density e^(-a^2 / 2) it comes with: erfc as t (a1 + .. + a5 t^4) e^(-x^2) with
// t = 1 / (1 + p x), x = a / sqrt(2) (Abramowitz and Stegun, 7.1.26: off by at most 1.5e-7, half of that in Q).  1 + erf(x) in 32 bits is
// off by as much (6e-8), and costs two branches of a polynomial each, which a wave takes both.  For f32 too: u comes from 8 bits here, off by up to
// half a step, 2^-8 of the largest of its group, so the derivative's last bits are not what limits du.
SITK_DEV float normal_tail(float a, float& e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.23164190f, a, 1.f));        // p / sqrt(2)
  e = fast_exp2(-0.72134752f * a * a);
  return t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5307027145f, -0.7265760135f), 0.7107068705f), -0.142248368f), 0.1274147960f) * e;
}
SITK_DEV float a8_gelu_grad(float u) {                  // Phi(u) + u density(u)
  float e;
  const float q = normal_tail(fabsf(u), e);
  return (u > 0.f ? 1.f - q : q) + u * 0.39894228040f * e;
}

// GELU == false: pack x; true: also g = gelu(x).  One lane = 8 elements, one quad = one group.
template <typename T, bool GELU>
__global__ __launch_bounds__(256) void act8_pack_kernel(const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ codes,
                                                        uint8_t* __restrict__ steps, T* __restrict__ g, int64_t ldg, int cols,
                                                        uint32_t total, int cpr, int vec) {
  const uint32_t id = blockIdx.x * 256u + threadIdx.x;
  if (id >= total) return;
  const uint32_t row = id / (uint32_t)cpr, c = id % (uint32_t)cpr;
  const int c0 = (int)c * 8;
  float v[8];
  a8_load<T>(v, x + (int64_t)row * ldx, c0, cols, vec);
  uint32_t step;
  const u32x2 o = a8_encode<T>(v, step);
  *reinterpret_cast<u32x2*>(codes + (size_t)row * (cpr * 8) + c0) = o;
  if ((c & 3) == 0) steps[(size_t)row * (cpr >> 2) + (c >> 2)] = (uint8_t)step;
  if constexpr (GELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = gelu_erf(v[i]);             // the same bits as GELU without the 8-bit copy
    a8_store<T>(g + (int64_t)row * ldg, v, c0, cols, vec);
  }
}

// GELU == false: y = value of the codes; true: y = dg * gelu'(value)
template <typename T, bool GELU>
__global__ __launch_bounds__(256) void act8_unpack_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ steps,
                                                          const T* __restrict__ dg, int64_t lddg, T* __restrict__ y, int64_t ldy,
                                                          int cols, uint32_t total, int cpr, int vec) {
  const uint32_t id = blockIdx.x * 256u + threadIdx.x;
  if (id >= total) return;
  const uint32_t row = id / (uint32_t)cpr, c = id % (uint32_t)cpr;
  const int c0 = (int)c * 8;
  float v[8];
  a8_decode(v, *reinterpret_cast<const u32x2*>(codes + (size_t)row * (cpr * 8) + c0), steps[(size_t)row * (cpr >> 2) + (c >> 2)]);
  if constexpr (GELU) {
    float d[8];
    a8_load<T>(d, dg + (int64_t)row * lddg, c0, cols, vec);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = d[i] * a8_gelu_grad(v[i]);
  }
  a8_store<T>(y + (int64_t)row * ldy, v, c0, cols, vec);
}

// ------------------------------------------------------------------------------------------
// weight gradient from the 8-bit rows: dW[n][k] = sum_m dY[m][n] X8[m][k], db[n] = sum_m dY[m][n].
// One workgroup = a 64 x 64 tile of dW over one part of the rows; 64 rows at a time of dY and of the decoded X sit in LDS as
// [row][128 bytes] images, read transposed (rows are the contraction).  Parts of the rows are joined in order by a second launch.
// ------------------------------------------------------------------------------------------
struct A8Wgrad {
  const void* dy;
  int64_t lddy;
  const int8_t* codes;
  const uint8_t* steps;
  float *dw, *db;       // split == 1: the result; else the slabs [split][N][K], [split][N]
  int lddw;             // split == 1: of dw; else K
  int M, N, K, rows_per_split, split, accumulate, vec;
};

// 16 x 16 x (rows of one step) products over a stage of STAGE rows; A and B fragments are read transposed from row-major images
template <typename T>
struct A8Geom;
template <>
struct A8Geom<h16> { static constexpr int STAGE = 64; };
template <>
struct A8Geom<float> { static constexpr int STAGE = 32; };

template <typename T>
__global__ __launch_bounds__(256) void act8_wgrad_kernel(A8Wgrad p) {
  constexpr int STAGE = A8Geom<T>::STAGE, PITCH = 64 + 16 / (int)sizeof(T);   // pad: rows start 4 banks apart
  __shared__ __attribute__((aligned(16))) T sy[STAGE * PITCH], sx[STAGE * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fq = lane >> 4;
  const int kt = blockIdx.x * 64, nt = blockIdx.y * 64, z = blockIdx.z;
  const int m0 = z * p.rows_per_split, m1 = min(p.M, m0 + p.rows_per_split);
  const int kp = a8_pad(p.K);
  const T* dy = reinterpret_cast<const T*>(p.dy);
  f32x4 acc[4];
  float bsum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < 4; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int m = m0; m < m1; m += STAGE) {
    __syncthreads();
    for (int i = tid; i < STAGE * 8; i += 256) {                // 8 elements per item
      const int r = i >> 3, c = (i & 7) * 8;
      float v[8];
      if (m + r < m1) a8_load<T>(v, dy + (int64_t)(m + r) * p.lddy, nt + c, p.N, p.vec);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
      a8_store<T>(sy + r * PITCH, v, c, 64, true);
      if (m + r < m1 && kt + c < kp) {
        const size_t o = (size_t)(m + r) * kp + kt + c;
        a8_decode(v, *reinterpret_cast<const u32x2*>(p.codes + o), p.steps[o / A8_GROUP]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
      }
      a8_store<T>(sx + r * PITCH, v, c, 64, true);
    }
    __syncthreads();
    // wave w: rows n = nt + 16 w .. + 15, all 64 columns
#pragma unroll
    for (int r0 = 0; r0 < STAGE; r0 += Mma<T>::KSTEP) {
      typedef __attribute__((ext_vector_type(Mma<T>::EPV))) T vec;
      vec a;
#pragma unroll
      for (int j = 0; j < Mma<T>::EPV; ++j) a[j] = sy[(r0 + Mma<T>::EPV * fq + j) * PITCH + 16 * wave + fr];
      if (kt == 0) {
#pragma unroll
        for (int j = 0; j < Mma<T>::EPV; ++j) bsum[0] += to_f32(a[j]);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        vec b;
#pragma unroll
        for (int j = 0; j < Mma<T>::EPV; ++j) b[j] = sx[(r0 + Mma<T>::EPV * fq + j) * PITCH + 16 * t + fr];
        acc[t] = Mma<T>::mma(__builtin_bit_cast(u32x4, a), __builtin_bit_cast(u32x4, b), acc[t]);
      }
    }
  }
  float* dw = p.split > 1 ? p.dw + (size_t)z * p.N * p.K : p.dw;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = nt + 16 * wave + 4 * fq + j, k = kt + 16 * t + fr;
      if (n < p.N && k < p.K) {
        float* d = dw + (size_t)n * p.lddw + k;
        *d = p.accumulate ? *d + acc[t][j] : acc[t][j];
      }
    }
  if (kt == 0 && p.db) {
    float s = bsum[0];
    s += __shfl_xor(s, 16, 64);
    s += __shfl_xor(s, 32, 64);
    const int n = nt + 16 * wave + fr;
    if (fq == 0 && n < p.N) {
      float* d = p.db + (p.split > 1 ? (size_t)z * p.N : 0) + n;
      *d = p.accumulate ? *d + s : s;
    }
  }
}

// The 16-bit kernel: 256 x 128 tiles of dW, four waves of 128 x 64 (128 accumulator registers: 12 transposed fragments are read for 32
// matrix instructions, where 64 x 64 per wave reads 16 for 32), 32 rows a stage.  dY comes by LDS-DMA through three stages; the codes go
// through registers a stage ahead, are decoded there (each byte once per 256 columns of dY) and written beside it.
// Bound: matrix instructions and the reads that feed them.  40992 rows, 768 -> 2304: 175 us, 830 TFLOP/s (the 64 x 64 kernel 1000 us); 20480
// rows, 612 -> 192: 21 us, its parts' sums leave through HBM (102 parts of 0.47 MB).
constexpr int W8_ROWS = 32, W8_N = 256, W8_K = 128;
constexpr int W8_Y = W8_ROWS * W8_N * 2, W8_X = W8_ROWS * W8_K * 2, W8_STAGES = 3;
__device__ u32x4 g_w8_zero[1];

// four transposed fragments (16 columns each) of the 32-row panel at LDS address `tile`
SITK_DEV void w8_tr4(u32x4 (&f)[4], uint32_t tile, const LaneOffs& lo) {
  u32x2 v[8];
  asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:2048\n\t"
               "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:2048\n\t"
               "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:2048\n\t"
               "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:2048\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
               : "v"(tile + lo.tr[0]), "v"(tile + lo.tr[1]), "v"(tile + lo.tr[2]), "v"(tile + lo.tr[3])
               : "memory");
#pragma unroll
  for (int d = 0; d < 4; ++d) f[d] = u32x4{v[2 * d][0], v[2 * d][1], v[2 * d + 1][0], v[2 * d + 1][1]};
}

__global__ __launch_bounds__(256, 2) void act8_wgrad_big_kernel(A8Wgrad p) {
  __shared__ __attribute__((aligned(256))) char sy[W8_STAGES * W8_Y];
  __shared__ __attribute__((aligned(256))) char sx[W8_STAGES * W8_X];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
  const int wn = wave >> 1, wk = wave & 1;
  const int kts = (p.K + W8_K - 1) / W8_K, nts = (p.N + W8_N - 1) / W8_N;
  const int L = xcd_remap(blockIdx.x, gridDim.x), kt = L % kts, nt = L / kts % nts, z = L / (kts * nts);   // one part's tiles share an XCD
  const int m0 = z * p.rows_per_split, m1 = min(p.M, m0 + p.rows_per_split), stages = (m1 - m0 + W8_ROWS - 1) / W8_ROWS;
  const int kp = a8_pad(p.K);
  // Every load below is issued on every lane whatever the bounds (rows and columns behind the end read a valid place and count zero): so the
  // number of loads in flight is known, and the wait for codes does not wait for the DMA behind them.
  // dY: 16 pieces of 8 rows x 64 columns a stage, four a wave (panel = wave)
  const int yrow = lane >> 3, yn = nt * W8_N + wave * 64 + ((lane & 7) ^ (attn_res_key(yrow) << 1)) * 8;
  const h16* zero = reinterpret_cast<const h16*>(g_w8_zero);
  const h16* yp = reinterpret_cast<const h16*>(p.dy) + (int64_t)(m0 + yrow) * p.lddy + yn;
  int yleft = yn < p.N ? m1 - m0 - yrow : 0;                 // rows of piece 0 and on that this lane still has
  auto issue = [&](int at) {                                // the next stage -> sy + at
    char* dst = sy + at + wave * 4096;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const h16* g = 8 * i < yleft ? yp + (int64_t)(8 * i) * p.lddy : zero;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                       (__attribute__((address_space(3))) void*)(dst + i * 1024), 16, 0, 0);
    }
    yp += (int64_t)W8_ROWS * p.lddy;
    yleft -= W8_ROWS;
  };
  // codes: a thread holds 16 of one row
  const int xrow = tid >> 3, xcol = (tid & 7) * 16;
  const bool xin = kt * W8_K + xcol < kp;
  const int8_t* xp = p.codes + (size_t)m0 * kp + (xin ? kt * W8_K + xcol : 0);
  const uint8_t* sp = p.steps + (size_t)m0 * (kp / A8_GROUP) + (xin ? (kt * W8_K + xcol) / A8_GROUP : 0);
  int xm = xrow;                                            // row of the part
  u32x4 cd;
  uint32_t st;
  auto load = [&]() {                                       // the next stage's codes
    const int m = min(xm, m1 - m0 - 1);
    cd = *reinterpret_cast<const u32x4*>(xp + (size_t)m * kp);
    st = sp[(size_t)m * (kp / A8_GROUP)];
  };
  auto put = [&](int at) {                                  // decoded -> sx + at
    const float f = xin && xm < m1 - m0 ? a8_step(st) : 0.f;
    const bool in = xin && xm < m1 - m0;
    char* dst = sx + at + (xcol >> 6) * 4096;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      h16x8 o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = (h16)(a8_code(cd[2 * h + (i >> 2)], i & 3) * f);
      const u32x4 w = __builtin_bit_cast(u32x4, o);
      *reinterpret_cast<u32x4*>(dst + attn_res_off(xrow, (xcol & 63) * 2 + 16 * h)) = in ? w : u32x4{0u, 0u, 0u, 0u};
    }
    xm += W8_ROWS;
  };
  f32x4 acc[8][4], bias[4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = splat4(0.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) bias[i] = splat4(0.f);
  const bool sums = p.db && kt == 0;                        // wave column wk sums dY's panel wk of this wave row
  const LaneOffs lo = lane_offs_h16(lane);
  const uint32_t ybase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)sy;
  const uint32_t xbase = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)sx;
  const u32x4 ones = {kOnesH16x2, kOnesH16x2, kOnesH16x2, kOnesH16x2};
  load();
  put(0);
  load();
  asm volatile("" ::: "memory");
  issue(0);
  issue(W8_Y);
  int now = 0, next = 1;                                    // stage numbers of s and s + 1
  for (int s = 0; s < stages; ++s) {
    // stage s of dY has landed (this wave's four pieces of stage s + 1 may be in flight), everybody's codes of stage s are written
    asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    put(next * W8_X);
    load();
    asm volatile("" ::: "memory");
    const int last = next == W8_STAGES - 1 ? 0 : next + 1;
    issue(last * W8_Y);
    const uint32_t yt = ybase + now * W8_Y + wn * 8192, xt = xbase + now * W8_X + wk * 4096;
    now = next;
    next = last;
    u32x4 b[4];
    w8_tr4(b, xt, lo);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 a[4];
      w8_tr4(a, yt + h * 4096, lo);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[4 * h + i][j] = Mma<h16>::mma(a[i], b[j], acc[4 * h + i][j]);
      if (sums && h == wk) {
#pragma unroll
        for (int i = 0; i < 4; ++i) bias[i] = Mma<h16>::mma(a[i], ones, bias[i]);
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // nothing may land in LDS that is no longer ours
  float* dw = p.split > 1 ? p.dw + (size_t)z * p.N * p.K : p.dw;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = nt * W8_N + wn * 128 + 16 * i + 4 * fq + e;
      if (n >= p.N) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = kt * W8_K + wk * 64 + 16 * j + fr;
        if (k >= p.K) continue;
        float* d = dw + (size_t)n * p.lddw + k;
        *d = p.accumulate ? *d + acc[i][j][e] : acc[i][j][e];
      }
    }
  if (sums && fr == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = nt * W8_N + wn * 128 + wk * 64 + 16 * i + 4 * fq + e;
        if (n >= p.N) continue;
        float* d = p.db + (p.split > 1 ? (size_t)z * p.N : 0) + n;
        *d = p.accumulate ? *d + bias[i][e] : bias[i][e];
      }
  }
}

// dst[i] (+)= sum over the parts; rows of `cols` floats, leading dimension ld.  The bias rides behind the weights.  WAYS == 4 (many parts of
// few values): a workgroup takes 64 values, its four waves a quarter of the parts each, joined in order.  Eight loads in flight.
template <int WAYS>
__global__ __launch_bounds__(256) void act8_join_kernel(const float* __restrict__ slab, float* __restrict__ dst, float* __restrict__ db,
                                                        int64_t rows, int cols, int ld, int split, int accumulate) {
  constexpr int PER = 256 / WAYS;
  __shared__ float part[WAYS][PER];
  const int at = threadIdx.x % PER, way = threadIdx.x / PER;
  const int64_t n = rows * cols, all = n + (db ? rows : 0);
  const int z0 = split * way / WAYS, z1 = split * (way + 1) / WAYS;
  for (int64_t i0 = (int64_t)blockIdx.x * PER; i0 < all; i0 += (int64_t)gridDim.x * PER) {
    const int64_t i = i0 + at;
    float s = 0.f;
    if (i < all) {
      const float* src = i < n ? slab + i : slab + split * n + (i - n);
      const int64_t step = i < n ? n : rows;
#pragma unroll 8
      for (int z = z0; z < z1; ++z) s += src[z * step];
    }
    if constexpr (WAYS > 1) {
      part[way][at] = s;
      __syncthreads();
      if (way == 0) s = (part[0][at] + part[1][at]) + (part[2][at] + part[3][at]);
    }
    if (way == 0 && i < all) {
      float* d = i < n ? dst + i / cols * ld + i % cols : db + (i - n);
      *d = accumulate ? *d + s : s;
    }
    if constexpr (WAYS > 1) __syncthreads();
  }
}

// What a call launches: the 256 x 128 kernel when dY can be read 16 bytes at a time, else (and f32) the 64 x 64 one; the rows in parts so
// that there are two workgroups per CU (four of the small ones), at least four stages each.
struct A8Plan {
  bool big;
  int split, rows_per_split;
};
static A8Plan act8_plan(int64_t M, int N, int K, int dtype, bool vec) {
  A8Plan r{};
  r.big = dtype != SITK_F32 && vec && N % 8 == 0;
  const int stage = dtype == SITK_F32 || r.big ? 32 : 64;
  const int64_t tiles = r.big ? (int64_t)cdiv(N, W8_N) * cdiv(K, W8_K) : (int64_t)cdiv(N, 64) * cdiv(K, 64), stages = cdiv64(M, stage);
  int64_t s = (r.big ? 512 : 1024) / tiles;
  if (s > stages / 4) s = stages / 4;
  r.split = (int)(s < 1 ? 1 : s > 128 ? 128 : s);
  r.rows_per_split = (int)(cdiv64(stages < 1 ? 1 : stages, r.split) * stage);
  r.split = (int)cdiv64(M < 1 ? 1 : M, r.rows_per_split);  // parts without rows are not launched
  return r;
}

}  // namespace sitk

extern "C" size_t sitk_act8_code_bytes(int64_t rows, int cols) {
  return rows < 0 || cols < 1 ? 0 : (size_t)rows * ((size_t)(cols + 31) / 32 * 32);
}
extern "C" size_t sitk_act8_step_bytes(int64_t rows, int cols) {
  return rows < 0 || cols < 1 ? 0 : (size_t)rows * ((size_t)(cols + 31) / 32);
}

#define A8_COMMON(name, rows, cols, dtype)                                                                                   \
  SITK_REQUIRE((rows) >= 0 && (cols) >= 1, name ": bad sizes rows=%lld cols=%d", (long long)(rows), (cols));                 \
  SITK_REQUIRE((dtype) == SITK_F32 || (dtype) == SITK_BF16 || (dtype) == SITK_F16, name ": unknown dtype %d", (dtype));      \
  SITK_REQUIRE((rows) * (int64_t)cdiv((cols), 32) * 4 < (int64_t)0xFFFFFF00, name ": %lld x %d: too large for one call",     \
               (long long)(rows), (cols))
#define A8_CODES(name, codes) SITK_REQUIRE((uintptr_t)(codes) % 16 == 0, name ": codes are not 16-byte aligned")
#define A8_LD(name, ld, cols) SITK_REQUIRE((ld) >= (cols), name ": leading dimension %lld < %d", (long long)(ld), (cols))
// rows that can be read `n` elements at a time
static inline int a8_vec(const void* p, int64_t ld, int es, int n = 4) { return (uintptr_t)p % (n * es) == 0 && ld % n == 0; }

#define A8_LAUNCH(K, GELU, ...)                                                                                              \
  do {                                                                                                                       \
    const int cpr = cdiv(cols, 32) * 4;                                                                                      \
    const uint32_t total = (uint32_t)(rows * cpr);                                                                           \
    const dim3 grid((unsigned)cdiv64(total, 256)), block(256);                                                               \
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);                                                                   \
    if (dtype == SITK_F32) { typedef float T; hipLaunchKernelGGL((sitk::K<float, GELU>), grid, block, 0, s, __VA_ARGS__); }  \
    else { typedef h16 T; hipLaunchKernelGGL((sitk::K<h16, GELU>), grid, block, 0, s, __VA_ARGS__); }                        \
  } while (0)

SITK_F16_TWIN(sitk_act8_pack)
extern "C" int sitk_act8_pack(const void* x, int64_t ldx, int8_t* codes, uint8_t* steps, int64_t rows, int cols, int dtype,
                              sitk_stream_t stream) {
  SITK_REQUIRE(x && codes && steps, "act8_pack: null pointer");
  A8_COMMON("act8_pack", rows, cols, dtype);
  A8_CODES("act8_pack", codes);
  A8_LD("act8_pack", ldx, cols);
  if (rows == 0) return SITK_OK;
  SITK_FORWARD_F16(dtype, sitk_act8_pack, x, ldx, codes, steps, rows, cols, dtype, stream);
  const int vec = a8_vec(x, ldx, dtype == SITK_F32 ? 4 : 2);
  A8_LAUNCH(act8_pack_kernel, false, reinterpret_cast<const T*>(x), ldx, codes, steps, (T*)nullptr, (int64_t)0, cols, total, cpr, vec);
  SITK_LAUNCH_CHECK("act8_pack");
  return SITK_OK;
}

SITK_F16_TWIN(sitk_act8_gelu_fwd)
extern "C" int sitk_act8_gelu_fwd(const void* u, int64_t ldu, void* g, int64_t ldg, int8_t* codes, uint8_t* steps, int64_t rows,
                                  int cols, int dtype, sitk_stream_t stream) {
  SITK_REQUIRE(u && g && codes && steps, "act8_gelu_fwd: null pointer");
  A8_COMMON("act8_gelu_fwd", rows, cols, dtype);
  A8_CODES("act8_gelu_fwd", codes);
  A8_LD("act8_gelu_fwd", ldu, cols);
  A8_LD("act8_gelu_fwd", ldg, cols);
  if (rows == 0) return SITK_OK;
  SITK_FORWARD_F16(dtype, sitk_act8_gelu_fwd, u, ldu, g, ldg, codes, steps, rows, cols, dtype, stream);
  const int es = dtype == SITK_F32 ? 4 : 2, vec = a8_vec(u, ldu, es) && a8_vec(g, ldg, es);
  A8_LAUNCH(act8_pack_kernel, true, reinterpret_cast<const T*>(u), ldu, codes, steps, reinterpret_cast<T*>(g), ldg, cols, total, cpr, vec);
  SITK_LAUNCH_CHECK("act8_gelu_fwd");
  return SITK_OK;
}

SITK_F16_TWIN(sitk_act8_unpack)
extern "C" int sitk_act8_unpack(const int8_t* codes, const uint8_t* steps, void* y, int64_t ldy, int64_t rows, int cols, int dtype,
                                sitk_stream_t stream) {
  SITK_REQUIRE(y && codes && steps, "act8_unpack: null pointer");
  A8_COMMON("act8_unpack", rows, cols, dtype);
  A8_CODES("act8_unpack", codes);
  A8_LD("act8_unpack", ldy, cols);
  if (rows == 0) return SITK_OK;
  SITK_FORWARD_F16(dtype, sitk_act8_unpack, codes, steps, y, ldy, rows, cols, dtype, stream);
  const int vec = a8_vec(y, ldy, dtype == SITK_F32 ? 4 : 2);
  A8_LAUNCH(act8_unpack_kernel, false, codes, steps, (const T*)nullptr, (int64_t)0, reinterpret_cast<T*>(y), ldy, cols, total, cpr, vec);
  SITK_LAUNCH_CHECK("act8_unpack");
  return SITK_OK;
}

SITK_F16_TWIN(sitk_act8_gelu_bwd)
extern "C" int sitk_act8_gelu_bwd(const void* dg, int64_t lddg, const int8_t* codes, const uint8_t* steps, void* du, int64_t lddu,
                                  int64_t rows, int cols, int dtype, sitk_stream_t stream) {
  SITK_REQUIRE(dg && du && codes && steps, "act8_gelu_bwd: null pointer");
  A8_COMMON("act8_gelu_bwd", rows, cols, dtype);
  A8_CODES("act8_gelu_bwd", codes);
  A8_LD("act8_gelu_bwd", lddg, cols);
  A8_LD("act8_gelu_bwd", lddu, cols);
  if (rows == 0) return SITK_OK;
  SITK_FORWARD_F16(dtype, sitk_act8_gelu_bwd, dg, lddg, codes, steps, du, lddu, rows, cols, dtype, stream);
  const int es = dtype == SITK_F32 ? 4 : 2, vec = a8_vec(dg, lddg, es) && a8_vec(du, lddu, es);
  A8_LAUNCH(act8_unpack_kernel, true, codes, steps, reinterpret_cast<const T*>(dg), lddg, reinterpret_cast<T*>(du), lddu, cols, total, cpr, vec);
  SITK_LAUNCH_CHECK("act8_gelu_bwd");
  return SITK_OK;
}

// the larger need of the two kernels: which one runs depends on dY's alignment
extern "C" size_t sitk_act8_wgrad_ws_bytes(int64_t M, int N, int K, int dtype) {
  if (M < 1 || N < 1 || K < 1) return 0;
  const int s0 = sitk::act8_plan(M, N, K, dtype, false).split, s1 = sitk::act8_plan(M, N, K, dtype, true).split, s = s0 > s1 ? s0 : s1;
  return s > 1 ? (size_t)s * N * ((size_t)K + 1) * 4 : 0;
}

SITK_F16_TWIN(sitk_act8_wgrad)
extern "C" int sitk_act8_wgrad(const void* dy, int64_t lddy, const int8_t* codes, const uint8_t* steps, float* dw, int lddw, float* db,
                               int64_t M, int N, int K, int accumulate, void* ws, size_t ws_bytes, int dtype, sitk_stream_t stream) {
  SITK_REQUIRE(dw, "act8_wgrad: null pointer");
  SITK_REQUIRE(M >= 0 && M < ((int64_t)1 << 31) - 8192 && N >= 1 && K >= 1 && K <= (1 << 30), "act8_wgrad: bad sizes M=%lld N=%d K=%d", (long long)M, N, K);
  SITK_REQUIRE(M == 0 || (dy && codes && steps), "act8_wgrad: null pointer");
  SITK_REQUIRE(((uintptr_t)codes | (uintptr_t)ws) % 16 == 0, "act8_wgrad: codes and workspace must be 16-byte aligned");
  SITK_REQUIRE(dtype == SITK_F32 || dtype == SITK_BF16 || dtype == SITK_F16, "act8_wgrad: unknown dtype %d", dtype);
  SITK_REQUIRE(lddw >= K && (M == 0 || lddy >= N), "act8_wgrad: leading dimension too small");
  SITK_REQUIRE(cdiv(N, 64) < 65536, "act8_wgrad: N=%d too large", N);
  SITK_FORWARD_F16(dtype, sitk_act8_wgrad, dy, lddy, codes, steps, dw, lddw, db, M, N, K, accumulate, ws, ws_bytes, dtype, stream);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const size_t need = sitk_act8_wgrad_ws_bytes(M, N, K, dtype);
  SITK_REQUIRE(ws_bytes >= need && (ws || need == 0), "act8_wgrad: workspace of %zu bytes, %zu needed", ws_bytes, need);
  if (M == 0) {                                              // no product kernel, which would look for a first row: a join of no parts
    if (accumulate) return SITK_OK;
    const int64_t blocks = cdiv64((int64_t)N * K + N, 256);
    hipLaunchKernelGGL(sitk::act8_join_kernel<1>, dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, s, (const float*)nullptr, dw, db,
                       (int64_t)N, K, lddw, 0, 0);
    SITK_LAUNCH_CHECK("act8_wgrad join");
    return SITK_OK;
  }
  const int vec = a8_vec(dy, lddy, dtype == SITK_F32 ? 4 : 2, dtype == SITK_F32 ? 4 : 8);
  const sitk::A8Plan plan = sitk::act8_plan(M, N, K, dtype, vec);
  sitk::A8Wgrad p{};
  p.dy = dy; p.lddy = lddy; p.codes = codes; p.steps = steps;
  p.M = (int)M; p.N = N; p.K = K; p.split = plan.split; p.rows_per_split = plan.rows_per_split; p.vec = vec;
  float* slab = reinterpret_cast<float*>(ws);
  const int64_t n = (int64_t)N * K;
  if (plan.split > 1) { p.dw = slab; p.lddw = K; p.db = db ? slab + (size_t)plan.split * n : nullptr; }
  else { p.dw = dw; p.lddw = lddw; p.db = db; p.accumulate = accumulate; }
  if (plan.big) {
    const dim3 grid((unsigned)(cdiv(K, sitk::W8_K) * cdiv(N, sitk::W8_N) * plan.split));
    hipLaunchKernelGGL(sitk::act8_wgrad_big_kernel, grid, dim3(256), 0, s, p);
  } else {
    const dim3 grid(cdiv(K, 64), cdiv(N, 64), plan.split);
    if (dtype == SITK_F32) hipLaunchKernelGGL((sitk::act8_wgrad_kernel<float>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((sitk::act8_wgrad_kernel<h16>), grid, dim3(256), 0, s, p);
  }
  SITK_LAUNCH_CHECK("act8_wgrad");
  if (plan.split > 1) {
    // four ways from 32 parts on: 117 k values in 102 parts 24 -> 10 us; 1.8 M values in 9 parts 16 us against 24
    const int ways = plan.split >= 32 ? 4 : 1;
    const int64_t blocks = cdiv64(n + N, 256 / ways);
    const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384)), block(256);
    if (ways == 4) hipLaunchKernelGGL(sitk::act8_join_kernel<4>, grid, block, 0, s, slab, dw, db, (int64_t)N, K, lddw, plan.split, accumulate);
    else hipLaunchKernelGGL(sitk::act8_join_kernel<1>, grid, block, 0, s, slab, dw, db, (int64_t)N, K, lddw, plan.split, accumulate);
    SITK_LAUNCH_CHECK("act8_wgrad join");
  }
  return SITK_OK;
}
