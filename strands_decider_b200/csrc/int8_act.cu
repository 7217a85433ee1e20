// Int8 codes with one fp32 scale per row: of an activation or a weight (b200_quantize_act_int8,
// b200_quantize), and of a residual stream's RMSNorm (b200_rmsnorm_int8).
//
// Codes of a row v: a = max |v|, scale = a / 127, q = rint(v * (127 / a)), each operation one
// fp32 rounding, so the codes are the same for every split of a row over threads; the norm's sum
// of squares is taken in fp64, where the order of its additions does not show after the one
// rounding of (S / hidden + eps)^-1/2 to fp32 (and no finite input overflows it). The maximum is
// taken over the bit patterns of |v| as integers: a NaN or infinity then is the largest, and the
// row gets scale NaN.
//
// Every row is read once: its elements stay in the registers of the threads that share it while
// the sum, the maximum and the codes follow one another. Bound by HBM where there are rows enough:
// norm 65536 x 2048 108 us = 6.2 TB/s (117 us a launch in a run of 5000), 12288 x 2048
// with an fp32 delta 50.7 us = 6.5 TB/s; codes of 65536 x 6144 bf16 174 us = 6.9 TB/s, of 12288 x
// 2048 two planes 19.4 us = 6.5 TB/s; one row is a chain of latencies, 2.0 us of norm (2048), 1.5 of
// codes (6144).
#include "common.cuh"

namespace sdb {

constexpr int I8_K_MAX = 65536;          // also keeps b200_linear_int8's sums below 2^31
constexpr int I8_ROWS_MAX = 1 << 30;     // counts of rows and tiles then fit 32 bits after rounding up

// The reductions of one row over its TPR threads: a group of 8 lanes, a warp, or a whole block.
template <int TPR>
__device__ __forceinline__ uint32_t row_lanes() {
  return TPR >= 32 ? 0xffffffffu : ((1u << TPR) - 1u) << (threadIdx.x & 31 & ~(TPR - 1));
}
template <int TPR>
__device__ __forceinline__ double row_sum(double v, double* part) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(row_lanes<TPR>(), v, o);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) v += part[i];
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* part) {
  v = __reduce_max_sync(row_lanes<TPR>(), v);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0u;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) v = max(v, part[i]);
  }
  return v;
}

// |v| as a double, put together from its bits: the conversion instruction runs at a quarter of the
// rate that these do and took 70 of 185 us at 65536 x 2048. Zeros and subnormals come out as
// numbers below 2^-126, whose squares (2^-252) are far below the last bit of any eps > 0 they are
// added to; an infinity or NaN comes out finite, and its row is marked by v itself. (The high word
// by a multiplication with addend: 16384 x 8192 108 us, by shift, mask and addition 114.)
__device__ __forceinline__ double abs_double(float v) {
  const uint32_t b = __float_as_uint(v) << 1;  // without the sign
  return __hiloint2double(int(__umulhi(b, 1u << 28) + 0x38000000u), int(b << 28));  // b >> 4, and the bias
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// A row's scale from the bits of its largest |v|, and the factor of its codes (0: all codes 0).
__device__ __forceinline__ void row_scale(uint32_t amax_bits, float& scale, float& inv) {
  scale = inv = 0.0f;
  if (amax_bits >= 0x7f800000u) {
    scale = __uint_as_float(0x7fc00000u);
    return;
  }
  const float a = __uint_as_float(amax_bits), s = __fdiv_rn(a, 127.0f);
  if (s < 1.1754943508222875e-38f) return;  // 2^-126
  scale = s;
  inv = __fdiv_rn(127.0f, a);
}

// Four codes. A product is at most 127 (1 + 2^-23), so adding 1.5 x 2^23 rounds it to a whole number,
// ties to even, whose low byte is the sum's; the conversion instruction runs at a quarter of the
// rate (norm 65536 x 2048 117 -> 109 us, codes of 12072 x 2400 bf16 19.0 -> 16.9). inv 0 gives codes
// 0, products that are NaN too.
__device__ __forceinline__ uint32_t code_bits(float v, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.0f));
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv) {
  const uint32_t lo = __byte_perm(code_bits(a, inv), code_bits(b, inv), 0x0040);
  const uint32_t q = __byte_perm(lo, __byte_perm(code_bits(c, inv), code_bits(d, inv), 0x0040), 0x5410);
  return inv != 0.0f ? q : 0u;
}

constexpr int ACT_NONE = -1, ACT_PLANES = 2;  // beside B200_ACT_F32 and B200_ACT_BF16

struct RowArgs {
  const void* x;        // quantise: fp32 or bf16; norm: fp32
  const uint16_t* lo;   // quantise: the low plane
  const void* delta;    // norm
  float* sum;           // norm
  const float* w;       // norm
  int8_t* q;
  float* scale;
  int ldx, ldd, lds, ldq;
  int rows, k;
  float eps;
};

// Rows per block of TPR threads each, and the block's threads.
template <int TPR>
constexpr int rows_per_block() { return TPR <= 32 ? 256 / TPR : 1; }
template <int TPR>
constexpr int row_threads() { return TPR * rows_per_block<TPR>(); }
template <int TPR>
__device__ __forceinline__ int row_of() {
  return int(blockIdx.x) * rows_per_block<TPR>() + int(threadIdx.x) / TPR;
}

// TPR threads per row, NV float4 per thread (k <= 4 TPR NV).
template <int TPR, int NV, int DELTA>
__global__ void __launch_bounds__(row_threads<TPR>()) rmsnorm_int8_kernel(const RowArgs a) {
  __shared__ double psum[TPR > 32 ? TPR / 32 : 1];
  __shared__ uint32_t pmax[TPR > 32 ? TPR / 32 : 1];
  pdl_wait();
  pdl_trigger();
  const int row = row_of<TPR>(), t = threadIdx.x % TPR;
  if (row >= a.rows) return;
  const int n4 = a.k / 4;
  const float4* xr = reinterpret_cast<const float4*>(static_cast<const float*>(a.x) + size_t(row) * a.ldx);
  float4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = t + TPR * i;
    v[i] = j < n4 ? xr[j] : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if constexpr (DELTA != ACT_NONE) {
    // every load before the first store: `sum` may be x or delta
    float4 d[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = t + TPR * i;
      d[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if constexpr (DELTA == B200_ACT_F32) {
        if (j < n4) d[i] = reinterpret_cast<const float4*>(static_cast<const float*>(a.delta) + size_t(row) * a.ldd)[j];
      } else {
        uint2 b = make_uint2(0u, 0u);
        if (j < n4) b = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.delta) + size_t(row) * a.ldd)[j];
        d[i] = make_float4(bf16x2_lo(b.x), bf16x2_hi(b.x), bf16x2_lo(b.y), bf16x2_hi(b.y));
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = make_float4(v[i].x + d[i].x, v[i].y + d[i].y, v[i].z + d[i].z, v[i].w + d[i].w);
    if (a.sum) {
      float4* sr = reinterpret_cast<float4*>(a.sum + size_t(row) * a.lds);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = t + TPR * i;
        if (j < n4) sr[j] = v[i];
      }
    }
  }
  double s0 = 0.0, s1 = 0.0, s2 = 0.0, s3 = 0.0;  // four chains: an fp64 FMA waits on the one before
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    s0 = fma(abs_double(v[i].x), abs_double(v[i].x), s0);
    s1 = fma(abs_double(v[i].y), abs_double(v[i].y), s1);
    s2 = fma(abs_double(v[i].z), abs_double(v[i].z), s2);
    s3 = fma(abs_double(v[i].w), abs_double(v[i].w), s3);
  }
  const double ss = row_sum<TPR>((s0 + s1) + (s2 + s3), psum);
  const float r = float(rsqrt(ss / double(a.k) + double(a.eps)));
  uint32_t mx = 0u;
  auto scaled = [&](float4& u, const float4& w) {
    u.x = __fmul_rn(__fmul_rn(u.x, r), 1.0f + w.x);
    u.y = __fmul_rn(__fmul_rn(u.y, r), 1.0f + w.y);
    u.z = __fmul_rn(__fmul_rn(u.z, r), 1.0f + w.z);
    u.w = __fmul_rn(__fmul_rn(u.w, r), 1.0f + w.w);
    mx = max(max(max(mx, abs_bits(u.x)), abs_bits(u.y)), max(abs_bits(u.z), abs_bits(u.w)));
  };
  const float4* wr = reinterpret_cast<const float4*>(a.w);
  // A warp's weights in batches, whose loads are in flight together (3844 x 784 9.0 -> 6.4 us, 20000 x
  // 1392 39.7 -> 32.6). Not of its longest rows, whose registers they would take (65536 x 2048: 202 us
  // against 116 at the time), and not in blocks of a row, of which enough are resident (28162 x 2512 73 : 68).
  constexpr int B = TPR > 32 || NV > 12 ? 1 : NV % 4 == 0 ? 4 : NV % 3 == 0 ? 3 : NV;
#pragma unroll
  for (int i0 = 0; i0 < NV; i0 += B) {
    if constexpr (B == 1) {
      const int j = t + TPR * i0;
      if (j < n4) scaled(v[i0], __ldg(wr + j));
    } else {
      float4 w[B];
#pragma unroll
      for (int i = 0; i < B; ++i) {
        const int j = t + TPR * (i0 + i);
        w[i] = j < n4 ? __ldg(wr + j) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int i = 0; i < B; ++i) scaled(v[i0 + i], w[i]);  // past the row's end: zeros
    }
  }
  mx = row_max<TPR>(mx, pmax);
  float scale, inv;
  row_scale(mx, scale, inv);
  if (t == 0) a.scale[row] = scale;
  uint32_t* qr = reinterpret_cast<uint32_t*>(a.q + size_t(row) * a.ldq);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = t + TPR * i;
    if (j < n4) qr[j] = codes4(v[i].x, v[i].y, v[i].z, v[i].w, inv);
  }
}

// TPR threads per row, NV groups of 4 (fp32) or 8 (bf16) elements per thread.
template <int TPR, int NV, int TYPE>
__global__ void __launch_bounds__(row_threads<TPR>()) quantize_int8_kernel(const RowArgs a) {
  constexpr int E = TYPE == B200_ACT_F32 ? 4 : 8;
  __shared__ uint32_t pmax[TPR > 32 ? TPR / 32 : 1];
  pdl_wait();
  pdl_trigger();
  const int row = row_of<TPR>(), t = threadIdx.x % TPR;
  if (row >= a.rows) return;
  const int ng = a.k / E;
  // all of the row's loads first
  uint4 raw[NV], low[TYPE == ACT_PLANES ? NV : 1];
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  const uint4* xr = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.x) + size_t(row) * a.ldx * (16 / E));
#pragma unroll
  for (int i = 0; i < NV; ++i) raw[i] = t + TPR * i < ng ? xr[t + TPR * i] : zero;
  if constexpr (TYPE == ACT_PLANES) {
    const uint4* lr = reinterpret_cast<const uint4*>(a.lo + size_t(row) * a.ldx);
#pragma unroll
    for (int i = 0; i < NV; ++i) low[i] = t + TPR * i < ng ? lr[t + TPR * i] : zero;
  }
  float v[NV][E];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t hw[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    if constexpr (TYPE == B200_ACT_F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = __uint_as_float(hw[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[i][2 * e] = bf16x2_lo(hw[e]);
        v[i][2 * e + 1] = bf16x2_hi(hw[e]);
      }
      if constexpr (TYPE == ACT_PLANES) {
        const uint32_t lw[4] = {low[i].x, low[i].y, low[i].z, low[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[i][2 * e] += bf16x2_lo(lw[e]);
          v[i][2 * e + 1] += bf16x2_hi(lw[e]);
        }
      }
    }
  }
  uint32_t mx = 0u;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) mx = max(mx, abs_bits(v[i][e]));
  mx = row_max<TPR>(mx, pmax);
  float scale, inv;
  row_scale(mx, scale, inv);
  if (t == 0) a.scale[row] = scale;
  int8_t* qr = a.q + size_t(row) * a.ldq;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = t + TPR * i;
    if (j < ng) {
      const uint32_t c = codes4(v[i][0], v[i][1], v[i][2], v[i][3], inv);
      if constexpr (E == 4)
        reinterpret_cast<uint32_t*>(qr)[j] = c;
      else
        reinterpret_cast<uint2*>(qr)[j] = make_uint2(c, codes4(v[i][4], v[i][5], v[i][6], v[i][7], inv));
    }
  }
}

// Threads per row and 16-byte groups per thread, for `units` groups a row. The fewest threads that
// hold the row in `cap` groups each: a warp's reductions need no barrier and all of its loads are
// in flight at once, but a row that comes in two arrays fills the registers sooner (planes at 12288
// x 2048: 19.5 us with 128 threads a row, 22.1 with 32; an fp32 delta at 12288 x 2048: 50.6 against
// 59.2; no delta at 65536 x 2048: 116 us with 32, 123 with 128, both before codes were rounded by an
// addition; 108 since). Four times as many while the
// device has under 512 threads per SM and the row has work for them (1 x 2048: 2.1 us against 2.5).
// Rows of at most 32 groups take 8 lanes, four rows to a warp. A thread's groups are 1, 2, 3, 4, 6, 8,
// 12 or 16: registers for twice as many as the row has would leave fewer rows in flight (codes of
// 65536 x 6144 bf16 in 8 groups 209 us, in 6 174; of 12072 x 2400 30.6 : 18.8).
struct RowShape {
  int tpr, nv;
};
constexpr int next_nv(int nv) { return nv == 3 ? 4 : nv == 6 ? 8 : nv == 12 ? 16 : nv + (nv + 1) / 2; }
static RowShape row_shape(int rows, int units, int cap) {
  int tpr = units <= 32 ? 8 : 32;
  while (tpr < 512 && (units > cap * tpr || (int64_t(rows) * tpr < 512 * int64_t(sm_count()) && units > tpr))) tpr *= 4;
  if (units > 16 * tpr) tpr = 1024;
  int nv = 1;
  while (nv * tpr < units) nv = next_nv(nv);
  return {tpr, nv};
}
template <bool NORM, int KIND>
constexpr int row_cap() { return NORM ? (KIND == ACT_NONE ? 16 : 8) : (KIND == ACT_PLANES ? 4 : 16); }

template <bool NORM, int KIND, int TPR, int NV>
static int launch_nv(const RowArgs& a, int nv, cudaStream_t st) {
  if (nv == NV) {
    constexpr int rpb = rows_per_block<TPR>();
    const dim3 grid((a.rows + rpb - 1) / rpb), block(row_threads<TPR>());
    if constexpr (NORM) SDB_CUDA(launch_pdl(rmsnorm_int8_kernel<TPR, NV, KIND>, grid, block, 0, st, a));
    else SDB_CUDA(launch_pdl(quantize_int8_kernel<TPR, NV, KIND>, grid, block, 0, st, a));
    return B200_OK;
  }
  // groups that row_shape gives a thread: 8 lanes hold at most 32, 32 and 128 threads the cap each
  constexpr int most = TPR == 8 ? 4 : TPR >= 512 ? 16 : row_cap<NORM, KIND>();
  if constexpr (next_nv(NV) <= most) return launch_nv<NORM, KIND, TPR, next_nv(NV)>(a, nv, st);
  else return sdb_fail(B200_ERR_SHAPE, "int8 rows: no such shape");
}
template <bool NORM, int KIND>
static int launch_rows(const RowArgs& a, cudaStream_t st) {
  constexpr int E = NORM || KIND == B200_ACT_F32 ? 4 : 8;
  const RowShape r = row_shape(a.rows, a.k / E, row_cap<NORM, KIND>());
  switch (r.tpr) {
    case 8: return launch_nv<NORM, KIND, 8, 1>(a, r.nv, st);
    case 32: return launch_nv<NORM, KIND, 32, 1>(a, r.nv, st);
    case 128: return launch_nv<NORM, KIND, 128, 1>(a, r.nv, st);
    case 512: return launch_nv<NORM, KIND, 512, 1>(a, r.nv, st);
    default:  // rows that no block of 512 holds
      if constexpr (I8_K_MAX / E > 16 * 512) return launch_nv<NORM, KIND, 1024, 16>(a, 16, st);
      else return sdb_fail(B200_ERR_SHAPE, "int8 rows: no such shape");
  }
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int sdb_quantize_int8(const void* x, const uint16_t* x_lo, int32_t type, int32_t rows, int32_t k, int32_t ldx,
                      int8_t* q, int32_t ldq, float* scale, cudaStream_t st) {
  if (!x || !q || !scale) return sdb_fail(B200_ERR_ARG, "b200_quantize_act_int8: null pointer");
  if (type != B200_ACT_F32 && type != B200_ACT_BF16)
    return sdb_fail(B200_ERR_ARG, "b200_quantize_act_int8: unknown activation type");
  if (x_lo && type != B200_ACT_BF16)
    return sdb_fail(B200_ERR_ARG, "b200_quantize_act_int8: a low plane belongs to bf16 activations");
  if (rows <= 0 || k <= 0) return sdb_fail(B200_ERR_SHAPE, "b200_quantize_act_int8: empty shape");
  if (rows > I8_ROWS_MAX) return sdb_fail(B200_ERR_SHAPE, "b200_quantize_act_int8: more than 2^30 rows");
  if (k % 16 != 0 || k > I8_K_MAX)
    return sdb_fail(B200_ERR_SHAPE, "b200_quantize_act_int8: k must be a multiple of 16, at most 65536");
  if (ldx < k || ldx % (type == B200_ACT_F32 ? 4 : 8) != 0 || ldq < k || ldq % 16 != 0)
    return sdb_fail(B200_ERR_SHAPE, "b200_quantize_act_int8: row strides must hold k and be multiples of 16 bytes");
  if (!aligned16(x) || !aligned16(x_lo) || !aligned16(q) || (reinterpret_cast<uintptr_t>(scale) & 3))
    return sdb_fail(B200_ERR_SHAPE, "b200_quantize_act_int8: x, x_lo and q must be 16-byte aligned");
  RowArgs a{};
  a.x = x;
  a.lo = x_lo;
  a.q = q;
  a.scale = scale;
  a.ldx = ldx;
  a.ldq = ldq;
  a.rows = rows;
  a.k = k;
  if (type == B200_ACT_F32) return launch_rows<false, B200_ACT_F32>(a, st);
  return x_lo ? launch_rows<false, ACT_PLANES>(a, st) : launch_rows<false, B200_ACT_BF16>(a, st);
}

int sdb_rmsnorm_int8(const float* x, int32_t ldx, const void* delta, int32_t delta_type, int32_t ldd, float* sum,
                     int32_t lds, int32_t rows, int32_t hidden, const float* w, float eps, int8_t* q, int32_t ldq,
                     float* scale, cudaStream_t st) {
  if (!x || !w || !q || !scale) return sdb_fail(B200_ERR_ARG, "b200_rmsnorm_int8: null pointer");
  if (sum && !delta) return sdb_fail(B200_ERR_ARG, "b200_rmsnorm_int8: sum needs a delta");
  if (delta && delta_type != B200_ACT_F32 && delta_type != B200_ACT_BF16)
    return sdb_fail(B200_ERR_ARG, "b200_rmsnorm_int8: unknown delta type");
  if (!(eps > 0.0f)) return sdb_fail(B200_ERR_ARG, "b200_rmsnorm_int8: eps must be positive");
  if (rows <= 0 || hidden <= 0) return sdb_fail(B200_ERR_SHAPE, "b200_rmsnorm_int8: empty shape");
  if (rows > I8_ROWS_MAX) return sdb_fail(B200_ERR_SHAPE, "b200_rmsnorm_int8: more than 2^30 rows");
  if (hidden % 16 != 0 || hidden > I8_K_MAX)
    return sdb_fail(B200_ERR_SHAPE, "b200_rmsnorm_int8: hidden must be a multiple of 16, at most 65536");
  if (ldx < hidden || ldx % 4 != 0 || ldq < hidden || ldq % 16 != 0 ||
      (delta && (ldd < hidden || ldd % (delta_type == B200_ACT_F32 ? 4 : 8) != 0)) ||
      (sum && (lds < hidden || lds % 4 != 0)))
    return sdb_fail(B200_ERR_SHAPE, "b200_rmsnorm_int8: row strides must hold hidden and be multiples of 16 bytes");
  if (!aligned16(x) || !aligned16(delta) || !aligned16(sum) || !aligned16(w) || !aligned16(q) ||
      (reinterpret_cast<uintptr_t>(scale) & 3))
    return sdb_fail(B200_ERR_SHAPE, "b200_rmsnorm_int8: x, delta, sum, w and q must be 16-byte aligned");
  RowArgs a{};
  a.x = x;
  a.delta = delta;
  a.sum = sum;
  a.w = w;
  a.q = q;
  a.scale = scale;
  a.ldx = ldx;
  a.ldd = ldd;
  a.lds = lds;
  a.ldq = ldq;
  a.rows = rows;
  a.k = hidden;
  a.eps = eps;
  if (!delta) return launch_rows<true, ACT_NONE>(a, st);
  return delta_type == B200_ACT_F32 ? launch_rows<true, B200_ACT_F32>(a, st) : launch_rows<true, B200_ACT_BF16>(a, st);
}

}  // namespace sdb

extern "C" int b200_quantize_act_int8(const void* x, const uint16_t* x_lo, int32_t type, int32_t rows, int32_t k,
                                      int32_t ldx, int8_t* q, int32_t ldq, float* scale, b200_stream stream) {
  return sdb::sdb_quantize_int8(x, x_lo, type, rows, k, ldx, q, ldq, scale, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int b200_rmsnorm_int8(const float* x, int32_t ldx, const void* delta, int32_t delta_type, int32_t ldd,
                                 float* sum, int32_t lds, int32_t rows, int32_t hidden, const float* w, float eps,
                                 int8_t* q, int32_t ldq, float* scale, b200_stream stream) {
  return sdb::sdb_rmsnorm_int8(x, ldx, delta, delta_type, ldd, sum, lds, rows, hidden, w, eps, q, ldq, scale,
                               reinterpret_cast<cudaStream_t>(stream));
}
