// W8A8 linears: y[t, n] = (sum_k q[t, k] w[n, k]) * scale[t] * row_scale[n], int32 sums.
#include <algorithm>

#include "common.cuh"

namespace sdb {

struct I8Args {
  const int8_t* q;      // [m, ldx]
  const float* xs;      // [m]
  const int8_t* w;      // [n, k]
  const float* ws;      // [n]
  b200_linear_out o;
  int m, n, k, ldx;
};

// The SwiGLU's output at token t, feature f: silu(g) * u as the bf16 hi plane and, if asked, the
// low plane.
__device__ __forceinline__ void store_swiglu(const b200_linear_out& o, int t, int f, float g, float u) {
  const float h = silu_approx(g) * u;
  const uint16_t hb = f32_to_bf16_rn(h);
  uint16_t* dst = static_cast<uint16_t*>(o.out);
  const size_t idx = size_t(t) * o.ldo + f;
  dst[idx] = hb;
  if (!o.lo_offset) return;
  if (o.lo_format == B200_LO_E4M3)
    reinterpret_cast<uint8_t*>(dst + o.lo_offset)[idx] = uint8_t(f32x2_to_e4m3x2(lo8_value(h, hb), 0.0f));
  else
    dst[o.lo_offset + idx] = f32_to_bf16_rn(h - bf16_to_f32(hb));
}

// One thread per output: 4 products per dp4a, straight from global memory.
__device__ __forceinline__ float dot_int8(const I8Args& a, int t, int n) {
  const int4* x = reinterpret_cast<const int4*>(a.q + size_t(t) * a.ldx);
  const int4* w = reinterpret_cast<const int4*>(a.w + size_t(n) * a.k);
  int acc = 0;
  for (int i = 0; i < a.k / 16; ++i) {
    const int4 p = x[i], r = __ldg(w + i);
    acc = __dp4a(p.x, r.x, acc);
    acc = __dp4a(p.y, r.y, acc);
    acc = __dp4a(p.z, r.z, acc);
    acc = __dp4a(p.w, r.w, acc);
  }
  return float(acc) * a.xs[t] * a.ws[n];
}

template <int EP>
__global__ void gemm_int8_kernel(const I8Args a) {
  pdl_wait();
  pdl_trigger();
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  for (int t = blockIdx.y; t < a.m; t += gridDim.y) {
    if constexpr (EP == B200_EP_SWIGLU) {
      if (2 * j >= a.o.n_valid) return;
      const int row = j / 64 * 128 + j % 64;
      store_swiglu(a.o, t, j, dot_int8(a, t, row), dot_int8(a, t, row + 64));
    } else {
      if (j >= a.o.n_valid) return;
      float* p = static_cast<float*>(a.o.out) + size_t(t) * a.o.ldo + j;
      const float y = dot_int8(a, t, j);
      if constexpr (EP == B200_EP_RESID_ADD) *p += y;
      else *p = y;
    }
  }
}

template <int EP>
static int launch_int8(const I8Args& a, cudaStream_t st) {
  const int cols = EP == B200_EP_SWIGLU ? a.o.n_valid / 2 : a.o.n_valid;
  SDB_CUDA(launch_pdl(gemm_int8_kernel<EP>, dim3((cols + 127) / 128, std::min(a.m, 65535)), dim3(128), 0, st, a));
  return B200_OK;
}

int sdb_linear_int8(const int8_t* q, const float* x_scale, int32_t m, int32_t k, int32_t ldx, const b200_qweight* w,
                    const b200_linear_out* out, cudaStream_t st) {
  if (!q || !x_scale || !w || !out || !w->data || !out->out)
    return sdb_fail(B200_ERR_ARG, "b200_linear_int8: null pointer");
  if (w->format != B200_W_INT8) return sdb_fail(B200_ERR_FORMAT, "b200_linear_int8: needs a B200_W_INT8 weight");
  if (!w->row_scale) return sdb_fail(B200_ERR_ARG, "b200_linear_int8: missing row_scale");
  if (m <= 0 || k <= 0 || w->n <= 0) return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: empty shape");
  if (w->k != k) return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: q and W disagree on k");
  if (k % 16 != 0 || k > 65536)
    return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: k must be a multiple of 16, at most 65536");
  if (ldx < k || ldx % 16 != 0 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(w->data)) & 15))
    return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: q and W must be 16-byte aligned with ldx a multiple of 16");
  if (out->epilogue < 0 || out->epilogue > 2) return sdb_fail(B200_ERR_ARG, "b200_linear_int8: unknown epilogue");
  if (out->n_valid <= 0 || out->n_valid > w->n)
    return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: n_valid must be in (0, n]");
  const bool swiglu = out->epilogue == B200_EP_SWIGLU;
  if (swiglu && out->n_valid % 128 != 0)
    return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: SwiGLU needs n_valid % 128 == 0");
  if (out->ldo < (swiglu ? out->n_valid / 2 : out->n_valid))
    return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: ldo does not hold a row");
  if (reinterpret_cast<uintptr_t>(out->out) & (swiglu ? 1 : 3))
    return sdb_fail(B200_ERR_SHAPE, "b200_linear_int8: out is not aligned to its elements");
  if (out->lo_format != B200_LO_BF16 && out->lo_format != B200_LO_E4M3)
    return sdb_fail(B200_ERR_ARG, "b200_linear_int8: unknown lo_format");
  I8Args a{q, x_scale, static_cast<const int8_t*>(w->data), w->row_scale, *out, m, w->n, k, ldx};
  switch (out->epilogue) {
    case B200_EP_STORE: return launch_int8<B200_EP_STORE>(a, st);
    case B200_EP_RESID_ADD: return launch_int8<B200_EP_RESID_ADD>(a, st);
    default: return launch_int8<B200_EP_SWIGLU>(a, st);
  }
}

}  // namespace sdb

extern "C" int b200_linear_int8(const int8_t* q, const float* x_scale, int32_t m, int32_t k, int32_t ldx,
                                const b200_qweight* w, const b200_linear_out* out, b200_stream stream) {
  return sdb::sdb_linear_int8(q, x_scale, m, k, ldx, w, out, reinterpret_cast<cudaStream_t>(stream));
}
