// Token-by-token decode from and into the int8 cache of states: the recurrence
// of gdn2_decode (one-token chunks, gdn2_fwd.py:264-362, every sanitiser where
// it stands there), with the state read as codes, held in float32 registers
// over the tokens of the call and stored as codes again.
//
// A step is bound by the state's bytes: 2 x 17 KB a head at D = 128, against
// 2 x 64 KB for float32 states.
//
// One CTA per (row, head).  A thread holds 8 columns (one 8-byte load of codes)
// of R key rows; the D / 8 lanes of a row sit in one warp, so the maximum of a
// group of 64 columns takes three shuffles.  The two products with the state
// (W^T h and qg^T h) are summed over a thread's rows, over the row lanes of the
// warp, then over the warps in shared memory, always in the same order.
#include "../../include/gdn2.h"
#include "gdn2_int8.cuh"

namespace gdn2 {
int report_error(int code, const char* msg);

namespace {

template <typename T, int D>
__global__ void __launch_bounds__(256)
k_decode_cached(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                const T* __restrict__ w, const T* __restrict__ b, const T* __restrict__ g,
                int8_t* codes, float* scales, const int* __restrict__ src,
                const int* __restrict__ dst, float* __restrict__ o, int B, int T_, int H, int S,
                float scale, float clip, int gates) {
  constexpr int NW = 8, CL = D / 8, RW = 32 / CL, R = D / (NW * RW), G = D / kGroup;
  __shared__ float4 vec[D];            // W, qg, kg, e^{gc_last} of a token
  __shared__ float2 part[NW][D];       // per warp: W^T h, qg^T h
  __shared__ float red[D / 32], su[D], snew[D];
  const int h = blockIdx.x, bb = blockIdx.y, tid = threadIdx.x;
  const int lane = tid & 31, warp = tid >> 5, cl = lane % CL, rl = lane / CL;

  // A destination that is another row's source or destination would make the
  // result depend on which block runs first; such a row, and one whose slots
  // lie outside the cache, gets NaN outputs and no state is written for it.
  const int from = src ? src[bb] : bb, to = dst ? dst[bb] : bb;
  int bad = from < -1 || from >= S || to < -1 || to >= S;
  if (to >= 0)
    for (int j = tid; j < B; j += 256)
      if (j != bb) {
        if (src) bad |= src[j] == to;
        if (dst != src) bad |= dst[j] == to;
      }
  bad = __syncthreads_or(bad);
  if (bad) {
    for (int t = 0; t < T_; ++t)
      if (tid < D) o[(((size_t)bb * T_ + t) * H + h) * D + tid] = __uint_as_float(0x7fc00000u);
    return;
  }

  float s[R][8];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = (r * NW + warp) * RW + rl;
    uint2 c = make_uint2(0, 0);
    float sc = 0.f;
    if (from >= 0) {
      const size_t at = (((size_t)from * H + h) * D + row);
      c = *reinterpret_cast<const uint2*>(codes + at * D + cl * 8);
      sc = scales[at * G + cl * 8 / kGroup];
    }
    if (!(fabsf(sc) <= 3.4e38f)) sc = 0.f;   // the sanitiser's NaN -> 0
    const unsigned lo = c.x ^ 0x80808080u, hi = c.y ^ 0x80808080u;
    s[r][0] = code_f<0>(lo) * sc; s[r][1] = code_f<1>(lo) * sc;
    s[r][2] = code_f<2>(lo) * sc; s[r][3] = code_f<3>(lo) * sc;
    s[r][4] = code_f<0>(hi) * sc; s[r][5] = code_f<1>(hi) * sc;
    s[r][6] = code_f<2>(hi) * sc; s[r][7] = code_f<3>(hi) * sc;
#pragma unroll
    for (int i = 0; i < 8; ++i) s[r][i] = san(s[r][i], clip);
  }

  const float a1 = san(1.f, clip);   // A = (I + Akk)^-1 of a one-token chunk, sanitised
  for (int t = 0; t < T_; ++t) {
    const size_t off = (((size_t)bb * T_ + t) * H + h) * D;
    if (tid < D) {
      const float qv = to_f<T>(q[off + tid]), kv = to_f<T>(k[off + tid]);
      const float gv = ld_gate<T>(g + off + tid, gates, kGateG), eg = expf(gv);
      vec[tid] = make_float4(
          san(a1 * (ld_gate<T>(b + off + tid, gates, kGateB) * kv * eg), clip),
          san(qv * eg, clip), san(kv, clip), expf(san(gv, clip)));
      su[tid] = san(a1 * (ld_gate<T>(w + off + tid, gates, kGateW) * to_f<T>(v[off + tid])), clip);
      float qk = qv * kv;
#pragma unroll
      for (int x = 16; x; x >>= 1) qk += __shfl_xor_sync(0xffffffffu, qk, x);
      if (lane == 0) red[warp] = qk;
    }
    __syncthreads();
    float a[8] = {}, c[8] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float4 z = vec[(r * NW + warp) * RW + rl];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] = fmaf(z.x, s[r][i], a[i]);
        c[i] = fmaf(z.y, s[r][i], c[i]);
      }
    }
#pragma unroll
    for (int x = CL; x < 32; x <<= 1)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] += __shfl_xor_sync(0xffffffffu, a[i], x);
        c[i] += __shfl_xor_sync(0xffffffffu, c[i], x);
      }
    if (rl == 0)
#pragma unroll
      for (int i = 0; i < 8; ++i) part[warp][cl * 8 + i] = make_float2(a[i], c[i]);
    __syncthreads();
    if (tid < D) {
      float dot = 0.f, wh = 0.f, qh = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) dot += red[i];
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const float2 p = part[i][tid];
        wh += p.x;
        qh += p.y;
      }
      const float vn = su[tid] - wh;
      snew[tid] = vn;
      o[off + tid] = san(scale * qh + san(scale * dot, clip) * vn, clip);
    }
    __syncthreads();
    float vn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) vn[i] = snew[cl * 8 + i];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float4 z = vec[(r * NW + warp) * RW + rl];
#pragma unroll
      for (int i = 0; i < 8; ++i) s[r][i] = san(fmaf(z.w, s[r][i], z.z * vn[i]), clip);
    }
    __syncthreads();   // the token vectors are rewritten
  }

  if (to < 0) return;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float top = fabsf(s[r][0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) top = max_abs(top, s[r][i]);
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) top = max_abs(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float inv = group_inv(top);
    uint2 c;
    auto code = [&](int i) { return int8_code_near(s[r][i], inv); };
    c.x = pack4(code(0), code(1), code(2), code(3));
    c.y = pack4(code(4), code(5), code(6), code(7));
    const size_t at = (((size_t)to * H + h) * D + (r * NW + warp) * RW + rl);
    *reinterpret_cast<uint2*>(codes + at * D + cl * 8) = c;
    if (cl % 8 == 0) scales[at * G + cl * 8 / kGroup] = group_scale(top);
  }
}

template <typename T, int D>
void launch(const void* q, const void* k, const void* v, const void* w, const void* b,
            const void* g, void* codes, float* scales, const int* src, const int* dst, float* o,
            int B, int T_, int H, int S, float scale, float clip, int gates, cudaStream_t s) {
  auto c = [](const void* x) { return static_cast<const T*>(x); };
  k_decode_cached<T, D><<<dim3(H, B), 256, 0, s>>>(c(q), c(k), c(v), c(w), c(b), c(g),
                                                   static_cast<int8_t*>(codes), scales, src, dst,
                                                   o, B, T_, H, S, scale, clip, gates);
}

}  // namespace
}  // namespace gdn2

extern "C" int gdn2_decode_cached(int dtype, const void* q, const void* k, const void* v,
                                  const void* w, const void* b, const void* g, void* codes,
                                  float* scales, const int* src, const int* dst, float* o, int B,
                                  int T, int H, int D, int S, float scale, float clip,
                                  void* stream) {
  using namespace gdn2;
  const int gates = (dtype & GDN2_GATES_RAW) != 0;
  dtype &= ~GDN2_GATES_RAW;
  if (dtype != GDN2_F32 && dtype != GDN2_BF16)
    return report_error(GDN2_ERR_INVALID, "gdn2_decode_cached: unsupported dtype code");
  if (B <= 0 || T <= 0 || H <= 0 || S <= 0)
    return report_error(GDN2_ERR_INVALID, "gdn2_decode_cached: empty problem (B, T, H, S)");
  if (B > 65535) return report_error(GDN2_ERR_INVALID, "gdn2_decode_cached: at most 65535 rows per call");
  if (D != 64 && D != 128)
    return report_error(GDN2_ERR_INVALID, "gdn2_decode_cached: head dim D unsupported (64 or 128)");
  if (!(clip > 0.f) || scale != scale)
    return report_error(GDN2_ERR_INVALID, "gdn2_decode_cached: clip must be positive, scale finite");
  if (!q || !k || !v || !w || !b || !g || !o || !codes || !scales)
    return report_error(GDN2_ERR_INVALID, "gdn2_decode_cached: null buffer pointer");
  if ((reinterpret_cast<uintptr_t>(codes) & 15) || (reinterpret_cast<uintptr_t>(scales) & 3))
    return report_error(GDN2_ERR_INVALID, "gdn2_decode_cached: codes must be 16-byte aligned");
  if ((!src || !dst) && B > S)
    return report_error(GDN2_ERR_INVALID, "gdn2_decode_cached: more rows than slots");
  if (!src != !dst)
    return report_error(GDN2_ERR_INVALID, "gdn2_decode_cached: give both slot lists or neither");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == GDN2_F32) {
    if (D == 128)
      launch<float, 128>(q, k, v, w, b, g, codes, scales, src, dst, o, B, T, H, S, scale, clip, gates, s);
    else
      launch<float, 64>(q, k, v, w, b, g, codes, scales, src, dst, o, B, T, H, S, scale, clip, gates, s);
  } else {
    if (D == 128)
      launch<__nv_bfloat16, 128>(q, k, v, w, b, g, codes, scales, src, dst, o, B, T, H, S, scale, clip, gates, s);
    else
      launch<__nv_bfloat16, 64>(q, k, v, w, b, g, codes, scales, src, dst, o, B, T, H, S, scale, clip, gates, s);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GDN2_OK : report_error(GDN2_ERR_CUDA, cudaGetErrorString(e));
}
