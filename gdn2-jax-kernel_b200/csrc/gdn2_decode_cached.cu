// Token-by-token decode from and into the int8 cache of states: the recurrence
// of gdn2_decode (one-token chunks, gdn2_fwd.py:264-362, every sanitiser where
// it stands there), with the state read as codes, held in float32 registers
// over the tokens of the call and stored as codes again.
//
// A step moves 2 x 17 KB a head at D = 128, against 2 x 64 KB for float32 states.
// Taking every code apart and putting it together again costs 16 instructions a
// value.  They are issued at 2.7 of 4 a cycle and no pipe is more than half busy:
// a CTA loads a head, works and stores, one after the other, and three neighbours
// do not fill its pauses (2048 CTAs are 3.5 waves).  One token for 256 rows
// x 8 heads of 128 takes 22.6 us, 48% of the copy rate (1024 rows: 86 us, 51%);
// one row 4.3 us, all of it latency.  Four tokens a call take 69 us, a
// quarter less than four calls (bytes ask for 13): a token after the first is two
// passes over the state and two synchronisations, at two CTAs an SM; 16 warps a CTA made that half as long again (more
// partial sums).
//
// One CTA per (row, head).  The head's codes and scales (17 KB, contiguous) come
// to shared memory by asynchronous copies, so the bytes in flight do not cost
// registers and four CTAs fit an SM (from registers, two: 35.5 us).  A thread
// works on 8 columns (one 8-byte word of codes) of R key rows; the D / 8 lanes of
// a row sit in one warp, so the maximum of a group of 64 columns takes three
// shuffles.  The two products with the state (W^T h and qg^T h) are summed over a
// thread's rows, over the row lanes of the warp, then over the warps in shared
// memory, always in the same order.  A call of one token takes the codes apart
// twice (for the products and for the update: 64 registers instead of 128); a
// call of more tokens keeps float32 values.
#include "../../include/gdn2.h"
#include "gdn2_int8.cuh"

namespace gdn2 {
int report_error(int code, const char* msg);

namespace {

template <int D> struct Shape {
  static constexpr int NW = D / 16;          // warps
  static constexpr int CL = D / 8;           // lanes of a row
  static constexpr int RW = 32 / CL;         // rows of a warp's load
  static constexpr int R = D / (NW * RW);    // rows of a thread
  static_assert(R % 4 == 0, "scales leave by fours");
  static constexpr int G = D / kGroup;
};

// 16 bytes to shared memory, asynchronously.
__device__ __forceinline__ void copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
               ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// The 8 codes of a row as float32 pairs: by byte moves and packed additions, or
// by the conversion unit, which is idle otherwise (an eighth of the rate, one
// instruction instead of one and a half).
__device__ __forceinline__ void codes8(uint2 c, float2 (&f)[4]) {
  const unsigned x = c.x ^ 0x80808080u, y = c.y ^ 0x80808080u;
  const float2 bias = both(-8388736.f);
  f[0] = add2(make_float2(biased_f<0>(x), biased_f<1>(x)), bias);
  f[1] = add2(make_float2(biased_f<2>(x), biased_f<3>(x)), bias);
  f[2] = add2(make_float2(biased_f<0>(y), biased_f<1>(y)), bias);
  f[3] = add2(make_float2(biased_f<2>(y), biased_f<3>(y)), bias);
}
__device__ __forceinline__ void convert8(uint2 c, float2 (&f)[4]) {
  auto at = [](unsigned x, int i) { return (float)(int8_t)(x >> 8 * i); };
  f[0] = make_float2(at(c.x, 0), at(c.x, 1));
  f[1] = make_float2(at(c.x, 2), at(c.x, 3));
  f[2] = make_float2(at(c.y, 0), at(c.y, 1));
  f[3] = make_float2(at(c.y, 2), at(c.y, 3));
}
__device__ __forceinline__ float top8(const float2 (&s)[4]) {
  return max_abs3(max_abs3(max_abs3(fabsf(s[0].x), s[0].y, s[1].x), s[1].y, s[2].x),
                  max_abs(s[2].y, s[3].x), s[3].y);
}

// h <- d h + kg vn on 8 columns.
__device__ __forceinline__ void update8(float2 (&x)[4], float d, float kg, const float2 (&vn)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = fma2(both(d), x[i], mul2(both(kg), vn[i]));
}

template <typename T, int D, bool ONE>
__global__ void __launch_bounds__(Shape<D>::NW * 32, D == 64 ? 6 : ONE ? 4 : 2)
k_decode_cached(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                const T* __restrict__ w, const T* __restrict__ b, const T* __restrict__ g,
                int8_t* codes, float* scales, const int* __restrict__ src,
                const int* __restrict__ dst, float* __restrict__ o, int B, int T_, int H, int S,
                float scale, float clip, int gates) {
  constexpr int NW = Shape<D>::NW, CL = Shape<D>::CL, RW = Shape<D>::RW, R = Shape<D>::R,
                G = Shape<D>::G;
  __shared__ __align__(16) int8_t scodes[D * D];
  __shared__ __align__(16) float sscales[D * G];
  // W, qg, kg, e^{gc_last} of a token.  Three tokens: the update of token t - 1 reads
  // its own, with no synchronisation of the CTA between it and the put of token t + 1.  (Two, put after
  // the first synchronisation: 69 to 71 us instead of 69 for the four tokens above.)
  __shared__ float4 vec[ONE ? 1 : 3][D];
  __shared__ float red[ONE ? 1 : 2][D / 32], su[ONE ? 1 : 2][D];
  __shared__ __align__(16) float2 part[NW][D];   // per warp: W^T h, qg^T h
  __shared__ __align__(16) float snew[D];
  const int h = blockIdx.x, bb = blockIdx.y, tid = threadIdx.x;
  const int lane = tid & 31, warp = tid >> 5, cl = lane % CL, rl = lane / CL;
  const float a1 = san(1.f, clip);   // A = (I + Akk)^-1 of a one-token chunk, sanitised

  const int from = src ? src[bb] : bb, to = dst ? dst[bb] : bb;
  const bool some = from >= 0 && from < S;
  if (some) {
    const size_t at = ((size_t)from * H + h) * D;
    const int8_t* c = codes + at * D;
    const float* z = scales + at * G;
#pragma unroll
    for (int i = 0; i < D * D / (NW * 32 * 16); ++i)
      copy16(scodes + (i * NW * 32 + tid) * 16, c + (i * NW * 32 + tid) * 16);
    if (tid < D * G / 4) copy16(sscales + tid * 4, z + tid * 4);
  } else {   // the zero state: scales of 0 beside codes of any value
    for (int i = tid; i < D * G; i += NW * 32) sscales[i] = 0.f;
  }

  // a token's vectors, by the first D threads: loaded, then put to shared memory
  float tq, tk, tv, tw, tb, tg;
  auto load = [&](size_t off) {
    tq = to_f<T>(q[off + tid]);
    tk = to_f<T>(k[off + tid]);
    tv = to_f<T>(v[off + tid]);
    tw = to_f<T>(w[off + tid]);
    tb = to_f<T>(b[off + tid]);
    tg = to_f<T>(g[off + tid]);
  };
  auto put = [&](int buf, int at) {   // at: of vec; buf: of red and su
    if (gates) {
      tw = gate_act(tw, kGateW);
      tb = gate_act(tb, kGateB);
      tg = gate_act(tg, kGateG);
    }
    const float eg = expf(tg);
    vec[at][tid] = make_float4(san(a1 * (tb * tk * eg), clip), san(tq * eg, clip), san(tk, clip),
                               expf(san(tg, clip)));
    su[buf][tid] = san(a1 * (tw * tv), clip);
    float qk = tq * tk;
#pragma unroll
    for (int x = 16; x; x >>= 1) qk += __shfl_xor_sync(0xffffffffu, qk, x);
    if (lane == 0) red[buf][warp] = qk;
  };
  size_t off = ((size_t)bb * T_ * H + h) * D;
  // a token is loaded a whole token before it is put, so that nothing waits for it
  if (tid < D) {
    load(off);
    put(0, 0);
    if (!ONE && T_ > 1) load(off + (size_t)H * D);
  }

  // A destination that is another row's source or destination would make the
  // result depend on which block runs first; such a row, and one whose slots
  // lie outside the cache, gets NaN outputs and no state is written for it.
  int bad = from < -1 || from >= S || to < -1 || to >= S;
  if (to >= 0)
    for (int j = tid; j < B; j += NW * 32)
      if (j != bb) {
        if (src) bad |= src[j] == to;
        if (dst != src) bad |= dst[j] == to;
      }
  copies_done();
  bad = __syncthreads_or(bad);
  if (bad) {
    for (int t = 0; t < T_; ++t, off += (size_t)H * D)
      if (tid < D) o[off + tid] = __uint_as_float(0x7fc00000u);
    return;
  }

  // row r of this thread, its scale (NaN as 0) and its codes
  auto row_of = [&](int r) { return (r * NW + warp) * RW + rl; };
  auto scale_of = [&](int row) { return fmaxf(sscales[row * G + cl * 8 / kGroup], 0.f); };
  auto word_of = [&](int row) { return *reinterpret_cast<const uint2*>(scodes + row * D + cl * 8); };

  float2 s[ONE ? 4 : R][4];
  if constexpr (!ONE) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float z = scale_of(row_of(r));
      codes8(word_of(row_of(r)), s[r]);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[r][i] = mul2(s[r][i], both(z));
    }
  }

  int at = 0;   // of token t in vec
  for (int t = 0; t < (ONE ? 1 : T_); ++t, off += (size_t)H * D) {
    const int buf = ONE ? 0 : t & 1, after = ONE || at == 2 ? 0 : at + 1;
    float2 wa[4] = {}, qa[4] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float4 z = vec[at][row_of(r)];
      if constexpr (ONE) {
        const float x = scale_of(row_of(r));
        convert8(word_of(row_of(r)), s[r & 3]);
        z.x *= x;
        z.y *= x;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        wa[i] = fma2(both(z.x), s[ONE ? r & 3 : r][i], wa[i]);
        qa[i] = fma2(both(z.y), s[ONE ? r & 3 : r][i], qa[i]);
      }
    }
#pragma unroll
    for (int x = CL; x < 32; x <<= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        wa[i].x += __shfl_xor_sync(0xffffffffu, wa[i].x, x);
        wa[i].y += __shfl_xor_sync(0xffffffffu, wa[i].y, x);
        qa[i].x += __shfl_xor_sync(0xffffffffu, qa[i].x, x);
        qa[i].y += __shfl_xor_sync(0xffffffffu, qa[i].y, x);
      }
    if (rl == 0)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4*>(&part[warp][cl * 8 + 2 * i]) =
            make_float4(wa[i].x, qa[i].x, wa[i].y, qa[i].y);
    if (!ONE && t + 1 < T_ && tid < D) {
      put(buf ^ 1, after);
      if (t + 2 < T_) load(off + 2 * (size_t)H * D);
    }
    __syncthreads();
    if (tid < D) {
      float dot = 0.f, wh = 0.f, qh = 0.f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) dot += red[buf][i];
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const float2 p = part[i][tid];
        wh += p.x;
        qh += p.y;
      }
      const float vn = su[buf][tid] - wh;
      snew[tid] = vn;
      o[off + tid] = san(scale * qh + san(scale * dot, clip) * vn, clip);
    }
    __syncthreads();
    if constexpr (!ONE) {
      float2 vn[4];
      *reinterpret_cast<float4*>(vn) = *reinterpret_cast<const float4*>(snew + cl * 8);
      *reinterpret_cast<float4*>(vn + 2) = *reinterpret_cast<const float4*>(snew + cl * 8 + 4);
      float top = 0.f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 z = vec[at][row_of(r)];
        update8(s[r], z.w, z.z, vn);
        top = max_abs(top, top8(s[r]));
      }
      if (!(top <= clip))   // seldom: the sanitiser acts
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[r][i] = make_float2(san(s[r][i].x, clip), san(s[r][i].y, clip));
    }
    at = after;
  }

  if (to < 0) return;
  float2 vn[4];
  *reinterpret_cast<float4*>(vn) = *reinterpret_cast<const float4*>(snew + cl * 8);
  *reinterpret_cast<float4*>(vn + 2) = *reinterpret_cast<const float4*>(snew + cl * 8 + 4);
  const size_t row0 = ((size_t)to * H + h) * D;
  // Four rows at a time: the maxima of the four are passed around the 8 lanes of a
  // group so that each lane ends with one row's, works out that row's scale, and
  // hands 127 / max back.
  const int own = cl & 3;
#pragma unroll
  for (int r0 = 0; r0 < R; r0 += 4) {
    float2 (&x)[4][4] = *reinterpret_cast<float2 (*)[4][4]>(&s[ONE ? 0 : r0]);
    float top[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (ONE) {
        const int row = row_of(r0 + j);
        const float4 z = vec[0][row];
        if (j & 1) convert8(word_of(row), x[j]);   // both ways: on different pipes
        else codes8(word_of(row), x[j]);
        update8(x[j], z.w * scale_of(row), z.z, vn);
      }
      top[j] = top8(x[j]);
    }
    auto around = [&] {
      const bool hi = own & 2, odd = own & 1;
      float t0 = hi ? top[2] : top[0], t1 = hi ? top[3] : top[1];
      const float u0 = hi ? top[0] : top[2], u1 = hi ? top[1] : top[3];
      t0 = max_abs(t0, __shfl_xor_sync(0xffffffffu, u0, 2));
      t1 = max_abs(t1, __shfl_xor_sync(0xffffffffu, u1, 2));
      float m = odd ? t1 : t0;
      m = max_abs(m, __shfl_xor_sync(0xffffffffu, odd ? t0 : t1, 1));
      return max_abs(m, __shfl_xor_sync(0xffffffffu, m, 4));
    };
    float m = around();   // of row r0 + own
    if (ONE && __any_sync(0xffffffffu, !(m <= clip))) {   // seldom: the sanitiser acts
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[j][i] = make_float2(san(x[j][i].x, clip), san(x[j][i].y, clip));
        top[j] = top8(x[j]);
      }
      m = around();
    }
    // (the scale need not be the correctly rounded quotient that packed tensors
    // promise, and its division was 3% of the instructions; m is infinite only
    // under a clip that is)
    if (cl % 8 < 4)
      scales[(row0 + row_of(r0 + own)) * G + cl * 8 / kGroup] =
          m > 3.402823466e38f ? __uint_as_float(0x7fc00000u)
          : m >= kInt8Tiny ? m * (1.f / 127.f) : 0.f;
    const float inv = group_inv(m);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // the nearest code by float32 arithmetic alone: the value carries rounding
      // errors of its own, 2.2e-5 of a step more do not matter
      const float y = __shfl_sync(0xffffffffu, inv, (lane & ~3) | j);
      float2 n[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) n[i] = fma2(x[j][i], both(y), both(kCodeBias));
      auto u = [](float f) { return __float_as_uint(f); };
      *reinterpret_cast<uint2*>(codes + (row0 + row_of(r0 + j)) * D + cl * 8) =
          make_uint2(pack4(u(n[0].x), u(n[0].y), u(n[1].x), u(n[1].y)),
                     pack4(u(n[2].x), u(n[2].y), u(n[3].x), u(n[3].y)));
    }
  }
}

template <typename T, int D>
void launch(const void* q, const void* k, const void* v, const void* w, const void* b,
            const void* g, void* codes, float* scales, const int* src, const int* dst, float* o,
            int B, int T_, int H, int S, float scale, float clip, int gates, cudaStream_t s) {
  auto c = [](const void* x) { return static_cast<const T*>(x); };
  auto go = [&](auto kernel) {
    kernel<<<dim3(H, B), Shape<D>::NW * 32, 0, s>>>(c(q), c(k), c(v), c(w), c(b), c(g),
                                                    static_cast<int8_t*>(codes), scales, src, dst,
                                                    o, B, T_, H, S, scale, clip, gates);
  };
  T_ == 1 ? go(k_decode_cached<T, D, true>) : go(k_decode_cached<T, D, false>);
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
  if ((reinterpret_cast<uintptr_t>(codes) & 15) || (reinterpret_cast<uintptr_t>(scales) & 15))
    return report_error(GDN2_ERR_INVALID, "gdn2_decode_cached: codes and scales must be 16-byte aligned");
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
