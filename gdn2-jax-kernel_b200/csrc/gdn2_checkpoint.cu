// int8 activation checkpoints (pack / unpack of whole tensors) and the int8
// cache of recurrent states (write / read by slot): the group form of
// gdn2_int8.cuh applied as values are stored and taken off as they are read.
//
// Every kernel moves each byte once and is bound by HBM: float32 values take
// 4 + 1.0625 bytes either way.  A thread holds four pieces of 16 bytes of values
// (4 float32 or 8 bf16), so a group of 64 is 16 or 8 neighbouring lanes, whose
// maximum takes 4 or 3 shuffles, and the codes of a warp leave as one contiguous
// store.  Five tensors of 50.3M values, of the measured copy rate: float32 packed
// in 192 us (101%) and restored in 193 us (101%), bf16 in 136 us (86%) and 119 us
// (99%).  States of 256 x 8 heads of 128 are written in 28.7 us (90%: the slots
// are looked through first) and read in 25.3 us (102%).
#include "../../include/gdn2.h"
#include "gdn2_int8.cuh"

namespace gdn2 {
int report_error(int code, const char* msg);

namespace {

constexpr int kMaxTensors = GDN2_INT8_MAX_TENSORS;
struct Tensors {
  const void* x[kMaxTensors];   // values (pack: source, unpack: destination)
  int8_t* codes;                // of all, one tensor after another
  float* scales;
};

// E values of one thread, 16 bytes of T.
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ void load(float (&x)[4], const float* p) {
    const float4 v = __ldcs(reinterpret_cast<const float4*>(p));
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&x)[4]) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int E = 8;
  static __device__ __forceinline__ void load(float (&x)[8], const __nv_bfloat16* p) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
    const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&x)[8]) {
    unsigned u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      u[i] = *reinterpret_cast<const unsigned*>(&h);
    }
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(u[0], u[1], u[2], u[3]));
  }
};

constexpr int kUnroll = 4;   // 16-byte pieces a thread holds at once

// Codes of the kUnroll pieces of a thread, one word per 4 values, and as the value
// the scale of piece (lane & 3): a group's lanes share its division (every lane
// dividing for every piece cost a third of the instructions).  Whole warps call.
// clip > 0: through the sanitiser, looked at only where a maximum asks for it.
template <typename T>
__device__ __forceinline__ float encode(float (&x)[kUnroll][Vec<T>::E],
                                        unsigned (&word)[kUnroll][Vec<T>::E / 4], float clip = 0.f) {
  constexpr int E = Vec<T>::E;
  float mine = 0.f;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    auto largest = [&] {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < E; i += 2) t = max_abs3(t, x[u][i], x[u][i + 1]);
#pragma unroll
      for (int o = 1; o < kGroup / E; o <<= 1) t = max_abs(t, __shfl_xor_sync(0xffffffffu, t, o));
      return t;
    };
    float top = largest();
    if (clip > 0.f && __any_sync(0xffffffffu, !(top <= clip))) {
#pragma unroll
      for (int i = 0; i < E; ++i) x[u][i] = san(x[u][i], clip);
      top = largest();
    }
    unsigned c[E];
    int8_codes<T, E>(x[u], top, c);
#pragma unroll
    for (int i = 0; i < E; i += 4) word[u][i / 4] = pack4(c[i], c[i + 1], c[i + 2], c[i + 3]);
    if ((threadIdx.x & 3) == u) mine = top;
  }
  return group_scale(mine);
}
template <int E>
__device__ __forceinline__ void decode(float (&x)[E], const unsigned (&word)[E / 4], float scale) {
#pragma unroll
  for (int i = 0; i < E; i += 4) {
    const unsigned b = word[i / 4] ^ 0x80808080u;
    x[i] = code_f<0>(b) * scale;
    x[i + 1] = code_f<1>(b) * scale;
    x[i + 2] = code_f<2>(b) * scale;
    x[i + 3] = code_f<3>(b) * scale;
  }
}
template <int E>
__device__ __forceinline__ void ld_words(unsigned (&w)[E / 4], const int8_t* p) {
  if constexpr (E == 4) w[0] = *reinterpret_cast<const unsigned*>(p);
  else { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
}
template <int E>
__device__ __forceinline__ void st_words(int8_t* p, const unsigned (&w)[E / 4]) {
  if constexpr (E == 4) *reinterpret_cast<unsigned*>(p) = w[0];
  else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}

// Lane u of a group (u < kUnroll) stores the scale of the group's piece u: value
// index of that piece for this lane, or no index.
template <int E>
__device__ __forceinline__ bool scale_place(size_t base, size_t n, size_t& group) {
  const int lane = threadIdx.x % (kGroup / E);
  const size_t i = base + (size_t)lane * 256 * E;
  group = i / kGroup;
  return lane < kUnroll && i < n;
}

// (The argument stays in constant memory: picked from by blockIdx.y it would be
// copied to the stack, 273 us instead of 192.)
// blockIdx.y: tensor; n: values of each (a multiple of 64).  The bounds are
// per thread, but a group's lanes are in or out of them together.
template <typename T>
__global__ void __launch_bounds__(256) k_pack(const __grid_constant__ Tensors a, size_t n) {
  constexpr int E = Vec<T>::E;
  const T* x = static_cast<const T*>(a.x[blockIdx.y]);
  int8_t* c = a.codes + blockIdx.y * n;
  float* s = a.scales + blockIdx.y * (n / kGroup);
  const size_t base = (size_t)blockIdx.x * (256 * E * kUnroll) + threadIdx.x * E;
  float v[kUnroll][E] = {};
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const size_t i = base + (size_t)u * 256 * E;
    if (i < n) Vec<T>::load(v[u], x + i);
  }
  unsigned w[kUnroll][E / 4];
  const float scale = encode<T>(v, w);
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const size_t i = base + (size_t)u * 256 * E;
    if (i < n) st_words<E>(c + i, w[u]);
  }
  size_t group;
  if (scale_place<E>(base, n, group)) s[group] = scale;
}

template <typename T>
__global__ void __launch_bounds__(256) k_unpack(const __grid_constant__ Tensors a, size_t n) {
  constexpr int E = Vec<T>::E;
  T* x = static_cast<T*>(const_cast<void*>(a.x[blockIdx.y]));
  const int8_t* c = a.codes + blockIdx.y * n;
  const float* s = a.scales + blockIdx.y * (n / kGroup);
  const size_t base = (size_t)blockIdx.x * (256 * E * kUnroll) + threadIdx.x * E;
  unsigned w[kUnroll][E / 4] = {};
  float scale[kUnroll] = {};
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const size_t i = base + (size_t)u * 256 * E;
    if (i < n) {
      ld_words<E>(w[u], c + i);
      scale[u] = s[i / kGroup];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const size_t i = base + (size_t)u * 256 * E;
    float v[E];
    decode<E>(v, w[u], scale[u]);
    if (i < n) Vec<T>::store(x + i, v);
  }
}

// State cache, blockIdx.y: batch row b; n = H * D * D values of a row.
// Where several rows name one slot the last of them is written, whatever the
// order in which blocks run.
__global__ void __launch_bounds__(256)
k_state_write(const float* __restrict__ h, int8_t* __restrict__ codes, float* __restrict__ scales,
              const int* __restrict__ slots, int S, size_t n, float clip) {
  constexpr int E = 4;
  const int b = blockIdx.y, B = gridDim.y;
  const size_t base = (size_t)blockIdx.x * (256 * E * kUnroll) + threadIdx.x * E;
  const float* x = h + (size_t)b * n;
  float v[kUnroll][E] = {};
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const size_t i = base + (size_t)u * 256 * E;
    if (i < n) Vec<float>::load(v[u], x + i);
  }
  const int slot = slots ? slots[b] : b;
  int later = 0;
  if (slots)
    for (int j = b + 1 + threadIdx.x; j < B; j += 256) later |= slots[j] == slot;
  if (__syncthreads_or(later) || slot < 0 || slot >= S) return;
  int8_t* c = codes + (size_t)slot * n;
  float* s = scales + (size_t)slot * (n / kGroup);
  unsigned w[kUnroll][1];
  const float scale = encode<float>(v, w, clip);
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const size_t i = base + (size_t)u * 256 * E;
    if (i < n) st_words<E>(c + i, w[u]);
  }
  size_t group;
  if (scale_place<E>(base, n, group)) s[group] = scale;
}

// A slot of -1 reads as the zero state; one outside the cache as NaN.
template <typename T>
__global__ void __launch_bounds__(256)
k_state_read(const int8_t* __restrict__ codes, const float* __restrict__ scales,
             const int* __restrict__ slots, T* __restrict__ out, int S, size_t n) {
  constexpr int E = Vec<T>::E;
  const int b = blockIdx.y;
  const int slot = slots ? slots[b] : b;
  const bool in = slot >= 0 && slot < S;
  const int8_t* c = codes + (size_t)(in ? slot : 0) * n;
  const float* s = scales + (size_t)(in ? slot : 0) * (n / kGroup);
  const float none = slot == -1 ? 0.f : __uint_as_float(0x7fc00000u);
  const size_t base = (size_t)blockIdx.x * (256 * E * kUnroll) + threadIdx.x * E;
  unsigned w[kUnroll][E / 4] = {};
  float scale[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const size_t i = base + (size_t)u * 256 * E;
    scale[u] = none;
    if (i < n && in) {
      ld_words<E>(w[u], c + i);
      scale[u] = s[i / kGroup];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const size_t i = base + (size_t)u * 256 * E;
    float v[E];
    decode<E>(v, w[u], scale[u]);
    if (i < n) Vec<T>::store(out + (size_t)b * n + i, v);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

unsigned blocks_for(size_t n, int elem_bytes) {
  const size_t per = (size_t)256 * (16 / elem_bytes) * kUnroll;
  return (unsigned)((n + per - 1) / per);
}

// The checks that pack and unpack share; fills `a`.
int check_tensors(int dtype, int n_tensors, const void* const* values, const void* codes,
                  const float* scales, size_t n, Tensors& a) {
  if (dtype != GDN2_F32 && dtype != GDN2_BF16)
    return report_error(GDN2_ERR_INVALID, "gdn2_int8: unsupported dtype code");
  if (n_tensors < 1 || n_tensors > kMaxTensors)
    return report_error(GDN2_ERR_INVALID, "gdn2_int8: between 1 and GDN2_INT8_MAX_TENSORS tensors");
  if (n == 0 || n % kGroup || n > ((size_t)1 << 40))
    return report_error(GDN2_ERR_INVALID, "gdn2_int8: a positive multiple of 64 values per tensor");
  if (!values || !codes || !scales)
    return report_error(GDN2_ERR_INVALID, "gdn2_int8: null buffer pointer");
  if (!aligned16(codes) || ((uintptr_t)scales & 3))
    return report_error(GDN2_ERR_INVALID, "gdn2_int8: values and codes must be 16-byte aligned");
  for (int i = 0; i < n_tensors; ++i) {
    if (!values[i]) return report_error(GDN2_ERR_INVALID, "gdn2_int8: null buffer pointer");
    if (!aligned16(values[i]))
      return report_error(GDN2_ERR_INVALID, "gdn2_int8: values and codes must be 16-byte aligned");
    a.x[i] = values[i];
  }
  a.codes = static_cast<int8_t*>(const_cast<void*>(codes));
  a.scales = const_cast<float*>(scales);
  return GDN2_OK;
}

int check_state(const void* h, const void* codes, const void* scales, int B, int S, int H, int D) {
  if (B <= 0 || S <= 0 || H <= 0)
    return report_error(GDN2_ERR_INVALID, "gdn2_state: empty problem (B, S, H)");
  if (B > 65535) return report_error(GDN2_ERR_INVALID, "gdn2_state: at most 65535 rows per call");
  if (D != 64 && D != 128 && D != 256)
    return report_error(GDN2_ERR_INVALID, "gdn2_state: head dim D unsupported (64, 128 or 256)");
  if (!h || !codes || !scales)
    return report_error(GDN2_ERR_INVALID, "gdn2_state: null buffer pointer");
  if (!aligned16(h) || !aligned16(codes) || ((uintptr_t)scales & 3))
    return report_error(GDN2_ERR_INVALID, "gdn2_state: states and codes must be 16-byte aligned");
  return GDN2_OK;
}

int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GDN2_OK : report_error(GDN2_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" int gdn2_int8_pack(int dtype, int n_tensors, const void* const* values, void* codes,
                              float* scales, size_t n, void* stream) {
  Tensors a{};
  const int rc = check_tensors(dtype, n_tensors, values, codes, scales, n, a);
  if (rc) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == GDN2_F32)
    k_pack<float><<<dim3(blocks_for(n, 4), n_tensors), 256, 0, s>>>(a, n);
  else
    k_pack<__nv_bfloat16><<<dim3(blocks_for(n, 2), n_tensors), 256, 0, s>>>(a, n);
  return launched();
}

extern "C" int gdn2_int8_unpack(int dtype, int n_tensors, void* const* values, const void* codes,
                                const float* scales, size_t n, void* stream) {
  Tensors a{};
  const int rc = check_tensors(dtype, n_tensors, values, codes, scales, n, a);
  if (rc) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == GDN2_F32)
    k_unpack<float><<<dim3(blocks_for(n, 4), n_tensors), 256, 0, s>>>(a, n);
  else
    k_unpack<__nv_bfloat16><<<dim3(blocks_for(n, 2), n_tensors), 256, 0, s>>>(a, n);
  return launched();
}

extern "C" int gdn2_state_write(const float* h, const int* slots, void* codes, float* scales, int B,
                                int S, int H, int D, float clip, void* stream) {
  const int rc = check_state(h, codes, scales, B, S, H, D);
  if (rc) return rc;
  if (!(clip > 0.f)) return report_error(GDN2_ERR_INVALID, "gdn2_state: clip must be positive");
  if (!slots && B > S) return report_error(GDN2_ERR_INVALID, "gdn2_state: more rows than slots");
  const size_t n = (size_t)H * D * D;
  k_state_write<<<dim3(blocks_for(n, 4), B), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      h, static_cast<int8_t*>(codes), scales, slots, S, n, clip);
  return launched();
}

extern "C" int gdn2_state_read(int dtype, const void* codes, const float* scales, const int* slots,
                               void* h, int B, int S, int H, int D, void* stream) {
  const int rc = check_state(h, codes, scales, B, S, H, D);
  if (rc) return rc;
  if (dtype != GDN2_F32 && dtype != GDN2_BF16)
    return report_error(GDN2_ERR_INVALID, "gdn2_state: unsupported dtype code");
  if (!slots && B > S) return report_error(GDN2_ERR_INVALID, "gdn2_state: more rows than slots");
  const size_t n = (size_t)H * D * D;
  const int8_t* c = static_cast<const int8_t*>(codes);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == GDN2_F32)
    k_state_read<float><<<dim3(blocks_for(n, 4), B), 256, 0, s>>>(c, scales, slots,
                                                                  static_cast<float*>(h), S, n);
  else
    k_state_read<__nv_bfloat16><<<dim3(blocks_for(n, 2), B), 256, 0, s>>>(
        c, scales, slots, static_cast<__nv_bfloat16*>(h), S, n);
  return launched();
}
