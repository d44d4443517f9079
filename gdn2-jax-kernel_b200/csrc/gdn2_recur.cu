// Gated linear recurrence (per channel, no counterpart in the reference): the
// diagonal member of the family that GDN-2 belongs to, on the same layouts and
// gates,
//     h_t = e^{g_t} h_{t-1} + w_t v_t,   o_t = h_t,   h_0 given,
// and its backward pass.  With c_t the gradient that leaves token t towards
// t-1, c_{T+1} = dh_final,
//     dh_t = dout_t + c_{t+1},   c_t = e^{g_t} dh_t,
//     dv_t = w_t dh_t,  dw_t = v_t dh_t,  dg_t = e^{g_t} h_{t-1} dh_t,  dh0 = c_1.
// Both directions are scans of maps x -> a x + b, joined by
//     (a2, b2) o (a1, b1) = (a2 a1, a2 b1 + b2).
//
// A CTA takes a tile of 64 tokens x 64 channels: 8 warps of 8 tokens, a lane
// holds 2 neighbouring channels, so a warp reads whole 64-value groups of a
// row.  A thread folds its 8 tokens, the warps join their maps through shared
// memory, and each thread walks its tokens again from the state that reaches
// it: every global byte moves once.  What moves bounds the kernels: float32
// 16 bytes a value forward, 28 backward.
//
// The tiles of a sequence run at the same time.  Each publishes its map before
// it waits for anything; sixteen tiles in a row form a group, and a tile walks
// from the state that enters its group through the maps of the tiles before it
// there.  The last tile of a group publishes the state that enters the next.
// So a sequence of n tiles is n / 16 dependent steps, every state is formed by
// the same operations whatever ran first (results do not depend on timing),
// and a tile reads at most 16 published maps of 512 bytes.  Tiles are taken in
// the order of time by a counter, so what a tile waits for has always started.
// A published word is 64 bits, (a, b) of one channel, with the sign bit of a
// (never negative) set: zeroed memory is "not yet", and no fence is needed.
//
// The forward keeps the state that enters each tile (1/64 of o).  The backward
// rebuilds the states inside a tile from it, so it does not read o; with int8
// checkpoints it does so from the 8-bit v and w, which makes its gradients
// those of the restored values, restarted from the true state every 64 tokens.
// Decays stay in their own type: a rounding of a log decay compounds over the
// sequence, one of v or w does not.
#include <type_traits>

#include "../../include/gdn2.h"
#include "gdn2_int8.cuh"

namespace gdn2 {
int report_error(int code, const char* msg);
}

using namespace gdn2;

namespace {

constexpr int kRows = 8;                 // tokens a thread holds
constexpr int kWarps = 8;
constexpr int kTile = kRows * kWarps;    // tokens of a tile: the interval of the kept states
static_assert(kTile == GDN2_RECUR_INTERVAL, "interval of the kept states");

// As loaded: what a row of two channels is before it is converted.
template <typename T> struct Raw;
template <> struct Raw<float> { using type = float2; };
template <> struct Raw<__nv_bfloat16> { using type = unsigned; };
template <> struct Raw<int8_t> { using type = unsigned short; };
template <typename T>
__device__ __forceinline__ typename Raw<T>::type ldraw(const T* p) {
  return __ldcs(reinterpret_cast<const typename Raw<T>::type*>(p));
}
__device__ __forceinline__ float2 value2(float2 v) { return v; }
__device__ __forceinline__ float2 value2(unsigned u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ float2 value2(unsigned short u) {
  const unsigned b = u ^ 0x8080u;
  return make_float2(code_f<0>(b), code_f<1>(b));
}
__device__ __forceinline__ void st2(float* p, float2 v) { __stcs(reinterpret_cast<float2*>(p), v); }
__device__ __forceinline__ void st2(__nv_bfloat16* p, float2 v) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  __stcs(reinterpret_cast<unsigned*>(p), *reinterpret_cast<const unsigned*>(&h));
}

// e^g, or from the pre-activation x of g = -softplus(x): sigmoid(-x), from
// e^{-|x|} so that neither end overflows or cancels.
__device__ __forceinline__ float sig_from(float e, bool high) { return (high ? 1.f : e) / (1.f + e); }
__device__ __forceinline__ float sig(float x) { return sig_from(expf(-fabsf(x)), x > 0.f); }
template <bool RAW>
__device__ __forceinline__ float2 decay2(float2 g) {
  return RAW ? make_float2(sig(-g.x), sig(-g.y)) : make_float2(expf(g.x), expf(g.y));
}
template <bool RAW>
__device__ __forceinline__ float2 gate2(float2 w) {
  return RAW ? make_float2(sig(w.x), sig(w.y)) : w;
}

// A map h -> a h + b of two channels.
struct Map { float2 a, b; };
__device__ __forceinline__ Map identity() { return {both(1.f), both(0.f)}; }
__device__ __forceinline__ Map after(Map m2, Map m1) { return {mul2(m2.a, m1.a), fma2(m2.a, m1.b, m2.b)}; }
__device__ __forceinline__ float2 apply(Map m, float2 h) { return fma2(m.a, h, m.b); }
__device__ __forceinline__ float4 flat(Map m) { return make_float4(m.a.x, m.a.y, m.b.x, m.b.y); }
__device__ __forceinline__ Map unflat(float4 f) { return {make_float2(f.x, f.y), make_float2(f.z, f.w)}; }

constexpr int kGroupTiles = 2 * kWarps;
constexpr int kPolls = 1 << 22;   // about two seconds, then the status word is set

// Scratch of one call with more than one tile, zeroed before the kernel.
struct Scratch {
  int* status;       // the header: [0] a wait ran out, [8] the tile counter
  ulonglong2* maps;  // [tile][chain][32 lanes]: the maps of two channels
  ulonglong2* enter; // [group][chain][32 lanes]: the states that enter groups 1..
};
size_t scratch_bytes(size_t tiles, size_t chains) {
  return 512 + (tiles + tiles / kGroupTiles + 1) * chains * 512;
}

__device__ __forceinline__ unsigned long long word(float a, float b) {
  return ((unsigned long long)__float_as_uint(b) << 32) | (__float_as_uint(a) | 0x80000000u);
}
__device__ __forceinline__ void publish(ulonglong2* p, Map m) {
  asm volatile("st.relaxed.gpu.global.v2.u64 [%0], {%1, %2};"
               ::"l"(p), "l"(word(m.a.x, m.b.x)), "l"(word(m.a.y, m.b.y)) : "memory");
}
__device__ __forceinline__ ulonglong2 peek(const ulonglong2* p) {
  ulonglong2 v;
  asm volatile("ld.relaxed.gpu.global.v2.u64 {%0, %1}, [%2];" : "=l"(v.x), "=l"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ bool there(ulonglong2 v) { return ((unsigned)v.x & (unsigned)v.y) >> 31; }
__device__ __forceinline__ Map unword(ulonglong2 v) {
  return {make_float2(__uint_as_float((unsigned)v.x & 0x7fffffffu), __uint_as_float((unsigned)v.y & 0x7fffffffu)),
          make_float2(__uint_as_float((unsigned)(v.x >> 32)), __uint_as_float((unsigned)(v.y >> 32)))};
}
// Waits until the words at p are there in every lane, kPolls times at most; a
// wait that runs out, here or elsewhere in the call, is in the status word and
// ends this one too.
__device__ Map await(const ulonglong2* p, int* status) {
  ulonglong2 v = peek(p);
  for (int i = 1; !__all_sync(0xffffffffu, there(v)); ++i) {
    if (i >= kPolls || (i % 4096 == 0 && *(volatile int*)status)) {
      if ((threadIdx.x & 31) == 0) atomicExch(status, 1);
      break;
    }
    v = peek(p);
  }
  return unword(v);
}

struct Args {
  const void *v, *w, *g;
  int8_t *v8, *w8;        // int8 checkpoints, or NULL
  float *vs, *ws;         // their scales
  const float *h0, *dout, *dhf;
  float *o, *hf, *kept;
  void *dv, *dw, *dg;
  float* dh0;
  Scratch s;
  int T, HD, tiles, chains;
};

// The tile of this CTA: (chain, index k in the order of the scan).
struct Place { int chain, k; };
__device__ __forceinline__ Place take_tile(const Args& p) {
  __shared__ int ticket;
  unsigned t = blockIdx.x;
  if (p.tiles > 1) {
    if (threadIdx.x == 0) ticket = atomicAdd(p.s.status + 8, 1);
    __syncthreads();
    t = (unsigned)ticket;
  }
  return {(int)(t % p.chains), (int)(t / p.chains)};
}

// The state that enters tile k of a chain, from the maps of its warps in the
// order of the scan (map, complete: the caller has synchronised) and `first`,
// the state that enters the sequence.
struct Joint {
  float4 mates[kGroupTiles][32];
  float2 enter[32];
};
__device__ __forceinline__ float2 enter_tile(const Args& p, const Place at,
                                             const float4 (*map)[32], Joint& joint,
                                             const float* first) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int mate = at.k % kGroupTiles, group = at.k / kGroupTiles;
  const bool last = at.k + 1 == p.tiles, hands_on = mate == kGroupTiles - 1 && !last;
  if (warp == 0 && !last && !hands_on) {
    Map m = unflat(map[0][lane]);
#pragma unroll
    for (int j = 1; j < kWarps; ++j) m = after(unflat(map[j][lane]), m);
    publish(p.s.maps + ((size_t)at.k * p.chains + at.chain) * 32 + lane, m);
  }
  const ulonglong2* mine = p.s.maps + ((size_t)(at.k - mate) * p.chains + at.chain) * 32 + lane;
  const size_t next = (size_t)p.chains * 32;
  if (warp < mate) {   // two waits at once: the second has mostly come when the first has
    const bool two = warp + kWarps < mate;
    const ulonglong2 second = two ? peek(mine + (warp + kWarps) * next) : ulonglong2{};
    joint.mates[warp][lane] = flat(await(mine + warp * next, p.s.status));
    if (two)
      joint.mates[warp + kWarps][lane] =
          flat(__all_sync(0xffffffffu, there(second)) ? unword(second)
                                                      : await(mine + (warp + kWarps) * next, p.s.status));
  }
  if (mate) __syncthreads();
  if (warp == 0) {
    // the step from group to group is the dependent one: everything else of it
    // is joined before the wait
    Map m = identity();
    if (hands_on) {
      for (int i = 0; i < mate; ++i) m = after(unflat(joint.mates[i][lane]), m);
#pragma unroll
      for (int j = 0; j < kWarps; ++j) m = after(unflat(map[j][lane]), m);
    }
    float2 h = both(0.f);
    if (group)
      h = await(p.s.enter + ((size_t)group * p.chains + at.chain) * 32 + lane, p.s.status).b;
    else if (first)
      h = *reinterpret_cast<const float2*>(first + (size_t)at.chain * kGroup + 2 * lane);
    if (hands_on)
      publish(p.s.enter + ((size_t)(group + 1) * p.chains + at.chain) * 32 + lane,
              {both(0.f), apply(m, h)});
    joint.enter[lane] = h;
  }
  __syncthreads();
  float2 h = joint.enter[lane];
  for (int i = 0; i < mate; ++i) h = apply(unflat(joint.mates[i][lane]), h);
  return h;
}

// The int8 forms of a warp's 16 groups (8 rows of two tensors): codes are
// stored here, lane 2 r + j keeps the scale of tensor j's row r (one division a
// lane instead of one a group).
__device__ __forceinline__ float put_int8(const float2 (&v)[kRows], const float2 (&w)[kRows],
                                          int8_t* v8, int8_t* w8, size_t stride, int rows, int lane) {
  float mine = 0.f;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const float tv = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(max_abs(v[r].x, v[r].y))));
    const float tw = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(max_abs(w[r].x, w[r].y))));
    unsigned c[2], d[2];
    int8_codes<2>({v[r].x, v[r].y}, group_inv(tv), tv, c);
    int8_codes<2>({w[r].x, w[r].y}, group_inv(tw), tw, d);
    if (r < rows) {
      *reinterpret_cast<unsigned short*>(v8 + r * stride) = (unsigned short)__byte_perm(c[0], c[1], 0x0040);
      *reinterpret_cast<unsigned short*>(w8 + r * stride) = (unsigned short)__byte_perm(d[0], d[1], 0x0040);
    }
    mine = lane == 2 * r ? tv : lane == 2 * r + 1 ? tw : mine;
  }
  return group_scale(mine);
}

template <typename T, bool SAVE8, bool RAW>
__global__ void __launch_bounds__(256) k_recur_fwd(const Args p) {
  __shared__ float4 map[kWarps][32];   // (a, b) of two channels
  __shared__ Joint joint;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place at = take_tile(p);
  const int groups = p.HD / kGroup, bb = at.chain / groups, cg = at.chain % groups;
  const int ch = cg * kGroup + 2 * lane, t0 = at.k * kTile + warp * kRows;
  const int rows = min(kRows, p.T - t0);   // of this warp; below 1: none
  const size_t i0 = ((size_t)bb * p.T + t0) * p.HD + ch;
  float2 a[kRows], x[kRows];
  if (rows > 0) {
    // every load before any arithmetic; rows behind the end read the last one
    typename Raw<T>::type rg[kRows], rv[kRows], rw[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const size_t i = i0 + (size_t)min(r, rows - 1) * p.HD;
      rg[r] = ldraw(static_cast<const T*>(p.g) + i);
      rv[r] = ldraw(static_cast<const T*>(p.v) + i);
      rw[r] = ldraw(static_cast<const T*>(p.w) + i);
    }
    if constexpr (SAVE8) {
      float2 v[kRows], w[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        v[r] = value2(rv[r]);
        w[r] = value2(rw[r]);
      }
      const float scale = put_int8(v, w, p.v8 + i0, p.w8 + i0, p.HD, rows, lane);
      if (lane < 2 * rows)
        (lane & 1 ? p.ws : p.vs)[(i0 - 2 * lane) / kGroup + (size_t)(lane >> 1) * groups] = scale;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      a[r] = decay2<RAW>(value2(rg[r]));
      x[r] = mul2(gate2<RAW>(value2(rw[r])), value2(rv[r]));
    }
  }
  if (rows < kRows) {
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (r >= rows) a[r] = both(1.f), x[r] = both(0.f);
  }
  Map m = {a[0], x[0]};
#pragma unroll
  for (int r = 1; r < kRows; ++r) m = after({a[r], x[r]}, m);
  map[warp][lane] = flat(m);
  __syncthreads();
  float2 h = enter_tile(p, at, map, joint, p.h0);
  if (warp == 0 && p.kept)
    *reinterpret_cast<float2*>(p.kept + ((size_t)bb * p.tiles + at.k) * p.HD + ch) = h;
  for (int j = 0; j < warp; ++j) h = apply(unflat(map[j][lane]), h);
  float* o = p.o + i0;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    h = apply({a[r], x[r]}, h);
    if (r < rows) st2(o + (size_t)r * p.HD, h);
  }
  // rows behind the end keep the state
  if (rows > 0 && t0 + rows == p.T) *reinterpret_cast<float2*>(p.hf + (size_t)bb * p.HD + ch) = h;
}

// Tiles in the order of the reverse scan: k = 0 is the last one in time, and the
// maps of its warps are kept from the last warp to the first.
template <typename T, bool FROM8, bool RAW>
__global__ void __launch_bounds__(256) k_recur_bwd(const Args p) {
  using V = typename std::conditional<FROM8, int8_t, T>::type;
  __shared__ float4 fmap[kWarps][32], rmap[kWarps][32];
  __shared__ Joint joint;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, back = kWarps - 1 - warp;
  const Place at = take_tile(p);
  const int groups = p.HD / kGroup, bb = at.chain / groups, cg = at.chain % groups;
  const int tile = p.tiles - 1 - at.k;
  const int ch = cg * kGroup + 2 * lane, t0 = tile * kTile + warp * kRows;
  const int rows = min(kRows, p.T - t0);
  const size_t i0 = ((size_t)bb * p.T + t0) * p.HD + ch;
  float2 h = *reinterpret_cast<const float2*>(p.kept + ((size_t)bb * p.tiles + tile) * p.HD + ch);
  float2 a[kRows], v[kRows], w[kRows], d[kRows];
  if (rows > 0) {
    typename Raw<T>::type rg[kRows];
    typename Raw<V>::type rv[kRows], rw[kRows];
    float scale = 0.f;   // lane 2 r + j: of tensor j's row r
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const size_t i = i0 + (size_t)min(r, rows - 1) * p.HD;
      rv[r] = ldraw((FROM8 ? reinterpret_cast<const V*>(p.v8) : static_cast<const V*>(p.v)) + i);
      rw[r] = ldraw((FROM8 ? reinterpret_cast<const V*>(p.w8) : static_cast<const V*>(p.w)) + i);
      rg[r] = ldraw(static_cast<const T*>(p.g) + i);
      d[r] = ldraw(p.dout + i);
    }
    if (FROM8 && lane < 2 * rows)
      scale = (lane & 1 ? p.ws : p.vs)[(i0 - 2 * lane) / kGroup + (size_t)(lane >> 1) * groups];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      v[r] = value2(rv[r]);
      w[r] = value2(rw[r]);
      if constexpr (FROM8) {
        v[r] = mul2(v[r], both(__shfl_sync(0xffffffffu, scale, 2 * r)));
        w[r] = mul2(w[r], both(__shfl_sync(0xffffffffu, scale, 2 * r + 1)));
      }
      w[r] = gate2<RAW>(w[r]);
      a[r] = decay2<RAW>(value2(rg[r]));
    }
  }
  if (rows < kRows) {   // the identity, in both directions
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (r >= rows) a[r] = both(1.f), v[r] = w[r] = d[r] = both(0.f);
  }
  Map m = {a[0], mul2(w[0], v[0])}, n = identity();
#pragma unroll
  for (int r = 1; r < kRows; ++r) m = after({a[r], mul2(w[r], v[r])}, m);
#pragma unroll
  for (int r = kRows - 1; r >= 0; --r) n.b = mul2(a[r], add2(d[r], n.b));
  n.a = m.a;
  fmap[warp][lane] = flat(m);
  rmap[back][lane] = flat(n);
  __syncthreads();
  float2 c = enter_tile(p, at, rmap, joint, p.dhf);
  for (int j = 0; j < warp; ++j) h = apply(unflat(fmap[j][lane]), h);
  for (int j = 0; j < back; ++j) c = apply(unflat(rmap[j][lane]), c);
  float2 before[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    before[r] = h;
    h = apply({a[r], mul2(w[r], v[r])}, h);
  }
#pragma unroll
  for (int r = kRows - 1; r >= 0; --r) {
    const float2 dh = add2(d[r], c);
    c = mul2(a[r], dh);
    if (r < rows) {
      const size_t i = i0 + (size_t)r * p.HD;
      float2 dw = mul2(v[r], dh), dg = mul2(before[r], c);
      if constexpr (RAW) {
        // d sigmoid(x) = w (1 - w); dg/dx = -sigmoid(x)
        dw = make_float2(dw.x * (w[r].x * (1.f - w[r].x)), dw.y * (w[r].y * (1.f - w[r].y)));
        const float2 g = value2(ldraw(static_cast<const T*>(p.g) + i));   // in L2
        dg = make_float2(-dg.x * sig(g.x), -dg.y * sig(g.y));
      }
      st2(static_cast<T*>(p.dv) + i, mul2(w[r], dh));
      st2(static_cast<T*>(p.dw) + i, dw);
      st2(static_cast<T*>(p.dg) + i, dg);
    }
  }
  if (tile == 0 && warp == 0) *reinterpret_cast<float2*>(p.dh0 + (size_t)bb * p.HD + ch) = c;
}

template <bool FWD, typename T>
void launch(const Args& p, bool int8, bool raw, cudaStream_t s) {
  const unsigned grid = (unsigned)((size_t)p.chains * p.tiles);
  auto go = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>(p); };
  if constexpr (FWD) {
    if (int8) raw ? go(k_recur_fwd<T, true, true>) : go(k_recur_fwd<T, true, false>);
    else raw ? go(k_recur_fwd<T, false, true>) : go(k_recur_fwd<T, false, false>);
  } else {
    if (int8) raw ? go(k_recur_bwd<T, true, true>) : go(k_recur_bwd<T, true, false>);
    else raw ? go(k_recur_bwd<T, false, true>) : go(k_recur_bwd<T, false, false>);
  }
}

int check(int dtype, int B, int T, int H, int D) {
  if (dtype != GDN2_F32 && dtype != GDN2_BF16)
    return report_error(GDN2_ERR_INVALID, "gdn2_recur: unsupported dtype code");
  if (B <= 0 || T <= 0 || H <= 0)
    return report_error(GDN2_ERR_INVALID, "gdn2_recur: empty problem B*T*H");
  if (D != 64 && D != 128 && D != 256)
    return report_error(GDN2_ERR_INVALID, "gdn2_recur: head dim D unsupported (64, 128 or 256)");
  const long chains = (long)B * ((long)H * (D / kGroup));
  if (T > (1 << 30) || (long)H * D > (1 << 24) || chains > (1 << 26) ||
      chains * ((T + kTile - 1) / kTile) > 0x7fffffffL)
    return report_error(GDN2_ERR_INVALID, "gdn2_recur: too many tokens or channels");
  return GDN2_OK;
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

// Zeroes the scratch: the status header that gdn2_workspace_status() reads, the
// tile counter and every published word.
int prepare(Args& p, int B, void* workspace, cudaStream_t s) {
  p.chains = B * (p.HD / kGroup);
  if (p.tiles == 1) return GDN2_OK;
  char* base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~(uintptr_t)255);
  p.s.status = reinterpret_cast<int*>(base);
  p.s.maps = reinterpret_cast<ulonglong2*>(base + 256);
  p.s.enter = p.s.maps + (size_t)p.tiles * p.chains * 32;
  const cudaError_t e = cudaMemsetAsync(base, 0, scratch_bytes(p.tiles, p.chains) - 256, s);
  return e == cudaSuccess ? GDN2_OK : report_error(GDN2_ERR_CUDA, cudaGetErrorString(e));
}

int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GDN2_OK : report_error(GDN2_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace

extern "C" size_t gdn2_recur_kept_floats(int B, int T, int H, int D) {
  if (check(GDN2_F32, B, T, H, D)) return 0;
  return (size_t)B * ((T + kTile - 1) / kTile) * H * D;
}

extern "C" size_t gdn2_recur_workspace_bytes(int B, int T, int H, int D) {
  if (check(GDN2_F32, B, T, H, D)) return 0;
  return scratch_bytes((T + kTile - 1) / kTile, (size_t)B * H * D / kGroup);
}

extern "C" int gdn2_recur_fwd(int dtype, const void* v, const void* w, const void* g,
                              const float* h0, float* o, float* h_final, float* kept, void* v8,
                              float* v_scales, void* w8, float* w_scales, void* workspace,
                              size_t workspace_bytes, int B, int T, int H, int D, void* stream) {
  const int raw = (dtype & GDN2_GATES_RAW) != 0;
  dtype &= ~GDN2_GATES_RAW;
  const int rc = check(dtype, B, T, H, D);
  if (rc) return rc;
  const bool save8 = v8 || w8 || v_scales || w_scales;
  if (!v || !w || !g || !o || !h_final || (save8 && (!v8 || !w8 || !v_scales || !w_scales)))
    return report_error(GDN2_ERR_INVALID, "gdn2_recur_fwd: null buffer pointer");
  if (misaligned(v) || misaligned(w) || misaligned(g) || misaligned(h0) || misaligned(o) ||
      misaligned(h_final) || misaligned(kept) || misaligned(v8) || misaligned(w8))
    return report_error(GDN2_ERR_INVALID, "gdn2_recur_fwd: buffers must be 16-byte aligned");
  if (T > kTile && (!workspace || workspace_bytes < gdn2_recur_workspace_bytes(B, T, H, D)))
    return report_error(GDN2_ERR_WORKSPACE, "gdn2_recur_fwd: workspace too small");
  Args p{};
  p.v = v; p.w = w; p.g = g; p.h0 = h0; p.o = o; p.hf = h_final; p.kept = kept;
  p.v8 = static_cast<int8_t*>(v8); p.w8 = static_cast<int8_t*>(w8);
  p.vs = v_scales; p.ws = w_scales;
  p.T = T; p.HD = H * D; p.tiles = (T + kTile - 1) / kTile;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int e = prepare(p, B, workspace, s);
  if (e) return e;
  if (dtype == GDN2_F32) launch<true, float>(p, save8, raw, s);
  else launch<true, __nv_bfloat16>(p, save8, raw, s);
  return launched();
}

extern "C" int gdn2_recur_bwd(int dtype, const void* v, const void* w, const void* g,
                              const void* v8, const float* v_scales, const void* w8,
                              const float* w_scales, const float* kept, const float* dout,
                              const float* dh_final, void* dv, void* dw, void* dg, float* dh0,
                              void* workspace, size_t workspace_bytes, int B, int T, int H, int D,
                              void* stream) {
  const int raw = (dtype & GDN2_GATES_RAW) != 0;
  dtype &= ~GDN2_GATES_RAW;
  const int rc = check(dtype, B, T, H, D);
  if (rc) return rc;
  const bool from8 = v8 || w8 || v_scales || w_scales;
  if (from8 ? (!v8 || !w8 || !v_scales || !w_scales) : (!v || !w))
    return report_error(GDN2_ERR_INVALID, "gdn2_recur_bwd: null buffer pointer");
  if (!g || !kept || !dout || !dv || !dw || !dg || !dh0)
    return report_error(GDN2_ERR_INVALID, "gdn2_recur_bwd: null buffer pointer");
  if (misaligned(v) || misaligned(w) || misaligned(g) || misaligned(v8) || misaligned(w8) ||
      misaligned(kept) || misaligned(dout) || misaligned(dh_final) || misaligned(dv) ||
      misaligned(dw) || misaligned(dg) || misaligned(dh0))
    return report_error(GDN2_ERR_INVALID, "gdn2_recur_bwd: buffers must be 16-byte aligned");
  if (T > kTile && (!workspace || workspace_bytes < gdn2_recur_workspace_bytes(B, T, H, D)))
    return report_error(GDN2_ERR_WORKSPACE, "gdn2_recur_bwd: workspace too small");
  Args p{};
  p.v = v; p.w = w; p.g = g;
  p.v8 = static_cast<int8_t*>(const_cast<void*>(v8));
  p.w8 = static_cast<int8_t*>(const_cast<void*>(w8));
  p.vs = const_cast<float*>(v_scales); p.ws = const_cast<float*>(w_scales);
  p.kept = const_cast<float*>(kept); p.dout = dout; p.dhf = dh_final;
  p.dv = dv; p.dw = dw; p.dg = dg; p.dh0 = dh0;
  p.T = T; p.HD = H * D; p.tiles = (T + kTile - 1) / kTile;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int e = prepare(p, B, workspace, s);
  if (e) return e;
  if (dtype == GDN2_F32) launch<false, float>(p, from8, raw, s);
  else launch<false, __nv_bfloat16>(p, from8, raw, s);
  return launched();
}
