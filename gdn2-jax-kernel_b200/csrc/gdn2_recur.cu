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
// it: every global byte moves once.  What moves bounds the float32 kernels:
// 16 bytes a value forward, 28 backward.  The bf16 and int8 ones move less for 64
// to 140 instructions a row of 64 channels, issued at 1.6 to 2.3 of 4 a cycle: what
// bounds them is the latency that 16 warps an SM, which wait for one another twice
// a tile, do not hide.  Of the measured copy rate, forward / backward:
//     B8 T8192 H6 D128    float32  133 us (92%) / 225 us (96%)
//                         with int8 checkpoints 176 (79%) / 231 (74%)
//     B1 T131072 H8 D128  float32  351 (93%) / 569 (101%)
//                         bf16     299 (69%) / 428 (77%), int8 383 (65%) / 459 (63%)
// Raw gates cost exponentials and reciprocals: 153 / 346 us, with
// int8 checkpoints 203 / 312, for the first; 357 / 703, 456 / 702 for the last.
//
// The tiles of a sequence run at the same time.  Each publishes its map before
// it waits for anything.  Eight tiles in a row form a group; a tile walks from
// the state that enters the group BEFORE its own through the maps of the 8 to 15
// tiles since, so that state is at least 8 tiles old and has mostly come long
// ago.  (Walking from its own group's state, with groups of 16, left no slack to
// the first tiles of a group: 398 us instead of 350 for one sequence of
// 131072 tokens and 1024 channels, float32 forward.)  The last tile of a group
// publishes the state that enters the next.  So a sequence of n tiles is n / 16
// dependent steps of 0.57 us (few chains wait for them: one of 131072 tokens and
// 64 channels takes 76 / 86 us, 27% / 42% of the copy rate), every state is formed by the same operations
// whatever ran first (results do not depend on timing), and a tile reads at most
// 16 published words of 512 bytes.  A published word is 64 bits, (a, b) of one
// channel, with the sign bit of a (never negative) set: zeroed memory is "not
// yet", and no fence is needed.
//
// What a tile waits for is resolved by others while its CTA works: a CTA folds
// and publishes the next tile before it finishes the present one, and the bytes
// of the tile after that are on their way to shared memory.  (With the join in
// the way of the loads the float32 kernels reached 73% and 80% of the copy rate.)
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
  return *reinterpret_cast<const typename Raw<T>::type*>(p);
}

// Asynchronous copies to shared memory of 8 rows of 64 channels by one warp;
// rows behind the end are left as they are.
template <typename T>
__device__ __forceinline__ void fetch(T* to, const T* from, size_t stride, int rows, int lane) {
  constexpr int kPieces = kGroup * sizeof(T) / 16, kAt = 32 / kPieces;   // of a row; rows at once
#pragma unroll
  for (int r0 = 0; r0 < kRows; r0 += kAt) {
    const int r = r0 + lane / kPieces, c = lane % kPieces * (16 / sizeof(T));
    if (r < rows)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                   ::"r"((unsigned)__cvta_generic_to_shared(to + r * kGroup + c)),
                     "l"(from + r * stride + c) : "memory");
  }
}
__device__ __forceinline__ void fetch4(float* to, const float* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;"
               ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void fetch_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All fetches but the latest `N` have landed, for the whole warp.
template <int N>
__device__ __forceinline__ void fetched() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
  __syncwarp();
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

// e^g as 2^(g log2 e): off by 2^-22 + |g| 2^-23 of itself (0 below 2^-126).  The
// part that grows with |g| does not add up over a sequence: after decays that
// sum to S a term has the weight e^-S, and S e^-S 2^-23 is at most 2^-24.4 of it
// where expf took 16 of the 40 instructions of a row.
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;
// sigmoid(x) and its derivative sigmoid(x) sigmoid(-x) from e^{-|x|}, so that
// neither end overflows or cancels (1 - sigmoid(x) does where a gate is open);
// subnormal values stay (the gradient of a gate that is nearly shut).
__device__ __forceinline__ float2 sig_slope(float x) {
  float e, r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(-kLog2e * fabsf(x)));
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return make_float2(x > 0.f ? r : e * r, e * r * r);
}
__device__ __forceinline__ float sig(float x) { return sig_slope(x).x; }
// e^g, or from the pre-activation x of g = -softplus(x): sigmoid(-x).
template <bool RAW>
__device__ __forceinline__ float2 decay2(float2 g) {
  if constexpr (RAW) return make_float2(sig(-g.x), sig(-g.y));
  const float2 t = mul2(g, both(kLog2e));
  return make_float2(ex2(t.x), ex2(t.y));
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

constexpr int kGroupTiles = kWarps;   // a warp looks at two of the maps of two groups
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
// Waits until the words at p are there in every lane, `polls` polls at most; a
// wait that runs out, here or elsewhere in the call, is in the status word and
// ends this one too.
__device__ Map await(const ulonglong2* p, int* status, int polls = kPolls) {
  ulonglong2 v = peek(p);
  for (int i = 1; !__all_sync(0xffffffffu, there(v)); ++i) {
    // (lanes may read different status words: the warp leaves together or not at all)
    if ((i >= polls || i % 4096 == 0) &&
        __any_sync(0xffffffffu, i >= polls || *(volatile int*)status)) {
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

// Tiles are taken in the order of time: ticket t is tile t / chains of chain
// t % chains, in the order of the scan.  A CTA holds the tile it works on, the
// next one and the one after; what a tile waits for has a lower ticket, and the
// lowest unfinished ticket is always being worked on.  Sequences of one tile
// wait for nothing and are dealt out by index.
// A ticket is taken apart by one thread for all (four divisions a warp for every
// tile cost a third of the instructions).
struct Place { int k, chain, bb, cg; };   // k < 0: none left
struct Tickets {
  bool drawn, more;   // from the counter; more than one a CTA
  int total, mine;    // mine: of thread 0, the latest
  __device__ __forceinline__ Tickets(const Args& p)
      : drawn(p.tiles > 1), more(p.tiles * p.chains > (int)gridDim.x), total(p.tiles * p.chains), mine(0) {}
  // thread 0: asks for a ticket, then takes it apart
  __device__ __forceinline__ void ask(const Args& p, bool first) {
    if (!first && !more) mine = total;
    else if (drawn) mine = atomicAdd(p.s.status + 8, 1);
    else mine = first ? (int)blockIdx.x : mine + (int)gridDim.x;
  }
  __device__ __forceinline__ int4 place(const Args& p) const {
    if (mine >= total) return make_int4(-1, 0, 0, 0);
    const unsigned chain = (unsigned)mine % p.chains, groups = p.HD / kGroup;
    return make_int4((unsigned)mine / p.chains, chain, chain / groups, chain % groups);
  }
};
__device__ __forceinline__ Place told(const int4& z) { return {z.x, z.y, z.z, z.w}; }

// How a tile of a chain gets the state that enters it.
using Maps = float4[kWarps][32];   // of the warps, in the order of the scan
struct Joint {
  Maps maps;                  // of the warps of one tile
  Maps upto[2];               // [w]: warps 0 .. w, of the present and the next tile
  float4 pairs[kWarps][32];   // the tiles 2 w and 2 w + 1 since the start
  float2 enter[32];           // the state at the start
  int4 place[2];
};
__device__ __forceinline__ ulonglong2* map_of(const Args& p, Place at, int k, int lane) {
  return p.s.maps + ((size_t)k * p.chains + at.chain) * 32 + lane;
}
__device__ __forceinline__ ulonglong2* enter_of(const Args& p, Place at, int group, int lane) {
  return p.s.enter + ((size_t)group * p.chains + at.chain) * 32 + lane;
}
// Where a tile's walk starts: the group before its own.
__device__ __forceinline__ int start_group(Place at) { return max(at.k / kGroupTiles - 1, 0); }
// One warp: maps -> the maps of warps 0 .. w, the whole tile's last.
__device__ __forceinline__ Map prefixes(const Maps& maps, Maps& upto, int lane) {
  Map m[kWarps];   // all loads before the first store, which they could alias for the compiler
#pragma unroll
  for (int j = 0; j < kWarps; ++j) m[j] = unflat(maps[j][lane]);
#pragma unroll
  for (int j = 1; j < kWarps; ++j) m[j] = after(m[j], m[j - 1]);
#pragma unroll
  for (int j = 0; j < kWarps; ++j) upto[j][lane] = flat(m[j]);
  return m[kWarps - 1];
}
__device__ __forceinline__ float2 past(const Maps& upto, int warps, int lane, float2 h) {
  return warps ? apply(unflat(upto[warps - 1][lane]), h) : h;
}
// The same warp publishes the tile's map, where another tile will look at it.
__device__ __forceinline__ void publish_map(const Args& p, Place at, Map m, int lane) {
  if (at.k + 1 < p.tiles) publish(map_of(p, at, at.k, lane), m);
}
// What a warp needs of others, looked at long before it is needed: two of at most
// 15 maps, or for the last warp one and the state at the start.
struct Early { ulonglong2 even, odd; };
__device__ __forceinline__ Early look(const Args& p, Place at, int warp, int lane) {
  const int start = start_group(at), k = start * kGroupTiles + 2 * warp;
  Early e{};
  if (k < at.k) e.even = peek(map_of(p, at, k, lane));
  if (k + 1 < at.k) e.odd = peek(map_of(p, at, k + 1, lane));
  if (warp == kWarps - 1 && start) e.odd = peek(enter_of(p, at, start, lane));
  return e;
}
__device__ __forceinline__ Map have(ulonglong2 early, const ulonglong2* p, int* status) {
  return __all_sync(0xffffffffu, there(early)) ? unword(early) : await(p, status);
}
// All warps, between two synchronisations of the CTA; fills `joint`.
__device__ __forceinline__ void join(const Args& p, Place at, const Maps& upto, Joint& joint,
                                     const float* first, const Early& e, int warp, int lane) {
  const int start = start_group(at), k = start * kGroupTiles + 2 * warp;
  const bool hands_on = at.k % kGroupTiles == kGroupTiles - 1 && at.k + 1 < p.tiles;
  Map m = identity();
  if (k < at.k) m = have(e.even, map_of(p, at, k, lane), p.s.status);
  if (k + 1 < at.k) m = after(have(e.odd, map_of(p, at, k + 1, lane), p.s.status), m);
  joint.pairs[warp][lane] = flat(m);
  if (hands_on) {
    // the step from group to group is the dependent one: everything else of it
    // is joined before the wait
    __syncthreads();
    if (warp == kWarps - 1) {
      m = unflat(joint.pairs[0][lane]);
#pragma unroll
      for (int i = 1; i < kWarps; ++i) m = after(unflat(joint.pairs[i][lane]), m);
      m = after(unflat(upto[kWarps - 1][lane]), m);
    }
  }
  if (warp == kWarps - 1) {
    float2 h = both(0.f);
    if (start)
      h = have(e.odd, enter_of(p, at, start, lane), p.s.status).b;
    else if (first)
      h = *reinterpret_cast<const float2*>(first + (size_t)at.chain * kGroup + 2 * lane);
    if (hands_on)
      publish(enter_of(p, at, at.k / kGroupTiles + 1, lane), {both(0.f), apply(m, h)});
    joint.enter[lane] = h;
  }
}
__device__ __forceinline__ float2 entering(const Joint& joint, int lane) {
  float2 h = joint.enter[lane];
#pragma unroll
  for (int i = 0; i < kWarps; ++i) h = apply(unflat(joint.pairs[i][lane]), h);
  return h;
}
// The int8 form of a warp's 8 rows (groups) of one tensor: 4 lanes take a row, 16
// values each, so a group's maximum takes two shuffles, every lane's division is
// a group's, and its codes leave as one 16-byte store.  (Lanes of two channels,
// as the recurrence has them, took 37 instructions a row instead of 10.)
template <typename T>
__device__ __forceinline__ void put_int8(const T (*x)[kGroup], int8_t* codes, float* scales,
                                         size_t stride, int groups, int rows, int lane) {
  constexpr int E = 16 / sizeof(T), N = 16 / E;   // values of a 16-byte piece; pieces of a lane
  const int r = lane >> 2, q = lane & 3;
  float v[16], top = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    // the quarter's pieces in an order of its own: fewer lanes on one bank
    const int piece = (i + q) % N;
    const uint4 u = *reinterpret_cast<const uint4*>(&x[r][q * 16 + piece * E]);
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (E == 4) v[i * 4 + k] = __uint_as_float(w[k]);
      else {
        v[i * 8 + 2 * k] = __uint_as_float(w[k] << 16);
        v[i * 8 + 2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 16; i += 2) top = max_abs3(top, v[i], v[i + 1]);
  top = max_abs(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max_abs(top, __shfl_xor_sync(0xffffffffu, top, 2));
  unsigned c[16];
  int8_codes<T, 16>(v, top, c);
  unsigned word[4], out[4];   // word i: in the order of the loads
#pragma unroll
  for (int i = 0; i < 4; ++i) word[i] = pack4(c[4 * i], c[4 * i + 1], c[4 * i + 2], c[4 * i + 3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {   // turned back by q pieces of 4 / N words
    if constexpr (N == 4) {
      const unsigned one = q & 1 ? word[(i + 3) & 3] : word[i];
      const unsigned two = q & 1 ? word[(i + 1) & 3] : word[(i + 2) & 3];
      out[i] = q & 2 ? two : one;
    } else {
      out[i] = q & 1 ? word[i ^ 2] : word[i];
    }
  }
  if (r < rows) {
    *reinterpret_cast<uint4*>(codes + r * stride + q * 16) = make_uint4(out[0], out[1], out[2], out[3]);
    if (q == 0) scales[(size_t)r * groups] = group_scale(top);
  }
}

// Where a tile lies for a warp: rows of it (8 and more: all eight), first element.
struct Rows { int rows; size_t i; };
__device__ __forceinline__ Rows rows_of(const Args& p, Place at, int tile, int warp) {
  const int t0 = tile * kTile + warp * kRows;
  return {p.T - t0, ((size_t)at.bb * p.T + t0) * p.HD + at.cg * kGroup};
}

// The first two tiles of a CTA: the first is folded and published, the second on
// its way.  False where there is none.
template <typename Prefetch, typename Fold>
__device__ __forceinline__ bool begin(const Args& p, Tickets& tickets, Joint& joint, Place& now,
                                      Place& next, Prefetch prefetch, Fold fold, int warp, int lane) {
  if (threadIdx.x == 0) {
    tickets.ask(p, true);
    joint.place[0] = tickets.place(p);
  }
  __syncthreads();
  now = told(joint.place[0]);
  if (now.k < 0) return false;
  prefetch(now);
  fold(now);
  // the second ticket once the first tile's bytes are there, when other CTAs have
  // theirs: one that drew two at once would leave another without any
  if (threadIdx.x == 0) {
    tickets.ask(p, false);
    joint.place[1] = tickets.place(p);
  }
  __syncthreads();
  next = told(joint.place[1]);
  prefetch(next);
  if (warp == 1) publish_map(p, now, prefixes(joint.maps, joint.upto[0], lane), lane);
  __syncthreads();
  return true;
}

// Shared memory of a warp: its 8 rows of the tile that comes next.
template <typename T> struct FwdStage { T g[kRows][kGroup], v[kRows][kGroup], w[kRows][kGroup]; };

template <typename T, bool SAVE8, bool RAW>
__global__ void __launch_bounds__(256, 2) k_recur_fwd(const Args p) {
  extern __shared__ __align__(16) unsigned char raw_stage[];
  __shared__ Joint joint;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  FwdStage<T>& st = reinterpret_cast<FwdStage<T>*>(raw_stage)[warp];
  Tickets tickets(p);
  auto prefetch = [&](Place at) {
    if (at.k >= 0) {
      const Rows z = rows_of(p, at, at.k, warp);
      fetch(&st.g[0][0], static_cast<const T*>(p.g) + z.i, p.HD, z.rows, lane);
      fetch(&st.v[0][0], static_cast<const T*>(p.v) + z.i, p.HD, z.rows, lane);
      fetch(&st.w[0][0], static_cast<const T*>(p.w) + z.i, p.HD, z.rows, lane);
    }
    fetch_end();
  };
  // the rows of a tile as maps (a, x), and the map of the warp
  auto fold = [&](Place at, float2 (&a)[kRows], float2 (&x)[kRows]) {
    const Rows z = rows_of(p, at, at.k, warp);
    fetched<0>();
    if constexpr (SAVE8) {
      put_int8(st.v, p.v8 + z.i, p.vs + z.i / kGroup, p.HD, p.HD / kGroup, z.rows, lane);
      put_int8(st.w, p.w8 + z.i, p.ws + z.i / kGroup, p.HD, p.HD / kGroup, z.rows, lane);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      a[r] = decay2<RAW>(value2(ldraw(&st.g[r][2 * lane])));
      x[r] = mul2(gate2<RAW>(value2(ldraw(&st.w[r][2 * lane]))), value2(ldraw(&st.v[r][2 * lane])));
    }
    __syncwarp();
    if (z.rows < kRows) {   // rows behind the end keep the state
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (r >= z.rows) a[r] = both(1.f), x[r] = both(0.f);
    }
    Map m = {a[0], x[0]};
#pragma unroll
    for (int r = 1; r < kRows; ++r) m = after({a[r], x[r]}, m);
    joint.maps[warp][lane] = flat(m);
  };

  Place now, next;
  float2 a[2][kRows], x[2][kRows];
  if (!begin(p, tickets, joint, now, next, prefetch, [&](Place at) { fold(at, a[0], x[0]); }, warp, lane))
    return;
  // One tile: `me` of the two register sets holds it, the other takes the next.
  auto turn = [&](auto me) {
    constexpr int N = decltype(me)::value, M = N ^ 1;
    const Early early = look(p, now, warp, lane);
    if (threadIdx.x == 0) tickets.ask(p, false);
    const bool on = next.k >= 0;
    if (on) fold(next, a[M], x[M]);
    __syncthreads();
    if (warp == 1 && on) publish_map(p, next, prefixes(joint.maps, joint.upto[M], lane), lane);
    if (threadIdx.x == 0) joint.place[0] = tickets.place(p);
    join(p, now, joint.upto[N], joint, p.h0, early, warp, lane);
    __syncthreads();
    const Place later = told(joint.place[0]);
    prefetch(later);
    const Rows z = rows_of(p, now, now.k, warp);
    const int ch = now.cg * kGroup + 2 * lane;
    float2 h = entering(joint, lane);
    if (warp == 0 && p.kept)
      *reinterpret_cast<float2*>(p.kept + ((size_t)now.bb * p.tiles + now.k) * p.HD + ch) = h;
    h = past(joint.upto[N], warp, lane, h);
    float* o = p.o + z.i + 2 * lane;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      h = apply({a[N][r], x[N][r]}, h);
      if (r < z.rows) st2(o + (size_t)r * p.HD, h);
    }
    if (z.rows > 0 && z.rows <= kRows)
      *reinterpret_cast<float2*>(p.hf + (size_t)now.bb * p.HD + ch) = h;
    now = next;
    next = later;
    return now.k >= 0;
  };
  while (turn(std::integral_constant<int, 0>{}) && turn(std::integral_constant<int, 1>{})) {
  }
}

// A few tokens (generation): a warp takes a chain alone, one token after another,
// the loads of AHEAD tokens at a time (4 for calls that short, else 16).  No maps,
// no shared memory, no scratch; bound by the latency of a load and a store for
// every AHEAD tokens.
constexpr int kStepTokens = 32;
template <typename T, bool RAW, int AHEAD>
__global__ void __launch_bounds__(128) k_recur_step(const Args p) {
  const int lane = threadIdx.x & 31, chain = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (chain >= p.chains) return;
  const int groups = p.HD / kGroup, ch = chain % groups * kGroup + 2 * lane;
  const size_t bb = chain / groups, j = bb * p.HD + ch;
  float2 h = p.h0 ? *reinterpret_cast<const float2*>(p.h0 + j) : both(0.f);
  if (p.kept) *reinterpret_cast<float2*>(p.kept + j) = h;   // of the one interval
  for (int t0 = 0; t0 < p.T; t0 += AHEAD) {
    const int rows = p.T - t0;
    const size_t i0 = (bb * p.T + t0) * p.HD + ch;
    typename Raw<T>::type g[AHEAD], v[AHEAD], w[AHEAD];
#pragma unroll
    for (int t = 0; t < AHEAD; ++t) {   // tokens behind the end read the last one
      const size_t i = i0 + (size_t)min(t, rows - 1) * p.HD;
      g[t] = ldraw(static_cast<const T*>(p.g) + i);
      v[t] = ldraw(static_cast<const T*>(p.v) + i);
      w[t] = ldraw(static_cast<const T*>(p.w) + i);
    }
#pragma unroll
    for (int t = 0; t < AHEAD; ++t)
      if (t < rows) {
        h = apply({decay2<RAW>(value2(g[t])), mul2(gate2<RAW>(value2(w[t])), value2(v[t]))}, h);
        st2(p.o + i0 + (size_t)t * p.HD, h);
      }
  }
  *reinterpret_cast<float2*>(p.hf + j) = h;
}

// The reverse scan needs g and dout alone until the state that enters a tile is
// known; v and w come while the next tile is folded.
template <typename T, typename V> struct BwdStage {
  T g[kRows][kGroup];
  float d[kRows][kGroup];
  V v[kRows][kGroup], w[kRows][kGroup];
  float scale[2 * kRows];   // of int8 v and w: 2 r + j of tensor j's row r
};

// Tiles in the order of the reverse scan: k = 0 is the last one in time, and the
// maps of its warps stand from the last warp to the first.
template <typename T, bool FROM8, bool RAW>
__global__ void __launch_bounds__(256, 2) k_recur_bwd(const Args p) {
  using V = typename std::conditional<FROM8, int8_t, T>::type;
  extern __shared__ __align__(16) unsigned char raw_stage[];
  __shared__ Joint joint;
  __shared__ Maps fmaps, fupto;   // of the present tile's states, in the order of time
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, back = kWarps - 1 - warp;
  BwdStage<T, V>& st = reinterpret_cast<BwdStage<T, V>*>(raw_stage)[warp];
  const V* pv = FROM8 ? reinterpret_cast<const V*>(p.v8) : static_cast<const V*>(p.v);
  const V* pw = FROM8 ? reinterpret_cast<const V*>(p.w8) : static_cast<const V*>(p.w);
  Tickets tickets(p);
  auto prefetch = [&](Place at) {
    if (at.k >= 0) {
      const Rows z = rows_of(p, at, p.tiles - 1 - at.k, warp);
      fetch(&st.g[0][0], static_cast<const T*>(p.g) + z.i, p.HD, z.rows, lane);
      fetch(&st.d[0][0], p.dout + z.i, p.HD, z.rows, lane);
    }
    fetch_end();
  };
  auto prefetch_vw = [&](Place at) {
    if (at.k >= 0) {
      const Rows z = rows_of(p, at, p.tiles - 1 - at.k, warp);
      fetch(&st.v[0][0], pv + z.i, p.HD, z.rows, lane);
      fetch(&st.w[0][0], pw + z.i, p.HD, z.rows, lane);
      if (FROM8 && lane < 2 * min(z.rows, kRows))
        fetch4(&st.scale[lane], (lane & 1 ? p.ws : p.vs) + z.i / kGroup +
                                    (size_t)(lane >> 1) * (p.HD / kGroup));
    }
    fetch_end();
  };
  // decays and cotangents of a tile, and the warp's map of the reverse scan
  auto fold = [&](Place at, float2 (&a)[kRows], float2 (&d)[kRows]) {
    const int rows = p.T - (p.tiles - 1 - at.k) * kTile - warp * kRows;
    fetched<1>();
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      a[r] = decay2<RAW>(value2(ldraw(&st.g[r][2 * lane])));
      d[r] = ldraw(&st.d[r][2 * lane]);
    }
    __syncwarp();
    if (rows < kRows) {   // rows behind the end hand the cotangent on
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (r >= rows) a[r] = both(1.f), d[r] = both(0.f);
    }
    Map m = identity();
#pragma unroll
    for (int r = kRows - 1; r >= 0; --r) m = {mul2(a[r], m.a), mul2(a[r], add2(d[r], m.b))};
    joint.maps[back][lane] = flat(m);
  };
  // v, w and with raw gates dw/dx of row r of the present tile; behind the end
  // anything: only states that nothing reads come of it
  auto vw = [&](int r, float2& v, float2& w, float2& slope) {
    v = value2(ldraw(&st.v[r][2 * lane]));
    w = value2(ldraw(&st.w[r][2 * lane]));
    if constexpr (FROM8) {
      v = mul2(v, both(st.scale[2 * r]));
      w = mul2(w, both(st.scale[2 * r + 1]));
    }
    if constexpr (RAW) {
      const float2 x = sig_slope(w.x), y = sig_slope(w.y);
      w = make_float2(x.x, y.x);
      slope = make_float2(x.y, y.y);
    }
  };

  Place now, next;
  float2 a[2][kRows], d[2][kRows];
  if (!begin(p, tickets, joint, now, next, prefetch, [&](Place at) {
        prefetch_vw(at);
        fold(at, a[0], d[0]);
      }, warp, lane))
    return;
  // in flight at the end of each turn: g, dout of the next tile, then v, w of the
  // present one; here, once, the other way round
  fetched<0>();
  int side = 0;
  auto turn = [&](auto me) {
    constexpr int N = decltype(me)::value, M = N ^ 1;
    const int tile = p.tiles - 1 - now.k, ch = now.cg * kGroup + 2 * lane;
    const Rows z = rows_of(p, now, tile, warp);
    const Early early = look(p, now, warp, lane);
    float2 h = *reinterpret_cast<const float2*>(p.kept + ((size_t)now.bb * p.tiles + tile) * p.HD + ch);
    if (threadIdx.x == 0) tickets.ask(p, false);
    const bool on = next.k >= 0;
    if (on) fold(next, a[M], d[M]);
    fetched<0>();
    float2 x[kRows];   // w v, then the state before each row
    Map m = identity();
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float2 v, w, slope;
      vw(r, v, w, slope);
      x[r] = mul2(w, v);
      m = after({a[N][r], x[r]}, m);
    }
    fmaps[warp][lane] = flat(m);
    __syncthreads();
    if (warp == 1 && on) publish_map(p, next, prefixes(joint.maps, joint.upto[side ^ 1], lane), lane);
    if (warp == 2) prefixes(fmaps, fupto, lane);
    if (threadIdx.x == 0) joint.place[0] = tickets.place(p);
    join(p, now, joint.upto[side], joint, p.dhf, early, warp, lane);
    __syncthreads();
    const Place later = told(joint.place[0]);
    prefetch(later);
    h = past(fupto, warp, lane, h);
    float2 c = past(joint.upto[side], back, lane, entering(joint, lane));
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float2 after_r = apply({a[N][r], x[r]}, h);
      x[r] = h;
      h = after_r;
    }
#pragma unroll
    for (int r = kRows - 1; r >= 0; --r) {
      const float2 dh = add2(d[N][r], c);
      c = mul2(a[N][r], dh);
      if (r < z.rows) {
        const size_t i = z.i + 2 * lane + (size_t)r * p.HD;
        float2 v, w, slope;
        vw(r, v, w, slope);
        float2 dw = mul2(v, dh), dg = mul2(x[r], c);
        if constexpr (RAW) {
          dw = mul2(dw, slope);
          // dg/dx = -sigmoid(x)
          const float2 g = value2(ldraw(static_cast<const T*>(p.g) + i));   // in L2
          dg = make_float2(-dg.x * sig(g.x), -dg.y * sig(g.y));
        }
        st2(static_cast<T*>(p.dv) + i, mul2(w, dh));
        st2(static_cast<T*>(p.dw) + i, dw);
        st2(static_cast<T*>(p.dg) + i, dg);
      }
    }
    if (tile == 0 && warp == 0) *reinterpret_cast<float2*>(p.dh0 + (size_t)now.bb * p.HD + ch) = c;
    __syncwarp();
    prefetch_vw(next);
    now = next;
    next = later;
    side ^= 1;
    return now.k >= 0;
  };
  // (Two register sets in turn spill here: 263 us instead of 224 for B8 T8192 H6
  // D128 float32.)
  while (turn(std::integral_constant<int, 0>{})) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      a[0][r] = a[1][r];
      d[0][r] = d[1][r];
    }
  }
}

// Two warps that wait for words that nothing publishes: one gives up after `polls`
// polls, the other because of the first.
__global__ void k_recur_timeout(const ulonglong2* words, int* status, int polls) {
  await(words + threadIdx.x % 32, status, threadIdx.x < 32 ? polls : kPolls);
}

// One CTA for every place on the GPU, or one a tile where there are fewer.
template <typename K>
cudaError_t launch_tiles(K kernel, size_t stage, int per_sm, const Args& p, cudaStream_t s) {
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)stage);
  if (e != cudaSuccess) return e;
  const size_t tiles = (size_t)p.chains * p.tiles, places = (size_t)sms * per_sm;
  kernel<<<(unsigned)(tiles < places ? tiles : places), 256, stage, s>>>(p);
  return cudaGetLastError();
}
template <bool FWD, typename T>
cudaError_t launch(const Args& p, bool int8, bool raw, cudaStream_t s) {
  if constexpr (FWD) {
    // Few tokens: 1, 16 and 32 of 64 x 6 x 128 channels take 2.3, 3.4 and 4.6 us
    // this way, 7.4, 7.5 and 7.7 as tiles; 64 of 6 x 128 channels 5.3 against 3.8.
    if (p.T <= kStepTokens && !int8) {
      const unsigned grid = (unsigned)((p.chains + 3) / 4);
      auto step = [&](auto kernel) { kernel<<<grid, 128, 0, s>>>(p); };
      if (p.T <= 4) raw ? step(k_recur_step<T, true, 4>) : step(k_recur_step<T, false, 4>);
      else raw ? step(k_recur_step<T, true, 16>) : step(k_recur_step<T, false, 16>);
      return cudaGetLastError();
    }
    auto go = [&](auto kernel) { return launch_tiles(kernel, sizeof(FwdStage<T>) * kWarps, 2, p, s); };
    if (int8) return raw ? go(k_recur_fwd<T, true, true>) : go(k_recur_fwd<T, true, false>);
    return raw ? go(k_recur_fwd<T, false, true>) : go(k_recur_fwd<T, false, false>);
  } else {
    auto go = [&](auto kernel, size_t stage) { return launch_tiles(kernel, stage * kWarps, 2, p, s); };
    const size_t n = sizeof(BwdStage<T, T>), n8 = sizeof(BwdStage<T, int8_t>);
    if (int8) return raw ? go(k_recur_bwd<T, true, true>, n8) : go(k_recur_bwd<T, true, false>, n8);
    return raw ? go(k_recur_bwd<T, false, true>, n) : go(k_recur_bwd<T, false, false>, n);
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
      chains * ((T + kTile - 1) / kTile) > (1L << 30))   // tickets stay in 31 bits
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

int launched(cudaError_t e) {
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
  return launched(dtype == GDN2_F32 ? launch<true, float>(p, save8, raw, s)
                                    : launch<true, __nv_bfloat16>(p, save8, raw, s));
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
  return launched(dtype == GDN2_F32 ? launch<false, float>(p, from8, raw, s)
                                    : launch<false, __nv_bfloat16>(p, from8, raw, s));
}

extern "C" int gdn2_selftest_recur_timeout(void* workspace, size_t workspace_bytes, int polls,
                                           void* stream) {
  if (!workspace || workspace_bytes < 1024 || polls < 1)
    return report_error(GDN2_ERR_INVALID, "gdn2_selftest_recur_timeout: bad workspace or poll count");
  char* base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~(uintptr_t)255);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = cudaMemsetAsync(base, 0, 768, s);   // the header and 512 bytes of words
  if (e != cudaSuccess) return launched(e);
  k_recur_timeout<<<1, 64, 0, s>>>(reinterpret_cast<const ulonglong2*>(base + 256),
                                   reinterpret_cast<int*>(base), polls);
  return launched(cudaGetLastError());
}
