// Keys and values of packed sequences into a 4-bit cache, and back (layout and rule: int4.cuh).
//
// One block per (tile of a sequence, head).  The 16-bit side: 16 bytes a lane, a head's row by 8 or 16 lanes.  The 4-bit side: a tile is put together in shared memory and
// copied whole, 16 bytes a lane; where a sequence begins or ends inside it, its rows' words are written one by one and the others left alone.
#include "int4.cuh"

#include <algorithm>

namespace {

constexpr int kThreads = 128;

struct CacheParams {
  void *k, *v;                      // [T, nkv, D], element (t, h, c) at t * ts + h * hs + c
  int64_t kt, kh, vt, vh;
  uint32_t* cache;                  // [slots, nkv, tiles, Tile<D>::kWords]
  const int *cu, *slots, *start;    // [n + 1], [n] or null (sequence i: slot i), [n] or null (from row 0)
  int n, nkv, n_slots, room, tiles, T;
};

template <typename T, int D, bool kStore>
__global__ void __launch_bounds__(kThreads) cache_rows_kernel(CacheParams p) {
  using Tl = q4::Tile<D>;
  constexpr int LPR = D / 8, kGroups = kThreads / LPR, kTurns = 16 / kGroups;
  __shared__ __align__(16) uint32_t tile_words[Tl::kWords];
  rb::pdl_trigger();
  rb::pdl_wait();
  const int seq = blockIdx.x, head = blockIdx.y, sub = threadIdx.x % LPR;
  const int tok0 = min(max(p.cu[seq], 0), p.T), tok1 = min(max(p.cu[seq + 1], tok0), p.T);
  const int slot = p.slots ? p.slots[seq] : seq;
  const int64_t start = p.start ? p.start[seq] : 0;
  const bool there = slot >= 0 && slot < p.n_slots;
  if (kStore && !there) return;
  if constexpr (!kStore) {                          // tokens before the first sequence and behind the last belong to none
    const int lo = seq == p.n - 1 ? tok1 : 0, hi = seq == p.n - 1 ? p.T : 0, front = seq == 0 ? tok0 : 0;
    for (int i = blockIdx.z * kGroups + threadIdx.x / LPR; i < front + (hi - lo); i += gridDim.z * kGroups) {
      const int64_t tok = i < front ? i : lo + (i - front);
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.k) + tok * p.kt + head * p.kh + sub * 8) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.v) + tok * p.vt + head * p.vh + sub * 8) = make_uint4(0, 0, 0, 0);
    }
  }
  const int64_t first = (start < 0 ? start - 15 : start) / 16, last = start + (tok1 - tok0);   // tiles first .. ; rows below `last`
  for (int64_t tile = first + blockIdx.z; tile * 16 < last; tile += gridDim.z) {
    uint32_t* at = p.cache + (((int64_t)slot * p.nkv + head) * p.tiles + tile) * Tl::kWords;
    const bool held = there && tile >= 0 && tile < p.tiles;        // (rows at or beyond `room` are looked at one by one)
    const bool whole = held && tile * 16 >= start && tile * 16 + 16 <= last && tile * 16 + 16 <= p.room;
    if constexpr (kStore) {
      if (!held) continue;
      rb::Pack<T, 8> a[kTurns], b[kTurns];
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int64_t row = tile * 16 + threadIdx.x / LPR + i * kGroups, tok = tok0 + (row - start);
        a[i] = b[i] = rb::Pack<T, 8>{};
        if (row >= start && row < last && row < p.room) {
          a[i] = *reinterpret_cast<const rb::Pack<T, 8>*>(reinterpret_cast<const T*>(p.k) + tok * p.kt + head * p.kh + sub * 8);
          b[i] = *reinterpret_cast<const rb::Pack<T, 8>*>(reinterpret_cast<const T*>(p.v) + tok * p.vt + head * p.vh + sub * 8);
        }
      }
      uint32_t* to = whole ? tile_words : at;
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int r = threadIdx.x / LPR + i * kGroups;
        const int64_t row = tile * 16 + r;
        float x[8], lo, hi;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = rb::to_f(a[i].v[e]);
        q4::extremes<4>(x, lo, hi);
        const uint32_t kg = q4::group_word<T>(lo, hi), kw = q4::pack8<q4::kKey>(x, q4::scale_of<T>(kg), lo);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = rb::to_f(b[i].v[e]);
        q4::extremes<8>(x, lo, hi);
        const uint32_t vg = q4::group_word<T>(lo, hi), vw = q4::pack8<q4::kValue>(x, q4::scale_of<T>(vg), lo);
        if (row >= start && row < last && row < p.room) {
          uint16_t* halves = reinterpret_cast<uint16_t*>(to + Tl::kValues) + q4::half_place(sub, r);
          to[r * Tl::W + q4::word_place<Tl::J>(sub)] = kw;
          halves[0] = (uint16_t)vw;
          halves[2] = (uint16_t)(vw >> 16);
          if (sub % 4 == 0) to[Tl::kKeyScales + r * Tl::J + sub / 4] = kg;
          if (sub % 8 == 0) to[Tl::kValueScales + r * Tl::H + sub / 8] = vg;
        }
      }
      if (whole) {
        __syncthreads();
        for (int i = threadIdx.x; i < Tl::kWords / 4; i += kThreads) reinterpret_cast<uint4*>(at)[i] = reinterpret_cast<const uint4*>(tile_words)[i];
        __syncthreads();
      }
    } else {
      if (held)
        for (int i = threadIdx.x; i < Tl::kWords / 4; i += kThreads) reinterpret_cast<uint4*>(tile_words)[i] = reinterpret_cast<const uint4*>(at)[i];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int r = threadIdx.x / LPR + i * kGroups;
        const int64_t row = tile * 16 + r, tok = tok0 + (row - start);
        if (row < start || row >= last) continue;
        rb::Pack<T, 8> a{}, b{};
        if (held && row < p.room) {
          float x[8];
          const uint16_t* halves = reinterpret_cast<const uint16_t*>(tile_words + Tl::kValues) + q4::half_place(sub, r);
          const uint32_t kg = tile_words[Tl::kKeyScales + r * Tl::J + sub / 4], vg = tile_words[Tl::kValueScales + r * Tl::H + sub / 8];
          q4::unpack8<q4::kKey>(tile_words[r * Tl::W + q4::word_place<Tl::J>(sub)], q4::scale_of<T>(kg), q4::low_of<T>(kg), x);
#pragma unroll
          for (int e = 0; e < 8; ++e) a.v[e] = rb::from_f<T>(x[e]);
          q4::unpack8<q4::kValue>(halves[0] | (uint32_t)halves[2] << 16, q4::scale_of<T>(vg), q4::low_of<T>(vg), x);
#pragma unroll
          for (int e = 0; e < 8; ++e) b.v[e] = rb::from_f<T>(x[e]);
        }
        *reinterpret_cast<rb::Pack<T, 8>*>(reinterpret_cast<T*>(p.k) + tok * p.kt + head * p.kh + sub * 8) = a;
        *reinterpret_cast<rb::Pack<T, 8>*>(reinterpret_cast<T*>(p.v) + tok * p.vt + head * p.vh + sub * 8) = b;
      }
      __syncthreads();
    }
  }
}

template <typename T, int D> int launch(const CacheParams& p, int store, int blocks, cudaStream_t s) {
  const dim3 grid(p.n, p.nkv, blocks);
  return (store ? rb::launch_pdl(cache_rows_kernel<T, D, true>, grid, dim3(kThreads), 0, s, p)
                : rb::launch_pdl(cache_rows_kernel<T, D, false>, grid, dim3(kThreads), 0, s, p)) == cudaSuccess ? 0 : -3;
}

}  // namespace

// `longest`: about the length of the longest sequence (how many blocks a sequence gets; any value is right).  dt: 1 bf16, 2 fp16.
extern "C" int rb_int4_cache_rows(void* k, void* v, int64_t kt, int64_t kh, int64_t vt, int64_t vh, void* cache, const int* cu, const int* slots,
                                  const int* start, int n, int nkv, int hd, int n_slots, int room, int T, int longest, int store, int dt, cudaStream_t s) {
  if (n == 0 || nkv == 0 || T == 0) return 0;
  const CacheParams p{k, v, kt, kh, vt, vh, reinterpret_cast<uint32_t*>(cache), cu, slots, start, n, nkv, n_slots, room, (room + 15) / 16, T};
  const int blocks = (int)std::min<int64_t>((std::max<int64_t>(longest, 1) + 15) / 16 + (start != nullptr), 65535);
  if (dt == 1 && hd == 128) return launch<__nv_bfloat16, 128>(p, store, blocks, s);
  if (dt == 1 && hd == 64) return launch<__nv_bfloat16, 64>(p, store, blocks, s);
  if (dt == 2 && hd == 128) return launch<__half, 128>(p, store, blocks, s);
  if (dt == 2 && hd == 64) return launch<__half, 64>(p, store, blocks, s);
  return -2;
}
