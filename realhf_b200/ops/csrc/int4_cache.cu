// Keys and values of packed sequences into a 4-bit cache, and back (layout and rule: int4.cuh).
//
// A warp has a tile of 16 rows of one head, so nothing waits for other warps: a row by 8 or 16 lanes, 16 bytes a lane of the 16-bit side, four turns' rows read ahead.  The 4-bit side
// is put together in the warp's part of shared memory and copied whole, 16 bytes a lane; where a sequence begins or ends inside a tile, the words of its rows alone are written.
//
// Memory bounds reading back, memory and issue slots storing: keys and values of 128 x 128 tokens of 32 x 128 channels (348 MB both ways, 53 us at the copy's rate) are stored in 65 us
// (5.4 TB/s; 14.8 instructions a number took 75, 27 with one number at a time and a division each took 124) and read back in 58 (6.0).  Calls of a few tokens are a chain of
// latencies, 3.6 and 1.9 us.
#include "int4.cuh"

#include <algorithm>

namespace {

constexpr int kWarps = 4;

struct CacheParams {
  void *k, *v;                      // [T, nkv, D], element (t, h, c) at t * ts + h * hs + c
  int64_t kt, kh, vt, vh;
  uint32_t* cache;                  // [slots, nkv, tiles, Tile<D>::kWords]
  const int *cu, *slots, *start;    // [n + 1], [n] or null (sequence i: slot i), [n] or null (from row 0)
  int n, nkv, n_slots, room, tiles, T;
  uint32_t magic;                   // q4::kWholeMagic
};

template <typename T, int D, bool kStore>
__global__ void __launch_bounds__(kWarps * 32, 8) cache_rows_kernel(CacheParams p) {
  using Tl = q4::Tile<D>;
  constexpr int LPR = D / 8, kPerTurn = 32 / LPR, kTurns = 16 / kPerTurn, kAhead = 4;   // lanes of a row; rows at once; turns of a tile; turns whose rows are read at once
  __shared__ __align__(16) uint32_t words[kWarps][Tl::kWords];
  rb::pdl_trigger();
  rb::pdl_wait();
  const int seq = blockIdx.x, head = blockIdx.y, lane = threadIdx.x & 31, sub = lane % LPR, mine = lane / LPR;
  const int worker = blockIdx.z * kWarps + threadIdx.x / 32, workers = gridDim.z * kWarps;
  uint32_t* const held_words = words[threadIdx.x / 32];
  const int tok0 = min(max(p.cu[seq], 0), p.T), tok1 = min(max(p.cu[seq + 1], tok0), p.T);
  const int slot = p.slots ? p.slots[seq] : seq;
  const int64_t start = p.start ? p.start[seq] : 0;
  const bool there = slot >= 0 && slot < p.n_slots;
  if (kStore && !there) return;
  T* const k = reinterpret_cast<T*>(p.k) + head * p.kh + sub * 8;
  T* const v = reinterpret_cast<T*>(p.v) + head * p.vh + sub * 8;
  if constexpr (!kStore) {                          // tokens before the first sequence and behind the last belong to none
    const int lo = seq == p.n - 1 ? tok1 : 0, hi = seq == p.n - 1 ? p.T : 0, front = seq == 0 ? tok0 : 0;
    for (int i = worker * kPerTurn + mine; i < front + (hi - lo); i += workers * kPerTurn) {
      const int64_t tok = i < front ? i : lo + (i - front);
      *reinterpret_cast<uint4*>(k + tok * p.kt) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(v + tok * p.vt) = make_uint4(0, 0, 0, 0);
    }
  }
  const int64_t first = (start < 0 ? start - 15 : start) / 16, last = start + (tok1 - tok0);   // tiles first .. ; rows below `last`
  for (int64_t tile = first + worker; tile * 16 < last; tile += workers) {
    const bool held = there && tile >= 0 && tile < p.tiles;
    uint4* const at = reinterpret_cast<uint4*>(p.cache + (((int64_t)slot * p.nkv + head) * p.tiles + tile) * Tl::kWords);
    // the tile's rows [r0, r1) are the sequence's, [r0, r2) of them in the cache
    const int r0 = (int)max(start - tile * 16, (int64_t)0), r1 = (int)min(last - tile * 16, (int64_t)16);
    const int r2 = held ? (int)min((int64_t)r1, p.room - tile * 16) : 0;
    const int64_t tok = tok0 + (tile * 16 - start) + mine;                                     // that of the lane's first row (it may lie before the sequence)
    T* const kr = k + tok * p.kt;
    T* const vr = v + tok * p.vt;
    if constexpr (kStore) {
      if (r2 <= r0) continue;
      const auto code = [&](auto whole) {            // (a whole tile asks nothing of its rows)
#pragma unroll 1
        for (int t0 = 0; t0 < kTurns; t0 += kAhead) {
          if (!whole.value && ((t0 + kAhead) * kPerTurn <= r0 || t0 * kPerTurn >= r2)) continue;
          uint4 a[kAhead], b[kAhead];
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            const int r = (t0 + i) * kPerTurn;
            if (!whole.value) a[i] = b[i] = make_uint4(0, 0, 0, 0);
            if (whole.value || (r + mine >= r0 && r + mine < r2)) {
              a[i] = *reinterpret_cast<const uint4*>(kr + r * p.kt);
              b[i] = *reinterpret_cast<const uint4*>(vr + r * p.vt);
            }
          }
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            const int r = (t0 + i) * kPerTurn + mine;
            float lo, hi;
            q4::extremes<T, 4>(a[i], lo, hi);
            const q4::Coded key = q4::code8<T, q4::kKey>(a[i], lo, hi);
            q4::extremes<T, 8>(b[i], lo, hi);
            const q4::Coded value = q4::code8<T, q4::kValue>(b[i], lo, hi);
            uint16_t* halves = reinterpret_cast<uint16_t*>(held_words + Tl::kValues) + q4::half_place(sub, r);
            held_words[r * Tl::W + q4::word_place<Tl::J>(sub)] = key.word;
            halves[0] = (uint16_t)value.word;
            halves[2] = (uint16_t)(value.word >> 16);
            if (sub % 4 == 0) held_words[Tl::kKeyScales + r * Tl::J + sub / 4] = key.group;
            if (sub % 8 == 0) held_words[Tl::kValueScales + r * Tl::H + sub / 8] = value.group;
          }
        }
      };
      if (r2 - r0 == 16) code(std::true_type{});
      else code(std::false_type{});
      __syncwarp();
      if (r2 - r0 == 16) {
#pragma unroll
        for (int i = 0; i < RB_CEIL_DIV(Tl::kWords / 4, 32); ++i)
          if (i * 32 + lane < Tl::kWords / 4) at[i * 32 + lane] = reinterpret_cast<const uint4*>(held_words)[i * 32 + lane];
      } else {                                       // the words of rows r0 .. alone
        uint32_t* const to = reinterpret_cast<uint32_t*>(at);
        const int n = r2 - r0;
        for (int i = r0 * Tl::W + lane; i < r2 * Tl::W; i += 32) to[i] = held_words[i];
        for (int i = Tl::kKeyScales + r0 * Tl::J + lane; i < Tl::kKeyScales + r2 * Tl::J; i += 32) to[i] = held_words[i];
        for (int i = Tl::kValueScales + r0 * Tl::H + lane; i < Tl::kValueScales + r2 * Tl::H; i += 32) to[i] = held_words[i];
        for (int i = lane; i < n * Tl::W * 2; i += 32) {
          const int word = i / 2 % Tl::W, r = r0 + i / (2 * Tl::W), half = 2 * Tl::kValues + q4::half_place(word, r) + 2 * (i & 1);
          reinterpret_cast<uint16_t*>(to)[half] = reinterpret_cast<const uint16_t*>(held_words)[half];
        }
      }
      __syncwarp();
    } else {
      if (r2 > r0) {
#pragma unroll
        for (int i = 0; i < RB_CEIL_DIV(Tl::kWords / 4, 32); ++i)
          if (i * 32 + lane < Tl::kWords / 4) reinterpret_cast<uint4*>(held_words)[i * 32 + lane] = at[i * 32 + lane];
      }
      __syncwarp();
#pragma unroll 2
      for (int t = 0; t < kTurns; ++t) {
        const int r = t * kPerTurn + mine;
        if (r < r0 || r >= r1) continue;
        uint4 a = make_uint4(0, 0, 0, 0), b = a;
        if (r < r2) {
          const uint16_t* halves = reinterpret_cast<const uint16_t*>(held_words + Tl::kValues) + q4::half_place(sub, r);
          a = q4::unpack8<T, q4::kKey>(held_words[r * Tl::W + q4::word_place<Tl::J>(sub)], held_words[Tl::kKeyScales + r * Tl::J + sub / 4], p.magic);
          b = q4::unpack8<T, q4::kValue>(halves[0] | (uint32_t)halves[2] << 16, held_words[Tl::kValueScales + r * Tl::H + sub / 8], p.magic);
        }
        *reinterpret_cast<uint4*>(kr + t * kPerTurn * p.kt) = a;
        *reinterpret_cast<uint4*>(vr + t * kPerTurn * p.vt) = b;
      }
      __syncwarp();
    }
  }
}

template <typename T, int D> int launch(const CacheParams& p, int store, int blocks, cudaStream_t s) {
  const dim3 grid(p.n, p.nkv, blocks);
  return (store ? rb::launch_pdl(cache_rows_kernel<T, D, true>, grid, dim3(kWarps * 32), 0, s, p)
                : rb::launch_pdl(cache_rows_kernel<T, D, false>, grid, dim3(kWarps * 32), 0, s, p)) == cudaSuccess ? 0 : -3;
}

}  // namespace

// `longest`: about the length of the longest sequence (how many blocks a sequence gets; any value is right).  dt: 1 bf16, 2 fp16.
extern "C" int rb_int4_cache_rows(void* k, void* v, int64_t kt, int64_t kh, int64_t vt, int64_t vh, void* cache, const int* cu, const int* slots,
                                  const int* start, int n, int nkv, int hd, int n_slots, int room, int T, int longest, int store, int dt, cudaStream_t s) {
  if (n == 0 || nkv == 0 || T == 0) return 0;
  const CacheParams p{k, v, kt, kh, vt, vh, reinterpret_cast<uint32_t*>(cache), cu, slots, start, n, nkv, n_slots, room, (room + 15) / 16, T, q4::kWholeMagic};
  const int64_t tiles = (std::max<int64_t>(longest, 1) + 15) / 16 + (start != nullptr);
  const int blocks = (int)std::min<int64_t>((tiles + kWarps - 1) / kWarps, 65535);
  if (dt == 1 && hd == 128) return launch<__nv_bfloat16, 128>(p, store, blocks, s);
  if (dt == 1 && hd == 64) return launch<__nv_bfloat16, 64>(p, store, blocks, s);
  if (dt == 2 && hd == 128) return launch<__half, 128>(p, store, blocks, s);
  if (dt == 2 && hd == 64) return launch<__half, 64>(p, store, blocks, s);
  return -2;
}
