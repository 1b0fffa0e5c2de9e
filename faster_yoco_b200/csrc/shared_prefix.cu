// Decode attention of a batch whose rows share long prefixes that are stored, and read, once (sm_100a, tcgen05).
//
// Query i of row b sees the prefix keys of its group and its row's own keys up to its position:
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = scale q . k_j
// The sum splits over the keys: each piece gives (m, l = sum e^(s - m), O = sum e^(s - m) v) and pieces join by weights
// e^(m - max m). All queries of a group against one key / value head (rows x queries x heads of the GQA group) are the
// rows of ONE matrix product over the prefix, so its keys and values are read once for all of them; the own keys of each
// row are a second, smaller product.
//
// Two kernels. spa_kernel, one persistent CTA an SM, walks 128-key tiles; spa_join_kernel joins the pieces. The tiles of
// all (group, head, 128-row block) are one line that is cut into equal ranges, so every SM has the same number of tiles
// whatever the number of heads, and a piece is the part of one block's tiles that falls into one range.
//
// Lengths are read on the device, so ranges are cut from the stored sizes and tiles behind a length are skipped: the SMs
// share evenly what is stored, not what is in use. 32 rows on 4,096 keys take 26 us from a buffer of 4,096 and 37 from one
// of 32,768; 1,000 keys 21 and 33; 16,384 keys 37 and 40.
//
// Scores, softmax statistics, sums and pieces are in fp32. The weights are rounded to the inputs' type for the product
// with the values, as the tensor cores take both operands in one type: half a step of that type for each weight, on top of
// the half step of the result. Against 64 bits a result errs by 2.2e-3 of its norm in bf16 and 2.8e-4 in fp16, where fp32
// weights would give 1.7e-3 and 2.1e-4.
//
// Inside a CTA two streams of tiles run side by side, each with its own query block, scores S and output O in tensor
// memory; one stream's softmax overlaps the other's products:
//   warp 0      loads K / V tiles by TMA, in the order in which they are multiplied, into one ring of slots
//   warp 1      issues S = Q K^T and O += P V (P lies over the first columns of S)
//   warps 2, 3  copy the query block of the next piece of stream 0 / 1 into shared memory (rows of any stride)
//   warps 4-7, 8-11   softmax of stream 0 / 1, a thread a query row: running maximum (O is rescaled only when it grows
//               by more than 2^8), exponentials, row sums, P back to tensor memory; at the end of a piece O, m, l to the
//               workspace
// Work comes in three classes: (0) prefix blocks in pairs, both streams on the same K / V tile (compute bound: halves
// the shared memory fills); (1) the odd last prefix block, each stream with tiles of its own; (2) own keys.
//
// Measured (B200, both kernels, bf16, 24 / 8 heads of 128): 32 rows on 16,384 shared keys with up to 256 of their own
// 37 us (2.5 TB/s of what has to be read; the floor by bytes is 14), 128 rows on 32,768 + 512 137 to 141 us (370 to 380
// TFLOP/s; floor 52), 20 x 24 queries on 2,000 + 24 40 us. What bounds it is neither memory nor the tensor cores (15 to
// 19 % busy) but the chain of a tile: about 2,000 cycles of softmax (exponentials 1,024 at the rate of the SFUs, the rest
// latency of warps that run alone) and 1,500 of products and hand-over, 4,800 a pair of tiles with two streams. Tried
// without gain: two threads a row, four threads a row by copies of short blocks, an issuing warp for each stream, one
// pass over S, turns at the exponentials, rows of 64 or 128 columns in registers (longer code: slower), launching the join
// ahead.
#include <ATen/ATen.h>
#include <c10/util/Optional.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cmath>

#include "common/host.h"
#include "common/ptx.cuh"

namespace fyb {
namespace {

constexpr int kT = 128;                 // tile: keys, and query rows
constexpr int kOwnBox = 32;             // key rows of one TMA box of own keys: what their last tile is rounded up to
constexpr int kAtom = kT * 128;         // 128 rows of a 128-byte swizzle atom
constexpr int kSpaThreads = 384;
constexpr int kJoinCols = 2;            // warps of a joining block that share out the columns
constexpr int kPieceTiles = 1 << 18;    // largest piece: 33 million keys against one block, a second
constexpr float kRescaleLog2 = 8.0f;

struct View {                           // [rows, keys, heads, D], last dim contiguous
  const void* p;
  int64_t s0, s1, s2;
};

struct Cuts {
  int units, len, rem;
};

struct PrefixParams {
  View q;
  int B, Lq, Hq, Hk, G, P, S;
  int rep, rows_p, rows_o;              // heads of a GQA group; query rows of (group, head), of (row, head)
  int pairs, odd, own_blocks;           // 128-row blocks: pairs and 0 / 1 more for the prefix, blocks of own keys
  int tiles_p, tiles_o;                 // stored tiles
  Cuts cuts[3];                         // of each class's tiles
  int shift;                            // first stream that takes a range of class 2
  int ctas;
  const void* lengths;                  // per row (int32 or int64), or null: S
  const void* prefix_lengths;
  int lengths_64, prefix_lengths_64;
  float scale_log2;
  void* o;                              // [B, Lq, Hq, D] contiguous
  float* part[3];                       // pieces: [slot][D / 4][rows of the class][4]
  float2* stat[3];                      // (m in log2 units, l) of each row
  int part_rows[3];
  int* status;
};

__device__ __forceinline__ int length_of(const void* p, int wide, int i, int most) {
  if (p == nullptr) return most;
  const int64_t n = wide ? reinterpret_cast<const int64_t*>(p)[i] : reinterpret_cast<const int*>(p)[i];
  return static_cast<int>(n < 0 ? 0 : (n > most ? most : n));
}

// a value that is the same in all lanes, as the compiler sees it
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ int uniform(bool x) { return __shfl_sync(0xffffffffu, static_cast<int>(x), 0); }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// A mean of fp16 values lies within them. Weights rounded for the product (2^-11 of each, and the sums' 2^-19) can lift
// one at the end of the range past it, where it would round to infinity; infinities and NaN stay.
template <typename T>
__device__ __forceinline__ float within_range(float x) {
  constexpr float kMost = 65504.0f;
  if (std::is_same<T, __half>::value && fabsf(x) < kMost * (1.0f + 0x1p-10f)) return fminf(fmaxf(x, -kMost), kMost);
  return x;
}

// instruction descriptor of kind::f16 with fp32 accumulation; the format bits are 1 for bf16 and 0 for fp16
template <typename T>
__device__ __forceinline__ constexpr uint32_t idesc_of(int N, bool b_mn) {
  const uint32_t d = idesc_bf16(128, N, false, b_mn);
  return sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value ? d & ~((7u << 7) | (7u << 10)) : d;
}

// A class's tiles in `units` ranges of len tiles, the first `rem` of them one longer; units <= tiles, so none is empty.
__host__ __device__ __forceinline__ int range_begin(const Cuts& c, int w) { return w * c.len + min(w, c.rem); }
__device__ __forceinline__ int range_of(const Cuts& c, int tile) {
  const int big = c.rem * (c.len + 1);
  return tile < big ? tile / (c.len + 1) : c.rem + (tile - big) / c.len;
}

// The pieces of one stream in order; every role walks its own copy.
struct Walk {
  int cls = -1;
  int pos = 0, end = 0;
  int seg = 0, t = 0, t1 = 0;     // current piece: tiles t .. t1 of block seg
  int row = 0, hk = 0, blk = 0;   // group (classes 0, 1) or batch row (2), key / value head, 128-row block
  int len = 0;                    // keys in use
  int range = 0;

  __device__ __forceinline__ bool next_piece(const PrefixParams& p, int cta, int stream) {
    for (;;) {
      while (pos >= end) {
        if (++cls > 2) return false;
        // class 0: a range a CTA; else a range a stream, first all CTAs' first streams, so that few ranges spread
        // over the machine; class 2 starts behind the streams that class 1 gave work to
        range = cls == 0 ? cta : stream * p.ctas + cta;
        if (cls == 2) range = range >= p.shift ? range - p.shift : range - p.shift + 2 * p.ctas;
        if (range < p.cuts[cls].units) {
          pos = range_begin(p.cuts[cls], range);
          end = range_begin(p.cuts[cls], range + 1);
        }
      }
      const int tiles = cls == 2 ? p.tiles_o : p.tiles_p;
      seg = pos / tiles;
      t = pos - seg * tiles;
      const int take = min(tiles - t, end - pos);
      pos += take;
      const int per = cls == 0 ? p.pairs : (cls == 1 ? 1 : p.own_blocks);
      const int x = seg / per;
      hk = x % p.Hk;
      row = x / p.Hk;
      blk = cls == 0 ? 2 * (seg % per) + stream : (cls == 1 ? 2 * p.pairs : seg % per);
      len = cls == 2 ? length_of(p.lengths, p.lengths_64, row, p.S)
                     : length_of(p.prefix_lengths, p.prefix_lengths_64, row, p.P);
      t1 = min(t + take, (len + kT - 1) / kT);
      if (t < t1) return true;
    }
  }
  __device__ __forceinline__ int rows(const PrefixParams& p) const {
    return min(kT, (cls == 2 ? p.rows_o : p.rows_p) - blk * kT);
  }
  // batch row, query and query head of row r of the block
  __device__ __forceinline__ void locate(const PrefixParams& p, int r, int& b, int& i, int& h) const {
    const int flat = blk * kT + r, tok = flat / p.rep;
    h = hk * p.rep + flat - tok * p.rep;
    const int bi = cls == 2 ? 0 : tok / p.Lq;
    i = tok - bi * p.Lq;
    b = cls == 2 ? row : row * (p.B / p.G) + bi;
  }
};

template <typename V>
__device__ __forceinline__ void exchange(V& a, V& b) {
  V c = a;
  a = b;
  b = c;
}

// The tiles of a CTA in the order in which they are loaded and multiplied: the two streams in turn, each with a role's
// state. The streams change places rather than being indexed, which keeps them in registers.
template <typename State>
struct Steps {
  Walk w, w_other;
  State s, s_other;                // of the stream whose turn it is, of the other one
  bool live, live_other;
  int turn = 0;                    // stream of the next step

  __device__ __forceinline__ void start(const PrefixParams& p, int cta) {
    live = w.next_piece(p, cta, 0);
    live_other = w_other.next_piece(p, cta, 1);
    if (!live && live_other) swap();
  }
  __device__ __forceinline__ void swap() {
    exchange(w, w_other);
    exchange(s, s_other);
    exchange(live, live_other);
    turn ^= 1;
  }
  // after a step: the stream's next tile, and the other stream's turn if it has one
  __device__ __forceinline__ void advance(const PrefixParams& p, int cta) {
    if (++w.t >= w.t1) live = w.next_piece(p, cta, turn);
    if (live_other) swap();
  }
  // in class 0 stream 1 multiplies by the tile that stream 0 had loaded
  __device__ __forceinline__ bool follows() const { return w.cls == 0 && turn == 1; }
};
struct Stateless {};

// Slots of the K / V ring: as many as fit (160 of 227 KB with two query blocks of 32 KB at D = 128). A tile is read about
// 1.6 us after its slot came free, in which the SM should have received 70 KB: two slots a K and a V of their own left
// the ring waiting (84 us for 32 rows on a 16k prefix).
template <int D>
constexpr int kSlots = D == 128 ? 5 : 8;

struct SpaBars {
  uint64_t full[8], empty[8];
  uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2];   // by stream
};

template <int D>
constexpr int spa_smem() {
  return (2 + kSlots<D>) * kT * D * 2 + 256 + 1024;
}

// position in the ring
template <int N>
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void step() {
    if (++slot == N) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kSpaThreads, 1)
    spa_kernel(const __grid_constant__ CUtensorMap tm_pk, const __grid_constant__ CUtensorMap tm_pv,
               const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
               const __grid_constant__ PrefixParams p) {
  constexpr int kTile = kT * D * 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                       // one block a stream
  uint8_t* sKV = sQ + 2 * kTile;            // ring
  SpaBars* bars = reinterpret_cast<SpaBars*>(sKV + kSlots<D> * kTile);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = blockIdx.x;
  if (threadIdx.x < sizeof(SpaBars) / 8) {   // a barrier a thread, each initialised once: p_full counts the four warps
    uint64_t* bar = reinterpret_cast<uint64_t*>(bars) + threadIdx.x;
    mbar_init(bar, bar == &bars->p_full[0] || bar == &bars->p_full[1] ? 4 : 1);
    fence_mbar_init();
  }
  if (threadIdx.x == 0) *abort_flag = 0;
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;         // S of stream s (P over its first columns) @ 128 s, O @ 256 + 128 s

  // a wait of a whole warp, with one outcome for all lanes (they meet again at warp-wide instructions)
  auto wait = [&](uint64_t* bar, uint32_t ph, int site) -> bool {
    return __all_sync(0xffffffffu, mbar_wait_short(bar, ph, abort_flag, p.status, site));
  };
  if (warp == 0) {
    // ------------------------------------------------------------------------------------------------ K / V loads
    // the whole warp walks, one lane issues: the operands of TMA and of products live in uniform registers
    struct Tile {
      bool pending = false;                  // the V tile of the stream's last step is still to be loaded
      int own = 0, row = 0, hk = 0, key = 0, rows = 0;
    };
    Steps<Tile> st;
    st.start(p, cta);
    Ring<kSlots<D>> ring;
    int n = 0;
    auto load = [&](const Tile& x, const CUtensorMap* prefix, const CUtensorMap* own) -> bool {
      const int slot = uniform(ring.slot), key = uniform(x.key), hk = uniform(x.hk), row = uniform(x.row);
      const bool is_own = uniform(x.own) != 0;
      uint64_t* bar = &bars->full[slot];
      if (!wait(&bars->empty[slot], ring.phase ^ 1u, 700)) return false;
      const CUtensorMap* m = is_own ? own : prefix;
      const int box = is_own ? kOwnBox : kT;
      const int boxes = uniform((x.rows + box - 1) / box);
      if (elect_one()) {
        uint8_t* dst = sKV + slot * kTile;
        mbar_arrive_expect_tx(bar, boxes * box * D * 2);
        for (int j = 0; j < boxes; ++j)
#pragma unroll
          for (int a = 0; a < D / 64; ++a)
            tma_load_4d(dst + a * kAtom + j * box * 128, m, bar, a * 64, hk, key + j * box, row);
      }
      __syncwarp();
      ring.step();
      ++n;
      return true;
    };
    auto load_v = [&](Tile& x) -> bool {
      if (!x.pending) return true;
      x.pending = false;
      return load(x, &tm_pv, &tm_v);
    };
    bool ok = true;
    for (; st.live; st.advance(p, cta)) {
      if (!(ok = load_v(st.s) && (st.live_other || load_v(st.s_other)))) break;
      if (st.follows()) continue;
      const Walk& x = st.w;
      st.s = Tile{true, x.cls == 2, x.row, x.hk, x.t * kT, min(kT, x.len - x.t * kT)};
      if (!(ok = load(st.s, &tm_pk, &tm_k))) break;
    }
    if (ok) ok = load_v(st.s_other) && load_v(st.s);
    // before the CTA ends its loads have landed, and without a timeout have been read
    const int left = min(n, kSlots<D>);
    for (int pass = 0; pass < 2; ++pass) {
      Ring<kSlots<D>> r = ring;
      for (int i = 0; i < left; ++i) {       // backwards: the last load is one position before `ring`
        if (r.slot == 0) {
          r.slot = kSlots<D>;
          r.phase ^= 1u;
        }
        --r.slot;
        if (pass == 0)
          mbar_wait_short(&bars->full[r.slot], r.phase, nullptr, p.status, 702);
        else if (!*abort_flag)
          mbar_wait_short(&bars->empty[r.slot], r.phase, abort_flag, p.status, 703);
      }
    }
  } else if (warp == 1) {
    // --------------------------------------------------------------------------------------------- matrix products
    struct Product {
      bool pending = false, first = true;    // P V of the stream's last tile is still to be issued; a piece starts
      bool opens = false, last = false;      // of that product: first / last of its piece
      bool frees = false, follows = false;   // last / second reader of its V tile
      int nv = 0;                            // keys of that tile
      uint32_t pph = 0, qph = 0;
    };
    Steps<Product> st;
    st.start(p, cta);
    Ring<kSlots<D>> ring;
    int k_slot = 0, v_slot = 0;              // of the last K / V tile met, for the stream that follows
    int freed = -1;                          // slot of a V tile whose products have been issued
    bool ok = true;
    // descriptors: a tile's own bits plus its address and the K step's offset, both in units of 16 bytes
    const uint64_t desc_km = sw128_desc(0, 16, 1024), desc_mn = sw128_desc(0, kAtom, 1024);
    const uint32_t q16 = uniform(smem_u32(sQ) >> 4), kv16 = uniform(smem_u32(sKV) >> 4), tm = uniform(tmem);
    auto meet_v = [&](const Product& v) -> bool {
      if (!v.pending || v.follows) return true;
      if (!wait(&bars->full[ring.slot], ring.phase, 711)) return false;
      v_slot = ring.slot;
      ring.step();
      return true;
    };
    auto issue_pv = [&](Product& v, int s) -> bool {
      if (!v.pending) return true;
      v.pending = false;
      if (!wait(&bars->p_full[s], v.pph, 710)) return false;
      v.pph ^= 1u;
      const int steps = (v.nv + 15) / 16;
      if (!v.follows && v.nv < steps * 16) {
        // a weight of zero times what lies behind the last key in use has to be zero (whole rows: no swizzle)
        uint8_t* tile = sKV + v_slot * kTile;
        for (int c = lane; c < (steps * 16 - v.nv) * (D / 8); c += 32) {
          const int r = v.nv + c / (D / 8), ch = c % (D / 8);
          *reinterpret_cast<uint4*>(tile + (ch >> 3) * kAtom + r * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      const int u = uniform(v_slot | s << 4 | (v.opens ? 32 : 0) | (v.last ? 64 : 0) | steps << 8);
      const int vs = u & 15, su = u >> 4 & 1, n16 = u >> 8;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t dv = desc_mn + kv16 + vs * (kTile >> 4);
        const uint32_t tp = tm + 128 * su, to = tm + 256 + 128 * su;
        umma_bf16_ts(to, tp, dv, idesc_of<T>(D, true), (u & 32) ? 0u : 1u);
#pragma unroll
        for (int k = 1; k < kT / 16; ++k)
          if (k < n16) umma_bf16_ts(to, tp + k * 8, dv + k * 128, idesc_of<T>(D, true), 1u);
        if (u & 64) umma_commit(&bars->o_full[su]);
      }
      __syncwarp();
      if (v.frees) freed = vs;
      return true;
    };
    // the slot of the last V tile is handed back after the next scores have been issued, so as not to hold them up
    auto free_v = [&]() {
      if (freed < 0) return;
      const int vs = uniform(freed);
      if (elect_one()) umma_commit(&bars->empty[vs]);
      __syncwarp();
      freed = -1;
    };
    for (; st.live; st.advance(p, cta)) {
      const int s = st.turn;
      const Walk& x = st.w;
      const bool follows = st.follows();
      const int nv = min(kT, x.len - x.t * kT);
      const bool last = x.t + 1 >= x.t1, frees = x.cls != 0 || follows;
      // what was loaded ahead is waited for before the softmax, so that both products go out together; the scores' tile
      // needs no slot that the product before it still holds
      const bool flush = !st.live_other && st.s_other.pending;
      if (!(ok = meet_v(st.s))) break;
      if (flush) {
        // a stream that has ended must not hold its V tile while the other goes on (its product is the younger one)
        if (!(ok = issue_pv(st.s, s))) break;
        free_v();
        if (!(ok = meet_v(st.s_other) && issue_pv(st.s_other, s ^ 1))) break;
      }
      if (!follows) {
        if (!(ok = wait(&bars->full[ring.slot], ring.phase, 712))) break;
        k_slot = ring.slot;
        ring.step();
      }
      if (st.s.first) {
        if (!(ok = wait(&bars->q_full[s], st.s.qph, 713))) break;
        st.s.qph ^= 1u;
      }
      if (!(ok = issue_pv(st.s, s))) break;
      const int u = uniform(k_slot | s << 4 | (frees ? 32 : 0) | (last ? 64 : 0) | (nv + 15) / 16 << 8);
      const int ks = u & 15, su = u >> 4 & 1;
      const uint32_t id = idesc_of<T>(0, false) | static_cast<uint32_t>(u >> 8) << 18;     // N = 16 x count
      tc_fence_after();
      if (elect_one()) {
        const uint64_t dq = desc_km + q16 + su * (kTile >> 4), dk = desc_km + kv16 + ks * (kTile >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int at = (k >> 2) * (kAtom >> 4) + (k & 3) * 2;
          umma_bf16(tm + 128 * su, dq + at, dk + at, id, k > 0 ? 1u : 0u);
        }
        umma_commit(&bars->s_full[su]);
        if (u & 32) umma_commit(&bars->empty[ks]);
        if (u & 64) umma_commit(&bars->q_empty[su]);
      }
      __syncwarp();
      free_v();
      st.s.pending = true;
      st.s.opens = st.s.first;
      st.s.last = last;
      st.s.frees = frees;
      st.s.follows = follows;
      st.s.nv = nv;
      st.s.first = last;
    }
    // the products left over: the stream that did not take the last step holds the older one
    if (ok) ok = meet_v(st.s_other) && issue_pv(st.s_other, st.turn ^ 1);
    free_v();
    if (ok) ok = meet_v(st.s) && issue_pv(st.s, st.turn);
    free_v();
  } else if (warp < 4) {
    // ----------------------------------------------------------------------------------------------- query blocks
    const int s = warp - 2;
    Walk x;
    uint32_t ph = 1;
    bool any = false, ok = true;
    while (ok && x.next_piece(p, cta, s)) {
      if (!(ok = wait(&bars->q_empty[s], ph, 720))) break;
      ph ^= 1u;
      any = true;
      // a lane copies whole rows: 16-byte pieces at consecutive addresses, one address computation a row
      const int rows = x.rows(p);
      for (int r = lane; r < rows; r += 32) {
        int b, i, h;
        x.locate(p, r, b, i, h);
        const T* src = reinterpret_cast<const T*>(p.q.p) + b * p.q.s0 + i * p.q.s1 + h * p.q.s2;
        uint8_t* dst = sQ + s * kTile + r * 128;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) cp_async16(dst + (c >> 3) * kAtom + (((c & 7) ^ (r & 7)) << 4), src + c * 8);
      }
      cp_async_wait_all();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->q_full[s]);
    }
    if (ok && any) wait(&bars->q_empty[s], ph, 721);
  } else {
    // ---------------------------------------------------------------------------------------------------- softmax
    const int s = (warp - 4) >> 2;
    const int quad = warp & 3;
    const int r = quad * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t tS = tmem + 128 * s + lanes, tO = tmem + 256 + 128 * s + lanes;
    // fp16 weights are lifted by 2^7 (at most 2^15 with the lazy maximum), which keeps what lies down to 2^-21 of the
    // largest in its normal range; bf16 has fp32's range
    constexpr float kLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;
    // scores of the keys behind the first n
    auto hide = [](uint32_t (&v)[32], int n) {
      if (__any_sync(0xffffffffu, n < 32)) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j >= n) v[j] = __float_as_uint(-INFINITY);
      }
    };
    Walk x;
    uint32_t s_ph = 0, o_ph = 0;
    bool ok = true;
    while (ok && x.next_piece(p, cta, s)) {
      const int rows = x.rows(p);
      const bool active = quad * 32 < rows;              // this warp has rows
      // keys that this row sees: all in use of a prefix, of its own those up to its position
      int sees = x.len;
      if (x.cls == 2) {
        int b, i, h;
        x.locate(p, min(r, rows - 1), b, i, h);
        sees = min(sees, x.len - p.Lq + i + 1);
      }
      float m_ref = -INFINITY, l = 0.f;
      for (; x.t < x.t1; ++x.t) {
        if (!(ok = wait(&bars->s_full[s], s_ph, 730))) break;
        s_ph ^= 1u;
        if (active) {
          tc_fence_after();
          // S is read twice, 32 columns at a time: a row of 128 in registers spills, and a warp that runs alone is bound
          // by the fetching of its instructions, so the loops are kept short
          const int vis = sees - x.t * kT, nc = (min(kT, x.len - x.t * kT) + 31) / 32;
          float mx = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < nc; ++c) {
            uint32_t v[32];
            tmem_ld32(tS + c * 32, v);
            tmem_ld_wait();
            hide(v, vis - c * 32);
            float m4[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 32; ++j) m4[j & 3] = fmaxf(m4[j & 3], __uint_as_float(v[j]));
            mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          }
          const float m_cand = fmaxf(m_ref, mx * p.scale_log2);
          const bool need = m_cand > m_ref + kRescaleLog2;
          const bool scale_o = need && m_ref != -INFINITY;
          if (__any_sync(0xffffffffu, scale_o)) {
            // the products up to the previous tile are complete: S, which this thread waited for, was issued after them
            const float f = scale_o ? fast_exp2(m_ref - m_cand) : 1.0f;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t w[32];
              tmem_ld32(tO + c, w);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(__uint_as_float(w[j]) * f);
              tmem_st32(tO + c, w);
            }
            if (scale_o) l *= f;
          }
          if (need) m_ref = m_cand;
          const float m = m_ref == -INFINITY ? 0.f : m_ref - kLift;
          __syncwarp();
          const float2 sc = make_float2(p.scale_log2, p.scale_log2), nm = make_float2(-m, -m);
          float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
          for (int c = 0; c < nc; ++c) {
            uint32_t v[32], w[16];
            tmem_ld32(tS + c * 32, v);
            tmem_ld_wait();
            hide(v, vis - c * 32);
#pragma unroll
            for (int j = 0; j < 16; ++j) {        // l sums the weights as they are, P takes them rounded
              const float2 t = fma2(make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), sc, nm);
              const float2 e = make_float2(fast_exp2(t.x), fast_exp2(t.y));
              l2[j & 1] = add2(l2[j & 1], e);
              w[j] = pack2<T>(e.x, e.y);
            }
            tmem_st16(tS + c * 16, w);      // over columns that have been read
          }
          l += (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[s]);
      }
      if (!ok || !(ok = wait(&bars->o_full[s], o_ph, 731))) break;
      o_ph ^= 1u;
      if (active) {
        tc_fence_after();
        const int64_t slot = x.cls == 0 ? 2 * (static_cast<int64_t>(x.range) + x.seg) + s
                                        : static_cast<int64_t>(x.range) + x.seg;
        const int64_t at = slot * p.part_rows[x.cls] + r;
        // four values of all rows side by side: the lanes of a warp, a row each, store whole lines
        float4* dst = reinterpret_cast<float4*>(p.part[x.cls]) + slot * p.part_rows[x.cls] * (D / 4) + r;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t v[32];
          tmem_ld32(tO + c, v);
          tmem_ld_wait();
          if (r < rows) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<uint4*>(dst + (c / 4 + j) * p.part_rows[x.cls]) =
                  make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
          __syncwarp();
        }
        if (r < rows) p.stat[x.cls][at] = make_float2(m_ref - kLift, l);
        tc_fence_before();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the pieces of each output row: o = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i. A block has eight consecutive
// rows of a (group, key / value head) and 1 / Split of their columns. Its warps share them out by columns (kJoinCols) and
// by pieces (Parts); a lane has one row and some columns in fours, so that a load of a warp covers whole 128-byte lines
// and a thread has its loads in flight together; the parts join in shared memory.
template <typename T, int D, int Parts, int Split>
__global__ void __launch_bounds__(kJoinCols * Parts * 32) spa_join_kernel(const __grid_constant__ PrefixParams p) {
  constexpr int F = D / 4 / Split / (4 * kJoinCols);     // float4s of a lane: from c0 on, lane / 8 + 4 (wc + kJoinCols f)
  const int c0 = static_cast<int>(blockIdx.y) * (D / 4 / Split);
  __shared__ float4 sO[Parts - 1][D / 4 / Split][8];
  __shared__ float2 sML[Parts][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wc = warp % kJoinCols, wp = warp / kJoinCols;
  const int per = (p.rows_p + 7) / 8;
  const int gh = blockIdx.x / per, flat = (blockIdx.x - gh * per) * 8 + (lane & 7);
  const bool live = flat < p.rows_p;
  const int hk = gh % p.Hk, g = gh / p.Hk;
  const int tok = flat / p.rep, hr = flat - tok * p.rep;
  const int bi = tok / p.Lq, i = tok - bi * p.Lq, b = g * (p.B / p.G) + bi;

  float M = -INFINITY, L = 0.f;
  float4 o[F];
#pragma unroll
  for (int f = 0; f < F; ++f) o[f] = make_float4(0.f, 0.f, 0.f, 0.f);
  auto piece = [&](const float4* src, const float2* stat, int rows) {
    const float2 ml = *stat;
    float4 t[F];
#pragma unroll
    for (int f = 0; f < F; ++f) t[f] = src[(c0 + (lane >> 3) + 4 * (wc + kJoinCols * f)) * rows];
    const bool any = ml.y != 0.f;            // a NaN score has to reach the result: its piece's sum is NaN
    const float Mn = any ? fmaxf(M, ml.x) : M;
    const float f0 = M == -INFINITY ? 0.f : fast_exp2(M - Mn), w = any ? fast_exp2(ml.x - Mn) : 0.f;
    M = Mn;
    L = L * f0 + w * ml.y;
#pragma unroll
    for (int f = 0; f < F; ++f) {
      if (!any) t[f] = make_float4(0.f, 0.f, 0.f, 0.f);
      o[f] = make_float4(o[f].x * f0 + w * t[f].x, o[f].y * f0 + w * t[f].y, o[f].z * f0 + w * t[f].z,
                         o[f].w * f0 + w * t[f].w);
    }
  };
  // pieces of the prefix: the same for the eight rows, which lie in one 128-row block
  const int used = (length_of(p.prefix_lengths, p.prefix_lengths_64, g, p.P) + kT - 1) / kT;
  if (used > 0) {
    const int blk = flat / kT;
    const bool pair = blk < 2 * p.pairs;
    const Cuts cuts = pair ? p.cuts[0] : p.cuts[1];
    const int rows = pair ? kT : p.part_rows[1], seg = pair ? gh * p.pairs + (blk >> 1) : gh;
    const int first = range_of(cuts, seg * p.tiles_p), n = range_of(cuts, seg * p.tiles_p + used - 1) + 1 - first;
    const float4* part = reinterpret_cast<const float4*>(pair ? p.part[0] : p.part[1]);
    const float2* stat = pair ? p.stat[0] : p.stat[1];
    const int r = live ? flat - blk * kT : 0;
#pragma unroll 4
    for (int k = wp; k < n; k += Parts) {
      const int64_t at = (pair ? 2 * (static_cast<int64_t>(first) + k + seg) + (blk & 1)
                               : static_cast<int64_t>(first) + k + seg) * rows;
      piece(part + at * (D / 4) + r, stat + at + r, rows);
    }
  }
  // pieces of the row's own keys
  const int used2 = live ? (length_of(p.lengths, p.lengths_64, b, p.S) + kT - 1) / kT : 0;
  if (used2 > 0) {
    const int own = i * p.rep + hr, blk = own / kT, rows = p.part_rows[2];
    const int seg = (b * p.Hk + hk) * p.own_blocks + blk;
    const int first = range_of(p.cuts[2], seg * p.tiles_o);
    const int n = range_of(p.cuts[2], seg * p.tiles_o + used2 - 1) + 1 - first;
    for (int k = Parts - 1 - wp; k < n; k += Parts) {
      const int64_t at = (static_cast<int64_t>(first) + k + seg) * rows;
      const int r = own - blk * kT;
      piece(reinterpret_cast<const float4*>(p.part[2]) + at * (D / 4) + r, p.stat[2] + at + r, rows);
    }
  }
  if (wc == 0 && lane < 8) sML[wp][lane] = make_float2(M, L);
  if (wp > 0) {
#pragma unroll
    for (int f = 0; f < F; ++f) sO[wp - 1][(lane >> 3) + 4 * (wc + kJoinCols * f)][lane & 7] = o[f];
  }
  __syncthreads();
  if (wp > 0 || !live) return;
  float top = M, total = 0.f, w[Parts];
#pragma unroll
  for (int q = 1; q < Parts; ++q) top = fmaxf(top, sML[q][lane & 7].x);
#pragma unroll
  for (int q = 0; q < Parts; ++q) {
    const float2 ml = sML[q][lane & 7];
    w[q] = ml.y != 0.f ? fast_exp2(ml.x - top) : 0.f;
    total += w[q] * ml.y;
  }
  const float inv = total != 0.f ? 1.0f / total : 0.f;       // no key seen: zeros; a NaN stays one
  T* out = reinterpret_cast<T*>(p.o) + ((static_cast<int64_t>(b) * p.Lq + i) * p.Hq + hk * p.rep + hr) * D;
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int c4 = (lane >> 3) + 4 * (wc + kJoinCols * f);
    float4 x = make_float4(w[0] * o[f].x, w[0] * o[f].y, w[0] * o[f].z, w[0] * o[f].w);
#pragma unroll
    for (int q = 1; q < Parts; ++q) {
      const float4 t = sO[q - 1][c4][lane & 7];
      x = make_float4(x.x + w[q] * t.x, x.y + w[q] * t.y, x.z + w[q] * t.z, x.w + w[q] * t.w);
    }
    *reinterpret_cast<uint2*>(out + 4 * (c0 + c4)) =
        make_uint2(pack2<T>(within_range<T>(x.x * inv), within_range<T>(x.y * inv)),
                   pack2<T>(within_range<T>(x.z * inv), within_range<T>(x.w * inv)));
  }
}

View view_of(const at::Tensor& t, const at::Tensor& q, const char* name) {
  FYB_SUITS(t.device() == q.device() && t.scalar_type() == q.scalar_type() && t.dim() == 4 &&
                t.size(3) == q.size(3) && t.stride(3) == 1,
            std::string("shared_prefix_attention: ") + name);
  FYB_SUITS(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
            std::string("shared_prefix_attention: 16-byte aligned ") + name);
  for (int d = 0; d < 3; ++d)
    FYB_SUITS(t.size(d) <= 1 || (t.stride(d) > 0 && t.stride(d) % 8 == 0),
              std::string("shared_prefix_attention: strides of ") + name + " must be positive multiples of 8 elements");
  return View{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

// {D, heads, keys, rows} with boxes of 64 x 1 x box_keys x 1; a dimension of one element has no stride to speak of
CUtensorMap tmap_cache(const at::Tensor& t, int box_keys) {
  if (t.numel() == 0) return CUtensorMap{};            // no tile of it is loaded
  CUtensorMap m;
  auto bytes = [&](int d) -> cuuint64_t { return t.size(d) > 1 ? t.stride(d) * 2 : t.size(3) * 2; };
  cuuint64_t dims[4] = {(cuuint64_t)t.size(3), (cuuint64_t)t.size(2), (cuuint64_t)t.size(1), (cuuint64_t)t.size(0)};
  cuuint64_t strides[3] = {bytes(2), bytes(1), bytes(0)};
  cuuint32_t box[4] = {64u, 1u, (cuuint32_t)box_keys, 1u};
  cuuint32_t one[4] = {1u, 1u, 1u, 1u};
  const CUresult r = encode_fn()(
      &m, t.scalar_type() == at::kHalf ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
      t.data_ptr(), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  FYB_CHECK(r == CUDA_SUCCESS,
            "shared_prefix_attention: cuTensorMapEncodeTiled code " + std::to_string(static_cast<int>(r)));
  return m;
}

const void* length_ptr(const c10::optional<at::Tensor>& t, const at::Tensor& q, int64_t n, int& wide) {
  wide = 0;
  if (!t.has_value() || !t->defined()) return nullptr;
  wide = t->scalar_type() == at::kLong;
  FYB_SUITS(t->device() == q.device() && (wide || t->scalar_type() == at::kInt) && t->dim() == 1 && t->size(0) == n &&
                (n <= 1 || t->stride(0) == 1),
            "shared_prefix_attention: lengths");
  return t->data_ptr();
}

template <typename T, int D>
void launch(const CUtensorMap& pk, const CUtensorMap& pv, const CUtensorMap& k, const CUtensorMap& v,
            const PrefixParams& p) {
  // once for each device: the attribute belongs to the one that is current
  static std::atomic<uint64_t> done{0};
  int dev;
  FYB_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || (done.load(std::memory_order_acquire) >> dev & 1u) == 0) {
    FYB_CUDA(cudaFuncSetAttribute(spa_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, spa_smem<D>()));
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
  }
  spa_kernel<T, D><<<p.ctas, kSpaThreads, spa_smem<D>(), cur_stream()>>>(pk, pv, k, v, p);
  check_launch("shared_prefix_attention");
  const int groups = p.G * p.Hk * ((p.rows_p + 7) / 8);
  // pieces of a row, about: ranges that meet a prefix block and those of its own keys
  const int segs = p.G * p.Hk * std::max(p.pairs, 1);
  const int pieces = (p.pairs > 0 ? p.cuts[0].units : p.cuts[1].units) / segs + 2;
  // Few blocks and many pieces: twice the blocks, each with half of the columns, and twice the warps on the pieces (both
  // kernels, us, with and without: 96 blocks of 39 pieces 37.4 and 40.3; 384 blocks of 20 pieces 144.7 and 137.8; 128
  // blocks of 11 pieces 52.2 and 49.9). With few pieces two warps share them.
  if (pieces > 16 && groups < 2 * p.ctas)
    spa_join_kernel<T, D, 8, 2><<<dim3(groups, 2), kJoinCols * 8 * 32, 0, cur_stream()>>>(p);
  else if (pieces > 8)
    spa_join_kernel<T, D, 4, 1><<<groups, kJoinCols * 4 * 32, 0, cur_stream()>>>(p);
  else
    spa_join_kernel<T, D, 2, 1><<<groups, kJoinCols * 2 * 32, 0, cur_stream()>>>(p);
  check_launch("shared_prefix_attention (join)");
}

}  // namespace

at::Tensor shared_prefix_attention(const at::Tensor& q, const at::Tensor& pk, const at::Tensor& pv,
                                   const at::Tensor& k, const at::Tensor& v,
                                   const c10::optional<at::Tensor>& lengths,
                                   const c10::optional<at::Tensor>& prefix_lengths, double scale) {
  FYB_RANGE("fyb::shared_prefix_attention");
  FYB_SUITS(q.is_cuda() && q.dim() == 4 && (q.size(3) == 64 || q.size(3) == 128) &&
                (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf),
            "shared_prefix_attention: bf16 or fp16 q [B, Lq, Hq, 64 or 128] expected");
  // as the kernel holds it: a factor of zero would make NaN of the -inf of hidden keys
  const float scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  FYB_SUITS(std::isnormal(scale_log2) && scale_log2 > 0,
            "shared_prefix_attention: scale must be positive and within fp32");
  const int64_t B = q.size(0), Lq = q.size(1), Hq = q.size(2), D = q.size(3);
  PrefixParams p{};
  p.q = view_of(q, q, "q");
  view_of(pk, q, "prefix_k");
  view_of(pv, q, "prefix_v");
  view_of(k, q, "k");
  view_of(v, q, "v");
  const int64_t G = pk.size(0), P = pk.size(1), Hk = pk.size(2), S = k.size(1);
  FYB_SUITS(pv.sizes() == pk.sizes() && v.sizes() == k.sizes() && k.size(0) == B && k.size(2) == Hk && Hk > 0 && G > 0 &&
                Hq > 0 && Hq % Hk == 0 && B % G == 0,
            "shared_prefix_attention: shape mismatch");
  FYB_SUITS(B * Lq * Hq < (1ll << 31) && P < (1ll << 30) && S < (1ll << 30), "shared_prefix_attention: sizes");
  c10::cuda::CUDAGuard guard(q.device());
  auto o = at::empty({B, Lq, Hq, D}, q.options());
  if (o.numel() == 0) return o;
  p.B = (int)B, p.Lq = (int)Lq, p.Hq = (int)Hq, p.Hk = (int)Hk, p.G = (int)G, p.P = (int)P, p.S = (int)S;
  p.rep = (int)(Hq / Hk);
  p.rows_p = (int)(B / G * Lq * p.rep);
  p.rows_o = (int)(Lq * p.rep);
  const int blocks = (p.rows_p + kT - 1) / kT;
  p.pairs = blocks / 2;
  p.odd = blocks & 1;
  p.own_blocks = (p.rows_o + kT - 1) / kT;
  p.tiles_p = (int)((P + kT - 1) / kT);
  p.tiles_o = (int)((S + kT - 1) / kT);
  const int64_t segs[3] = {G * Hk * p.pairs, G * Hk * p.odd, B * Hk * p.own_blocks};
  int total[3];
  for (int c = 0; c < 3; ++c) {
    const int64_t tiles = segs[c] * (c == 2 ? p.tiles_o : p.tiles_p);
    FYB_SUITS(tiles < (1ll << 31), "shared_prefix_attention: more than 2^31 tiles");
    total[c] = (int)tiles;
  }
  p.ctas = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  for (int c = 0; c < 3; ++c) {
    const int units = std::min(total[c], c == 0 ? p.ctas : 2 * p.ctas);
    p.cuts[c] = units > 0 ? Cuts{units, total[c] / units, total[c] % units} : Cuts{0, 1, 0};
    // the loader of the next query block waits for a whole piece: at up to 4 us a tile well within the limit of a wait
    FYB_SUITS(std::min(p.cuts[c].len + 1, c == 2 ? p.tiles_o : p.tiles_p) <= kPieceTiles,
              "shared_prefix_attention: too many keys for this many queries in one call");
  }
  p.shift = p.cuts[1].units % (2 * p.ctas);
  p.lengths = length_ptr(lengths, q, B, p.lengths_64);
  p.prefix_lengths = length_ptr(prefix_lengths, q, G, p.prefix_lengths_64);
  p.scale_log2 = scale_log2;
  p.o = o.data_ptr();
  p.status = status_ptr();
  // a slot for each (range, block) that can meet: ranges + blocks, as both only move forward
  p.part_rows[0] = kT;
  p.part_rows[1] = p.rows_p - 2 * p.pairs * kT;
  p.part_rows[2] = std::min(p.rows_o, kT);
  int64_t rows[3], all = 0;
  for (int c = 0; c < 3; ++c) {
    const int64_t slots = (p.cuts[c].units + segs[c]) * (c == 0 ? 2 : 1);
    rows[c] = total[c] > 0 ? slots * p.part_rows[c] : 0;
    all += rows[c];
  }
  auto ws = at::empty({std::max<int64_t>(all, 1) * (D + 2)}, q.options().dtype(at::kFloat));
  float* at_ = ws.data_ptr<float>();
  for (int c = 0; c < 3; ++c) {
    p.part[c] = at_;
    at_ += rows[c] * D;
  }
  for (int c = 0; c < 3; ++c) {
    p.stat[c] = reinterpret_cast<float2*>(at_);
    at_ += rows[c] * 2;
  }
  const CUtensorMap mpk = tmap_cache(pk, kT), mpv = tmap_cache(pv, kT);
  const CUtensorMap mk = tmap_cache(k, kOwnBox), mv = tmap_cache(v, kOwnBox);
  if (q.scalar_type() == at::kBFloat16)
    D == 64 ? launch<__nv_bfloat16, 64>(mpk, mpv, mk, mv, p) : launch<__nv_bfloat16, 128>(mpk, mpv, mk, mv, p);
  else
    D == 64 ? launch<__half, 64>(mpk, mpv, mk, mv, p) : launch<__half, 128>(mpk, mpv, mk, mv, p);
  return o;
}

}  // namespace fyb
