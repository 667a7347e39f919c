// cross_attention_sm100.cu - attention of many queries over states of another
// length on the fifth-generation tensor cores.
//
//   S_j = Q K_j^T     tcgen05.mma 128 x 128 x D, accumulator in TMEM
//   P_j = exp2(S_j c - m)   one thread per query row, 16-bit pairs to TMEM
//   O  += P_j V_j     tcgen05.mma 128 x D x 128, A = P from TMEM
//
// with the running maximum and sum of each row (rows, heads and keys as in
// cross_attention.cuh).  One CTA per SM computes two 128-row tiles against the
// same K and V: a K / V tile read from L2 serves 256 rows, and while one tile's
// softmax runs the tensor cores work for the other.  Twelve warps:
//   warp 0      TMA: the Q tiles, then K and V through rings of their own
//   warp 1      MMA issue, in the order P0.V S0 P1.V S1, which sets the two
//               tiles half a turn apart (an issuing warp for each tile let them
//               fall into step: 184 -> 235 us on the case below); allocates TMEM
//   warps 4-7, 8-11   softmax and epilogue of tile 0 and 1; warp w owns TMEM
//               lanes 32 (w % 4) .. + 31, a thread a whole row of S
// TMEM (512 columns): S0 S1 (128 each; P takes the place of its S), O0 O1 (D
// each).  O is rescaled lazily, when a row's maximum has grown by more than
// 2^8.  Every mbarrier wait is bounded.
//
// What bounds it: a 128 x 128 tile takes 1024 clocks of the exponential units
// (16 results per clock and SM) and 8 D clocks of the tensor cores (4 x 128 x
// 128 D flops at 8192 per clock and SM): as many at D = 128, half at 64.
// Neither is what the kernel waits for: at D = 128 both are half busy (ncu:
// 0.51 and 0.46), at 64 the exponential units 0.51.  What is missing is the
// way from S to P and back (waits, two TMEM loads, the maximum), which two
// warps on a scheduler do not hide.  Measured: 20/4 heads of 128, 2 x 1729
// queries, 6001 and 4501 keys 187 us, 992 TFLOP/s, 0.59 of the measured GEMM
// rate (205 - 208 us, 0.54, once the card is at its power limit); 2 x 16 heads
// of 64, 5184 queries, 20736 keys 1.54 - 1.55 ms, 570 TFLOP/s.
//
// Other forms, the last case, measured while the kernel was written: P beside S
// and all 128 scores of a row in registers, so that the next S is made during
// the softmax: 1.36 ms with one item a CTA (212 us for the first case); walking
// several items as well, that form spilled, and with 96 + 32 scores as below it
// took 1.84 ms.  No maximum before the exponentials (made again where a row's P
// would overflow): 1.59 ms.  S read twice in 64-column halves: 1.87 ms.  One or
// two of eight exponentials by polynomial: 1.51 and 1.60 ms.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cstring>

#include "attention_math.cuh"
#include "cross_attention.cuh"
#include "sam3cu_internal.h"
#include "sm100_ptx.cuh"
#include "tma_host.cuh"

namespace s3 {

S3_DEV_ERROR_ACCESSOR(dev_error_cross)

namespace {

constexpr int kQ = 128;        // rows of a tile
constexpr int kKV = 128;       // keys of a tile
constexpr int kThreads = 384;
constexpr float kRescaleLog2 = 8.f;
// One multiply-add takes a score to its exponent, which rounds maximum * factor:
// a row's P get a factor that cancels in O / sum, 2^-12 off 1 at most up to
// here.  It would be 2^4 at 2^27 (past f16's range) and 2^64 at 2^31: past this
// value the maximum is taken off the scores first.  That costs 2 x 5184 queries
// over 20736 keys 1536 -> 1546 us where it does not happen, in this form; taken
// off always 1595, by a branch before the exponentials 1590 - 1617.
constexpr float kFarLog2 = 4096.f;
// f16 P below 2^-14 loses bits: with a maximum of 2^9 there is room for a
// factor 2^6 under 65504.  It cancels in O / sum.
constexpr float kF16Shift = 6.f;

template <int kD>
struct Cfg {
  static constexpr int kRowBytes = kD == 32 ? 64 : 128;  // a swizzled row (half of one for D = 128)
  static constexpr int kHalves = kD == 128 ? 2 : 1;
  static constexpr int kTile = 128 * kD * 2;             // Q, K or V tile
  static constexpr int kStages = kD == 128 ? 2 : kD == 64 ? 4 : 8;  // of K, and of V
  static constexpr int kSmem = 2 * kTile + 2 * kStages * kTile;
  // one CTA per SM: each allocates all of TMEM
  static_assert(kSmem > 116 * 1024 && kSmem < 226 * 1024, "one CTA per SM");
  static constexpr uint32_t kOCol = 256;
  static constexpr int kPitch = kD + 4;                  // floats of a partial row
  static_assert(2 * kQ * kPitch * 4 <= kSmem, "partial rows fit over the rings");
};

struct TcParams {
  CrossParams c;
  int qpt;        // queries of a tile: 128 / group
  int items_x;    // row items of a (batch, key head)
  int n_items;    // items_x * kv_heads * batch
  int tiles;      // 128-row tiles of an item: 1 or 2
  int splits;     // CTAs of the cluster that share an item's keys (then one item a CTA)
  int qmul_b;     // 0: the batch shares its queries
  KvShare kv;
};

// One work item: up to two query tiles of a (batch, key head) and the key
// tiles [j0, j0 + n_kv) that this CTA takes.
struct Item {
  int b, kvh, q0, tiles, len, j0, n_kv;
};
__device__ __forceinline__ Item item_of(const TcParams& prm, int idx, int split) {
  Item it;
  const int bh = idx / prm.items_x;
  it.q0 = (idx - bh * prm.items_x) * prm.tiles * prm.qpt;
  it.tiles = it.q0 + prm.qpt < prm.c.sq ? prm.tiles : 1;  // the second may lie past the last query
  it.b = bh / prm.c.kv_heads;
  it.kvh = bh - it.b * prm.c.kv_heads;
  it.len = cross_len(prm.c, it.b);
  const int all = (it.len + kKV - 1) / kKV;
  it.j0 = static_cast<int>(static_cast<int64_t>(all) * split / prm.splits);
  it.n_kv = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / prm.splits) - it.j0;
  return it;
}

// Walks the (item, key tile) pairs of a CTA; items without keys are passed over.
struct Cursor {
  int idx, j;      // item, key tile of it
  int kt;          // key tiles before it: place in the rings
  int nth, nth_b;  // items before it, and those with a second query tile,
  int kt_b;        //   and their key tiles: phases of the query tiles' barriers
  Item it;
  __device__ __forceinline__ bool more(const TcParams& prm) const { return idx < prm.n_items; }
  __device__ __forceinline__ void find(const TcParams& prm, int step, int split) {
    for (; idx < prm.n_items; idx += step) {
      it = item_of(prm, idx, split);
      if (it.n_kv > 0) break;
    }
  }
  __device__ __forceinline__ void start(const TcParams& prm, int first, int step, int split) {
    idx = first;
    j = kt = nth = nth_b = kt_b = 0;
    find(prm, step, split);
  }
  __device__ __forceinline__ void next(const TcParams& prm, int step, int split) {
    ++kt;
    kt_b += it.tiles > 1;
    if (++j == it.n_kv) {
      j = 0;
      ++nth;
      nth_b += it.tiles > 1;
      idx += step;
      find(prm, step, split);
    }
  }
  __device__ __forceinline__ int items(int t) const { return t ? nth_b : nth; }
  __device__ __forceinline__ int turns(int t) const { return t ? kt_b : kt; }
  // keys of the tile, rounded up to a multiple of 16
  __device__ __forceinline__ int keys() const {
    const int left = it.len - (it.j0 + j) * kKV;
    return left >= kKV ? kKV : ((left + 15) & ~15);
  }
};

// P = exp2(S sl2 + add) of kN keys as 16-bit pairs to TMEM from column tp on,
// added up into l2.
template <bool kBf16, int kN>
__device__ __forceinline__ void exp_store(const float (&sv)[kN], float sl2, float add, uint32_t tp, uint64_t (&l2)[2]) {
  const uint64_t sc2 = f2pack(sl2, sl2), ad2 = f2pack(add, add);
#pragma unroll
  for (int c0 = 0; c0 < kN; c0 += 16) {  // 16 keys -> 8 P columns
    uint32_t pk[8];
#pragma unroll
    for (int c = c0; c < c0 + 16; c += 2) {
      float e0, e1;
      f2unpack(ffma2(f2pack(sv[c], sv[c + 1]), sc2, ad2), e0, e1);
      const float p0 = ex2(e0), p1 = ex2(e1);
      l2[(c >> 1) & 1] = fadd2(l2[(c >> 1) & 1], f2pack(p0, p1));
      pk[(c - c0) / 2] = pack2(p0, p1, kBf16);
    }
    tmem_st_32x32b_x8(tp + c0 / 2, *reinterpret_cast<const uint32_t(*)[8]>(pk));
  }
}

template <bool kBf16, int kD, bool kMask>
__global__ void __launch_bounds__(kThreads, 1)
    cross_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                    const __grid_constant__ CUtensorMap tv, const __grid_constant__ TcParams prm) {
  using Cf = Cfg<kD>;
  constexpr int kStages = Cf::kStages, kTile = Cf::kTile;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t bars[13 + 4 * kStages];
  __shared__ float2 ml[2 * kQ];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag_s;
  // [2] by tile; phases: per item (q, o) or per key tile (s, p)
  uint64_t* q_full = &bars[0];
  uint64_t* q_empty = &bars[2];
  uint64_t* o_full = &bars[4];
  uint64_t* o_empty = &bars[6];
  uint64_t* s_full = &bars[8];
  uint64_t* p_full = &bars[10];
  // [kStages]
  uint64_t* k_full = &bars[12];
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* mma_done = v_empty + kStages;
  volatile int* abort_flag = &abort_flag_s;

  const CrossParams& p = prm.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x % prm.splits;
  const int first = blockIdx.x / prm.splits, step = gridDim.x / prm.splits;

  uint8_t* sQ = smem;
  auto sK = [&](int st) { return smem + 2 * kTile + st * kTile; };
  auto sV = [&](int st) { return smem + 2 * kTile + (kStages + st) * kTile; };
  const bool aligned = (smem_u32(smem) & 1023u) == 0;  // the swizzled layouts need it

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&o_full[t], 1);
      mbar_init(&o_empty[t], 4);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(mma_done, 1);
    abort_flag_s = aligned ? 0 : 1;
    if (!aligned) atomicCAS(&g_dev_error, 0u, static_cast<unsigned>(kErrTmemAlloc));
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  // The copies fill qpt * group of a query tile's 128 rows.  The others become
  // zeros, once: what another kernel left there would have a say in when their
  // warp's rows are rescaled, and with it in how those round.
  for (int i = threadIdx.x; i < 2 * kTile / 16; i += kThreads) {
    const int row = i % (kTile / Cf::kHalves / 16) / (Cf::kRowBytes / 16);
    if (row >= prm.qpt * p.group) *reinterpret_cast<uint4*>(sQ + i * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  auto tS = [&](int t) { return tmem + static_cast<uint32_t>(t * 128); };
  auto tO = [&](int t) { return tmem + Cf::kOCol + static_cast<uint32_t>(t * kD); };

  if (warp == 0 && aligned) {
    // ------------------------------------------------------------ TMA
    if (elect_one()) {
      tma_prefetch_desc(&tq);
      tma_prefetch_desc(&tk);
      tma_prefetch_desc(&tv);
    }
    __syncwarp();
    int k_issued = 0, v_issued = 0, q0_issued = 0, q1_issued = 0;
    Cursor c;
    c.start(prm, first, step, split);
    for (; c.more(prm); c.next(prm, step, split)) {
      const Item& it = c.it;
      const int st = c.kt % kStages;
      const uint32_t ph = ((c.kt / kStages) & 1) ^ 1;
      const int row = (it.j0 + c.j) * kKV;
      if (!mbar_wait_warp(&k_empty[st], ph, kErrStageFree, abort_flag)) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(&k_full[st], kTile);
        for (int h = 0; h < Cf::kHalves; ++h)
          tma_load_4d(sK(st) + h * (kTile / 2), &tk, &k_full[st], h * 64, row, it.kvh * prm.kv.kh,
                      it.b * prm.kv.kb);
      }
      __syncwarp();
      ++k_issued;
      if (c.j == 0) {
        bool ok = true;
        for (int t = 0; ok && t < it.tiles; ++t) {
          // the item before has made its last S from this tile's queries
          ok = mbar_wait_warp(&q_empty[t], (c.items(t) & 1) ^ 1, kErrStageFree, abort_flag);
          if (ok && elect_one()) {
            mbar_arrive_expect_tx(&q_full[t],
                                  static_cast<uint32_t>(Cf::kHalves * Cf::kRowBytes * p.group * prm.qpt));
            for (int h = 0; h < Cf::kHalves; ++h)
              tma_load_4d(sQ + t * kTile + h * (kTile / 2), &tq, &q_full[t], h * 64, it.kvh * p.group,
                          it.q0 + t * prm.qpt, it.b * prm.qmul_b);
          }
          __syncwarp();
          q0_issued += ok && t == 0;
          q1_issued += ok && t == 1;
        }
        if (!ok) break;
      }
      if (!mbar_wait_warp(&v_empty[st], ph, kErrStageFree, abort_flag)) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(&v_full[st], kTile);
        for (int h = 0; h < Cf::kHalves; ++h)
          tma_load_4d(sV(st) + h * (kTile / 2), &tv, &v_full[st], h * 64, row, it.kvh * prm.kv.vh,
                      it.b * prm.kv.vb);
      }
      __syncwarp();
      ++v_issued;
    }
    // The last copies are seen in, also where a wait gave up: this shared
    // memory may be another CTA's as soon as this one ends.
    for (int i = max(0, k_issued - kStages); i < k_issued; ++i)
      mbar_wait_warp(&k_full[i % kStages], (i / kStages) & 1, kErrTmaWait, nullptr);
    for (int i = max(0, v_issued - kStages); i < v_issued; ++i)
      mbar_wait_warp(&v_full[i % kStages], (i / kStages) & 1, kErrTmaWait, nullptr);
    if (q0_issued > 0) mbar_wait_warp(&q_full[0], (q0_issued - 1) & 1, kErrTmaWait, nullptr);
    if (q1_issued > 0) mbar_wait_warp(&q_full[1], (q1_issued - 1) & 1, kErrTmaWait, nullptr);
  } else if (warp == 1 && aligned) {
    // ------------------------------------------------------------ MMA
    const uint32_t fmt = kBf16 ? 1u : 0u;
    const uint32_t idesc_pv = make_idesc(fmt, kQ, kD, 1u);
    auto sdesc_k = [](uint32_t a) { return kD == 32 ? make_sdesc_sw64(a) : make_sdesc_sw128(a); };
    auto sdesc_mn = [](uint32_t a) { return kD == 32 ? make_sdesc_sw64_mn(a) : make_sdesc_sw128_mn(a); };
    constexpr uint32_t kHalfStep = kTile / 2 >> 4;            // the second 64 columns of a D = 128 tile
    constexpr uint32_t kVStep = 16 * Cf::kRowBytes >> 4;      // 16 keys of V
    // S_t = Q_t K_j^T, over the P (and S) that the MMAs issued before have read
    auto issue_s = [&](int t, const Cursor& c) -> bool {
      const int st = c.kt % kStages;
      if (t == 0 && !mbar_wait_warp(&k_full[st], (c.kt / kStages) & 1, kErrTmaWait, abort_flag)) return false;
      if (c.j == 0 && !mbar_wait_warp(&q_full[t], c.items(t) & 1, kErrTmaWait, abort_flag)) return false;
      tc_fence_after();
      const uint64_t qdesc = sdesc_k(smem_u32(sQ + t * kTile)), kdesc = sdesc_k(smem_u32(sK(st)));
      const uint32_t idesc_s = make_idesc(fmt, kQ, c.keys());
#pragma unroll
      for (int kk = 0; kk < kD / 16; ++kk) {  // 16 elements = 32 bytes along D
        const uint64_t at = (kk / 4) * kHalfStep + 2 * (kk % 4);
        umma_ss_warp(tS(t), qdesc + at, kdesc + at, idesc_s, kk ? 1u : 0u);
      }
      umma_commit_warp(&s_full[t]);
      if (c.j == c.it.n_kv - 1) umma_commit_warp(&q_empty[t]);
      if (t == c.it.tiles - 1) umma_commit_warp(&k_empty[st]);
      return true;
    };
    Cursor s, c;  // of the next S, and of P.V behind it
    s.start(prm, first, step, split);
    c = s;
    bool ok = true;
    if (s.more(prm)) {
      for (int t = 0; ok && t < s.it.tiles; ++t) ok = issue_s(t, s);
      s.next(prm, step, split);
    }
    for (; ok && c.more(prm); c.next(prm, step, split)) {
      const int st = c.kt % kStages, n = c.keys();
      const bool ahead = s.more(prm);
      if (!mbar_wait_warp(&v_full[st], (c.kt / kStages) & 1, kErrTmaWait, abort_flag)) break;
      const uint64_t vdesc = sdesc_mn(smem_u32(sV(st)));
      for (int t = 0; ok && t < 2; ++t) {
        if (t < c.it.tiles) {
          // the epilogue of the item before has read O
          ok = c.j > 0 || c.items(t) == 0 ||
               mbar_wait_warp(&o_empty[t], (c.items(t) - 1) & 1, kErrAccFree, abort_flag);
          ok = ok && mbar_wait_warp(&p_full[t], c.turns(t) & 1, kErrAccFull, abort_flag);
          if (!ok) break;
          tc_fence_after();
          if (n == kKV) {
#pragma unroll
            for (int kk = 0; kk < kKV / 16; ++kk)  // A = P from TMEM: 16 keys = 8 columns
              umma_ts_warp(tO(t), tS(t) + kk * 8, vdesc + kk * kVStep, idesc_pv, (c.j | kk) ? 1u : 0u);
          } else {
#pragma unroll 1
            for (int kk = 0; kk < n / 16; ++kk)
              umma_ts_warp(tO(t), tS(t) + kk * 8, vdesc + kk * kVStep, idesc_pv, (c.j | kk) ? 1u : 0u);
          }
          if (t == c.it.tiles - 1) umma_commit_warp(&v_empty[st]);
          if (c.j == c.it.n_kv - 1) umma_commit_warp(&o_full[t]);
        }
        if (ahead && t < s.it.tiles) ok = issue_s(t, s);
      }
      if (ahead) s.next(prm, step, split);
    }
    // and so are the last MMAs, before TMEM is given back
    umma_commit_warp(mma_done);
    mbar_wait_warp(mma_done, 0, kErrAccFull, nullptr);
  } else if (warp >= 4) {
    // ------------------------------------------------ softmax + epilogue
    const int t = (warp - 4) >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;  // row within the tile
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const float sl2 = p.scale_log2;
    bool ok = aligned && t < prm.tiles;
    int kt = 0, turn = 0, nth = 0;  // key tiles in the rings, of this query tile, its items
    for (int idx = first; ok && idx < prm.n_items; idx += step) {
      int n_kv, n;  // key tiles, keys left
      const uint8_t* mask = nullptr;
      {
        const Item it = item_of(prm, idx, split);
        n_kv = it.n_kv;
        n = it.len - it.j0 * kKV;
        if (kMask) mask = p.key_mask + it.b * p.mask_stride + it.j0 * kKV;
        if (t >= it.tiles) {
          kt += n_kv;
          if (prm.splits == 1) continue;
          n_kv = 0;  // (a cluster's CTA still meets its barriers)
        }
      }
      float m_used = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int j = 0; j < n_kv; ++j, ++kt, ++turn, n -= kKV) {
        const int st = kt % kStages;
        // the tile's key bits, by 32 keys
        uint32_t w[4] = {~0u, ~0u, ~0u, ~0u};
        if (kMask) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = i * 32 + lane;
            w[i] = __ballot_sync(0xffffffffu, key < n && mask[j * kKV + key] != 0);
          }
        }
        const bool some_off = (w[0] & w[1] & w[2] & w[3]) != ~0u;
        if (!mbar_wait_warp(&s_full[t], turn & 1, kErrAccFull, abort_flag)) { ok = false; break; }
        tc_fence_after();
        // Columns c0 .. of S, with -inf where a key does not count.
        auto masked = [&](float* sv, int c0, int cols) {
          if (kMask) {
#pragma unroll
            for (int i = 0; i < cols / 32; ++i) {
              if (w[c0 / 32 + i] != 0xffffffffu) {
#pragma unroll
                for (int c = 0; c < 32; ++c)
                  if (!(w[c0 / 32 + i] >> c & 1)) sv[i * 32 + c] = -INFINITY;
              }
            }
          } else if (n < c0 + cols) {
#pragma unroll
            for (int c = 0; c < cols; ++c)
              if (c0 + c >= n) sv[c] = -INFINITY;
          }
        };
        // A thread keeps 96 of its 128 values from the maximum to the
        // exponentials and loads the other 32 again: with all of them the
        // registers do not do, and spilled ones gave wrong values (they are
        // targets of asynchronous loads).
        float sv[96], mt;
        {
          float last[32];
          tmem_ld_wait_32x32b_32(tS(t) + lane_off + 96, last);
          masked(last, 96, 32);
          mt = max32(last);
        }
        tmem_ld_wait_32x32b_96(tS(t) + lane_off, sv);
        masked(sv, 0, 96);
        mt = fmaxf(mt, fmaxf(max64(sv), max32(sv + 64)));
        const bool need = (mt - m_used) * sl2 > kRescaleLog2;  // false for -inf - -inf
        const float m_new = fmaxf(m_used, mt), top = fabsf(m_new * sl2);
        const bool far_row = top > kFarLog2 && fabsf(m_new) < INFINITY;
        if (__any_sync(0xffffffffu, need || far_row)) {
          const float corr = m_used == -INFINITY ? 0.f : ex2((m_used - m_new) * sl2);
          l *= corr;
          m_used = m_new;
          if (j > 0) {  // (O is at rest: s_full counts the P.V issued before this S)
#pragma unroll
            for (int c = 0; c < kD / 8; ++c) {
              uint32_t u[8];
              tmem_ld_wait_32x32b_x8(tO(t) + lane_off + c * 8, u);
#pragma unroll
              for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * corr);
              tmem_st_32x32b_x8(tO(t) + lane_off + c * 8, u);
            }
            tmem_st_wait();
          }
          if (__any_sync(0xffffffffu, far_row)) {
            const float off = far_row ? m_used : 0.f;
#pragma unroll
            for (int c = 0; c < 96; ++c) sv[c] -= off;
#pragma unroll
            for (int c = 96; c < 128; c += 8) {  // and off those that are loaded again
              uint32_t u[8];
              tmem_ld_wait_32x32b_x8(tS(t) + lane_off + c, u);
#pragma unroll
              for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) - off);
              tmem_st_32x32b_x8(tS(t) + lane_off + c, u);
            }
            tmem_st_wait();
          }
        }
        // no key yet: every exponent is -inf against 0
        const float add = (m_used == -INFINITY || far_row ? 0.f : -m_used * sl2) + (kBf16 ? 0.f : kF16Shift);
        uint64_t l2[2] = {f2pack(0.f, 0.f), f2pack(0.f, 0.f)};
        exp_store<kBf16, 96>(sv, sl2, add, tS(t) + lane_off, l2);  // P takes the place of S
        if (n > 96) {  // (P of keys past the last 16 is not multiplied)
          float last[32];
          tmem_ld_wait_32x32b_32(tS(t) + lane_off + 96, last);
          masked(last, 96, 32);
          exp_store<kBf16, 32>(last, sl2, add, tS(t) + lane_off + 48, l2);
        }
        float a0, a1;
        f2unpack(fadd2(l2[0], l2[1]), a0, a1);
        l += a0 + a1;
        tmem_st_wait();
        // V rows that P.V reads and that do not count: 0 * NaN would reach O.
        // (Both query tiles' warps write the same zeros.)
        const int n16 = min((n + 15) & ~15, kKV);
        if (kMask ? some_off : n < n16 && p.k_lens != nullptr) {
          if (!mbar_wait_warp(&v_full[st], (kt / kStages) & 1, kErrTmaWait, abort_flag)) { ok = false; break; }
          const int v = quarter * 32 + lane;
          if (v < n16 && (v >= n || (kMask && mask[j * kKV + v] == 0))) {
            for (int h = 0; h < Cf::kHalves; ++h)
#pragma unroll
              for (int k = 0; k < Cf::kRowBytes; k += 16)
                *reinterpret_cast<uint4*>(sV(st) + h * (kTile / 2) + v * Cf::kRowBytes + k) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      if (ok && n_kv > 0) ok = mbar_wait_warp(&o_full[t], nth & 1, kErrAccFull, abort_flag);
      if (!ok && prm.splits == 1) break;  // (a cluster's CTA still meets its barriers)
      tc_fence_after();
      const Item it = item_of(prm, idx, split);
      const int rq = r / p.group, rh = r - rq * p.group, query = it.q0 + t * prm.qpt + rq;
      const bool row_live = r < prm.qpt * p.group && query < p.sq;
      if (prm.splits > 1) {
        // this CTA's share of the keys: (max, sum) and the partial row, over
        // the rings once neither tile's MMAs read them
        asm volatile("bar.sync 1, %0;" ::"r"(prm.tiles * kQ) : "memory");
        ml[t * kQ + r] = make_float2(m_used, l);
        float* part = reinterpret_cast<float*>(smem) + (t * kQ + r) * Cf::kPitch;
#pragma unroll
        for (int c0 = 0; c0 < kD; c0 += 16) {
          uint32_t u[16];
          tmem_ld_wait_32x32b_x16(tO(t) + lane_off + c0, u);
#pragma unroll
          for (int i = 0; i < 16; i += 4)  // (without a key tile O holds nothing)
            *reinterpret_cast<float4*>(part + c0 + i) =
                n_kv ? make_float4(__uint_as_float(u[i]), __uint_as_float(u[i + 1]), __uint_as_float(u[i + 2]),
                                      __uint_as_float(u[i + 3]))
                        : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      } else {
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no key: zeros; NaN stays NaN
        uint16_t* orow = p.o + it.b * p.ob + query * p.os + static_cast<int64_t>(it.kvh * p.group + rh) * p.oh;
#pragma unroll
        for (int c0 = 0; c0 < kD; c0 += 16) {
          uint32_t u[16];
          tmem_ld_wait_32x32b_x16(tO(t) + lane_off + c0, u);
          if (row_live) {
#pragma unroll
            for (int q8 = 0; q8 < 2; ++q8) {
              if (c0 + q8 * 8 < p.head_dim) {
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = n_kv ? __uint_as_float(u[q8 * 8 + i]) * inv : 0.f;
                uint4 w;
                w.x = pack2(f[0], f[1], kBf16);
                w.y = pack2(f[2], f[3], kBf16);
                w.z = pack2(f[4], f[5], kBf16);
                w.w = pack2(f[6], f[7], kBf16);
                *reinterpret_cast<uint4*>(orow + c0 + q8 * 8) = w;
              }
            }
          }
        }
      }
      if (n_kv > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[t]);  // the next item's P.V may overwrite O
        ++nth;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (prm.splits == 1) return;
  // The cluster's CTAs sum a share of the item's rows each, over all of them
  // in rank order.
  cluster_sync();
  const Item it = item_of(prm, first, split);
  const int chunks = p.head_dim / 8;
  const uint32_t part_s = smem_u32(smem), ml_s = smem_u32(ml);
  for (int i = threadIdx.x + kThreads * split; i < it.tiles * kQ * chunks; i += kThreads * prm.splits) {
    const int row = i / chunks, c = (i % chunks) * 8;
    const int t = row / kQ, r = row % kQ, rq = r / p.group, query = it.q0 + t * prm.qpt + rq;
    if (r >= prm.qpt * p.group || query >= p.sq) continue;
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, l = 0.f, m = -INFINITY;
    for (int w = 0; w < prm.splits; ++w) m = fmaxf(m, ld_cluster_f2(mapa_shared(ml_s + row * 8, w)).x);
    const float base = m == -INFINITY ? 0.f : m;
    for (int w = 0; w < prm.splits; ++w) {
      const float2 s = ld_cluster_f2(mapa_shared(ml_s + row * 8, w));
      const float f = ex2((s.x - base) * p.scale_log2);
      l = fmaf(f, s.y, l);
      const uint32_t src = mapa_shared(part_s + (row * Cf::kPitch + c) * 4, w);
      const float4 x = ld_cluster_f4(src), y = ld_cluster_f4(src + 16);
      const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = fmaf(f, v[e], o[e]);
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    uint4 w4;
    w4.x = pack2(o[0] * inv, o[1] * inv, kBf16);
    w4.y = pack2(o[2] * inv, o[3] * inv, kBf16);
    w4.z = pack2(o[4] * inv, o[5] * inv, kBf16);
    w4.w = pack2(o[6] * inv, o[7] * inv, kBf16);
    *reinterpret_cast<uint4*>(p.o + it.b * p.ob + query * p.os +
                              static_cast<int64_t>(it.kvh * p.group + r - rq * p.group) * p.oh + c) = w4;
  }
  cluster_sync();  // the others may still read this CTA's partial rows
}

std::atomic<bool> as_if_spilled{false};
std::atomic<int> builds_spilled{0};

template <bool kBf16, int kD, bool kMask>
int launch_variant(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, TcParams& prm, int key_tiles,
                   cudaStream_t st) {
  const auto kernel = cross_tc_kernel<kBf16, kD, kMask>;
  static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
  static std::atomic<int> spills{-1};     // of this build: see the softmax's registers
  if (spills.load() < 0) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kernel) != cudaSuccess) {
      cudaGetLastError();
      return kErrCuda;
    }
    const int s = fa.localSizeBytes != 0;
    if (spills.exchange(s) < 0) builds_spilled.fetch_add(s);
  }
  if (spills.load() || as_if_spilled.load()) return kCrossTcSpills;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return kErrCuda;
  if (dev >= 64 || !(ready.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<kD>::kSmem) != cudaSuccess) {
      cudaGetLastError();
      return kErrCuda;
    }
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  static ClusterTable clusters;
  prm.splits = cluster_splits(kernel, kThreads, Cfg<kD>::kSmem, prm.n_items, key_tiles, 4, 8, clusters);
  // Short items: one CTA per SM that walks them, so that an item's first loads
  // and S overlap the epilogue before it (4 x 8 heads x 5184 queries, 77 / 512 /
  // 2048 keys, D = 64: 26 / 54 / 167 us against 36 / 64 / 176 with a CTA each;
  // 4096 keys 320 and 327, but lengths that differ would leave SMs without work).
  // Long ones have a CTA each, dealt out as SMs come free (lengths differ).
  int64_t ctas = static_cast<int64_t>(prm.n_items) * prm.splits;
  if (prm.splits == 1 && key_tiles <= 16) ctas = std::min<int64_t>(ctas, num_sms());
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg<kD>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  if (prm.splits > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = prm.splits;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
  count_launches(1);
  if (cudaLaunchKernelEx(&cfg, kernel, mq, mk, mv, prm) == cudaSuccess) return kOk;
  cudaGetLastError();  // the next call's own check must not see it
  return kErrLaunch;
}

template <int kD>
int launch_typed(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, TcParams& prm, int dtype,
                 int key_tiles, cudaStream_t st) {
  const bool mask = prm.c.key_mask != nullptr;  // (lengths alone need none of it)
  if (dtype == kBF16)
    return mask ? launch_variant<true, kD, true>(mq, mk, mv, prm, key_tiles, st)
                : launch_variant<true, kD, false>(mq, mk, mv, prm, key_tiles, st);
  return mask ? launch_variant<false, kD, true>(mq, mk, mv, prm, key_tiles, st)
              : launch_variant<false, kD, false>(mq, mk, mv, prm, key_tiles, st);
}

}  // namespace

int cross_tc_as_if_spilled(bool on) {
  as_if_spilled.store(on);
  return builds_spilled.load();
}

bool cross_tc_takes(const CrossParams& p) {
  if (p.bias || !cross_kv_maps(p)) return false;
  constexpr int64_t kMost = 1ll << 39;
  if (p.qb >= kMost || p.qs >= kMost || p.qh >= kMost) return false;
  return (p.sq == 1 || p.qs != 0) && (p.kv_heads * p.group == 1 || p.qh != 0);
}

int launch_cross_tc(const CrossParams& p, int dtype, cudaStream_t st) {
  TcParams prm;
  memset(&prm, 0, sizeof(prm));
  prm.c = p;
  prm.qpt = kQ / p.group;
  const int64_t row_tiles = (static_cast<int64_t>(p.sq) + prm.qpt - 1) / prm.qpt;
  const int64_t heads = static_cast<int64_t>(p.kv_heads) * p.batch;
  const int key_tiles = (p.sk + kKV - 1) / kKV;
  // Two query tiles to a CTA; one, where even then there are SMs to spare, and
  // the keys over the CTAs of a cluster while there still are (with at least
  // four key tiles each).
  prm.tiles = heads * row_tiles <= num_sms() ? 1 : 2;
  prm.items_x = static_cast<int>((row_tiles + prm.tiles - 1) / prm.tiles);
  if (heads * prm.items_x > 0x3fffffffLL) return kErrShape;
  prm.n_items = static_cast<int>(heads * prm.items_x);
  prm.splits = 1;
  CUtensorMap mq, mk, mv;
  const TensorDim dq[3] = {{static_cast<int64_t>(p.kv_heads) * p.group, p.qh, nullptr}, {p.sq, p.qs, nullptr},
                           {p.batch, p.qb, &prm.qmul_b}};
  const int bq[3] = {p.group, prm.qpt, 1};
  if (!make_cross_map(&mq, p.q, dtype, p.head_dim, dq, bq) || !make_kv_maps(p, dtype, kKV, &mk, &mv, &prm.kv))
    return kErrTma;
  if (p.head_dim <= 32) return launch_typed<32>(mq, mk, mv, prm, dtype, key_tiles, st);
  if (p.head_dim <= 64) return launch_typed<64>(mq, mk, mv, prm, dtype, key_tiles, st);
  return launch_typed<128>(mq, mk, mv, prm, dtype, key_tiles, st);
}

}  // namespace s3
