// C ABI launch layer of the low-bit decode operators (declarations:
// include/b200q.h): 4-bit weight linears, the norms before and after a block,
// and the paged 8-bit key/value cache.  As in capi.cu: arguments are checked on
// the host before any launch, nothing is allocated, nothing synchronises, and
// kernels go to the caller's stream as programmatic dependents.
#include "../../include/b200q.h"
#include <algorithm>

#include "block_norm.cuh"
#include "host.h"
#include "kv8.cuh"
#include "kv8_prefill.cuh"
#include "w4_tile.cuh"
#include "w4a16.cuh"

using namespace b200q;

namespace b200q {
namespace host {
int lowbit_device_status(unsigned int* status, bool reset) {
  if (cudaMemcpyFromSymbol(status, g_device_status, sizeof(unsigned int)) != cudaSuccess)
    return B200Q_ERR_CUDA;
  const unsigned int zero = 0;
  if (reset && cudaMemcpyToSymbol(g_device_status, &zero, sizeof(unsigned int)) != cudaSuccess)
    return B200Q_ERR_CUDA;
  return B200Q_OK;
}
}  // namespace host
}  // namespace b200q

namespace {

constexpr int64_t kIntMax = (int64_t(1) << 31) - 1;

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A launch with optional dynamic shared memory, as a programmatic dependent of the kernel
// before it (B200Q_PDL=0: plainly).
template <typename... KArgs, typename... Args>
int launch(void (*kern)(KArgs...), dim3 grid, int block, int smem, cudaStream_t st, Args... args) {
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
    cudaGetLastError();
    return B200Q_ERR_CUDA;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(block));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = host::pdl_on() ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kern, args...);  // errors surface in finish_launch
  return host::finish_launch();
}

// ------------------------------------------------------------ 4-bit linear
// Largest M of the warp-MMA kernels, whose products are exact.
constexpr int64_t kW4MaxSmallM = 32;

// K slices and row parts of the slice kernel: the split whose busiest warp has the
// fewest groups to go through, x's slice beside the rings.  More than kWsMaxSlices only where
// x's slice fits no otherwise (32 tokens: K above 42,000 to 57,000 by the group size).
constexpr int kWsMaxSlices = 32;
struct WsPlan {
  int slices, parts, smem;
};
bool ws_plan(int sms, int64_t M, int64_t N, int64_t K, int G, WsPlan* p) {
  const int64_t KG = K / G, tiles = cdiv(N, 16);
  int64_t best = -1;
  for (int s = 1; s <= KG && s <= sms && (s <= kWsMaxSlices || best < 0); ++s) {
    const int64_t gs = cdiv(KG, s);
    const int64_t smem = kWsWarps * kWsStages * 2048 + M * 2 * gs * G;  // (without the pitch's padding: 64 bits)
    if (smem > 227 * 1024 || ws_smem_bytes(int(M), int(gs) * G, G) > 227 * 1024) continue;
    const int64_t parts = sms / s;
    // a slice more costs its partial sums' round trip, about 2 groups of a warp
    const int64_t cost = cdiv(tiles, parts * kWsWarps) * gs * G / 32 + (s > 1 ? 8 + s / 4 : 0);
    if (best < 0 || cost < best) {
      best = cost;
      p->slices = s;
      p->parts = static_cast<int>(parts < cdiv(tiles, kWsWarps) ? parts : cdiv(tiles, kWsWarps));
      p->smem = ws_smem_bytes(int(M), int(gs) * G, G);
    }
  }
  return best >= 0;
}

int launch_join(const float* part, int slices, int64_t ld, const EpiArgs& ep, cudaStream_t st) {
  const int64_t chunks = cdiv(ep.N, 256);
  if (ep.M * chunks > kIntMax) return B200Q_ERR_UNSUPPORTED;
  return launch(w4_join_kernel, dim3(static_cast<unsigned>(ep.M * chunks)), 256, 0, st, part, slices, ld,
                static_cast<int>(chunks), ep);
}

template <int LW>
int launch_slice_cols(const W4SliceArgs& a, const EpiArgs& ep, const WsPlan& p, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.slices * p.parts));
  if (a.M <= 8) return launch(w4_slice_kernel<LW, 1>, grid, kWsWarps * 32, p.smem, st, a, ep);
  if (a.M <= 16) return launch(w4_slice_kernel<LW, 2>, grid, kWsWarps * 32, p.smem, st, a, ep);
  return launch(w4_slice_kernel<LW, 4>, grid, kWsWarps * 32, p.smem, st, a, ep);
}
int launch_slice(const W4SliceArgs& a, int G, const EpiArgs& ep, const WsPlan& p, cudaStream_t st) {
  int s = G == 32   ? launch_slice_cols<1>(a, ep, p, st)
          : G == 64 ? launch_slice_cols<2>(a, ep, p, st)
                    : launch_slice_cols<4>(a, ep, p, st);
  if (s != B200Q_OK || !a.part) return s;
  return launch_join(a.part, a.slices, a.N, ep, st);
}

// The integer kernel for few tokens, when x's digits fit beside the rings.  (Against the slice
// kernel, us.  1 token, N 1024 / 5120 / 13824: K 5120 4.5 7.9 11.8 against 7.3 11.5 17.4, K
// 13824 9.3 15.0 21.2 against 9.9 18.3 33.7, K 24576 13.7 23.7 33.3 against 10.9 27.6 51.9; 2
// tokens: K 5120 5.4 8.2 12.1 against 7.2 12.1 17.6, K 12288 10.8 15.1 20.1 against 9.4 17.3
// 28.8: longer rows lose at narrow N only.  N 5120: 3 tokens K 1536 5.4 / 7.5, K 2560 8.0 / 9.5,
// K 5120 14.4 / 12.2; 5 tokens K 1536 6.8 / 7.6; 8 tokens K 1024 6.9 / 6.9, K 1536 9.2 / 8.0:
// more than two tokens while M * K is small.)
struct WdPlan {
  int smem, grid, threads;
};
bool wd_plan(int sms, int64_t M, int64_t N, int64_t K, int G, WdPlan* p) {
  if (M > 8 || M * K > (M <= 2 ? 24 : 8) * 1024) return false;
  const int nc = M <= 2 ? 1 : M <= 5 ? 2 : 3;
  int teams = wd_teams(nc);
  for (; teams > 0; --teams) {
    p->smem = wd_layout(int(M), int(K), G, nc, teams).total;
    if (p->smem <= 227 * 1024) break;
  }
  if (!teams) return false;
  // no more teams than tiles per SM, and the fewest CTAs that need as few rounds
  const int64_t tiles = cdiv(N, 16);
  teams = static_cast<int>(cdiv(tiles, sms) < teams ? cdiv(tiles, sms) : teams);
  const int64_t rounds = cdiv(tiles, int64_t(sms) * teams);
  p->smem = wd_layout(int(M), int(K), G, nc, teams).total;
  p->threads = teams * kW4Warps * 32;
  p->grid = static_cast<int>(cdiv(tiles, rounds * teams));
  return true;
}
template <typename T, int LW>
int launch_digits_cols(const W4DigitArgs& a, const EpiArgs& ep, const WdPlan& p, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.grid));
  if (a.M <= 2) return launch(w4_digit_kernel<T, LW, 1>, grid, p.threads, p.smem, st, a, ep);
  if (a.M <= 5) return launch(w4_digit_kernel<T, LW, 2>, grid, p.threads, p.smem, st, a, ep);
  return launch(w4_digit_kernel<T, LW, 3>, grid, p.threads, p.smem, st, a, ep);
}
template <typename T>
int launch_digits(const W4DigitArgs& a, int G, const EpiArgs& ep, const WdPlan& p, cudaStream_t st) {
  if (G == 32) return launch_digits_cols<T, 1>(a, ep, p, st);
  if (G == 64) return launch_digits_cols<T, 2>(a, ep, p, st);
  return launch_digits_cols<T, 4>(a, ep, p, st);
}

// Rows of N % 8 != 0 outputs start off the tile GEMM's vector stores (its element stores, a
// row per lane, took 35 us for 144 x 4135): fp32 rows of a padded stride go to the
// workspace instead, and the join kernel runs the epilogue from there.
bool w4_joins(int64_t N) { return N % 8 != 0; }
int64_t w4_join_ld(int64_t N) { return cdiv(N, 32) * 32; }
struct W4Work {
  size_t w, x, row, last, col, out, total;  // byte offsets
};
W4Work w4_work(int64_t M, int64_t N, int64_t K) {
  auto up = [](size_t b) { return (b + 255) & ~size_t(255); };
  W4Work o{};
  o.x = up(size_t(N) * K * 2);
  o.row = o.x + up(size_t(M) * K * 2);
  o.last = o.row + up(size_t(M) * 4);
  o.col = o.last + up(4);
  o.out = o.col + up(size_t(N) * 4);
  o.total = o.out + (w4_joins(N) ? up(size_t(M) * w4_join_ld(N) * 4) : 0);
  return o;
}

// 33 to 256 tokens: one token tile of the tile kernel.  (Measured at K 5120, N 13824: 64 tokens
// 50 us, 64 on the slice kernel in two passes; 256 tokens 63 us, 80 decoded; K 13824, N 5120:
// 200 tokens 56 us, 129 decoded.  With more token tiles the weight is decoded again for each,
// and the decoded copy with the pair GEMM is ahead: 300 tokens 98 us, 164 by tiles.)
constexpr int64_t kW4MaxTileM = 256;
bool w4_tiles(int64_t M, int64_t N, int64_t K) {
  return M <= kW4MaxTileM && N <= (int64_t(1) << 30) && K <= (int64_t(1) << 24);
}
// K slices of the tile kernel: the split with the lowest estimate, in cycles.  A slot takes four
// times the longest of a stage's MMAs, its bytes from L2 and its decode; a tile its start and
// store besides, and slices the sums' round trip and the join's launch.
struct W4TilePlan {
  int tn, slices;
};
constexpr int kW4TileMaxSlices = 16;
W4TilePlan w4_tile_plan(int sms, int64_t M, int64_t N, int64_t K) {
  const int64_t slots = cdiv(K, 256), tiles = cdiv(N, 128);
  const int tn = M <= 64 ? 64 : M <= 128 ? 128 : 256;
  const int64_t slot = 4 * std::max<int64_t>({2 * tn, (tn * 128 + 5120) / 64, 300});
  W4TilePlan best{tn, 1};
  int64_t least = -1;
  for (int s = 1; s <= kW4TileMaxSlices && s <= slots; ++s) {
    const int64_t cost = cdiv(tiles * s, sms ? sms : 148) * (cdiv(slots, s) * slot + 2000 + 16 * tn) +
                         (s > 1 ? 4000 + s * M * N * 8 / 3000 : 0);
    if (least < 0 || cost < least) {
      least = cost;
      best.slices = s;
    }
  }
  return best;
}
struct W4TileWork {
  size_t x, x_pow, w_pow, sz, part, total;  // byte offsets
};
W4TileWork w4_tile_work(const W4TilePlan& p, int64_t M, int64_t N, int64_t K, int64_t G) {
  auto up = [](size_t b) { return (b + 255) & ~size_t(255); };
  W4TileWork o{};
  o.x_pow = up(size_t(M) * K * 2);
  o.w_pow = o.x_pow + up(size_t(M) * 4);
  o.sz = o.w_pow + up(size_t(N) * 4);
  o.part = o.sz + up(size_t(cdiv(K, 256) * (256 / G)) * cdiv(N, 128) * 128 * 8);
  o.total = o.part + (p.slices > 1 ? up(size_t(p.slices) * M * N * 4) : 0);
  return o;
}
template <int TN, bool LO>
int launch_tile(const CUtensorMap& tx, const CUtensorMap& tw, const W4TileArgs& a, const EpiArgs& ep, int64_t ctas,
                cudaStream_t st) {
  return launch(w4_tile_kernel<TN, LO>, dim3(static_cast<unsigned>(ctas)), kW4TileThreads, w4_tile_smem_bytes<TN>(),
                st, tx, tw, a, ep);
}
int launch_w4_tile(const W4TilePlan& p, const void* x, int x_dtype, int64_t ldx, bool x_vec, const uint8_t* w,
                   int64_t ldw, const void* scales, int scale_dtype, const uint8_t* zeros, int64_t G, int64_t M,
                   int64_t N, int64_t K, const EpiArgs& ep, uint8_t* base, cudaStream_t st) {
  const W4TileWork o = w4_tile_work(p, M, N, K, G);
  const int64_t slots = cdiv(K, 256), ctas = cdiv(N, 128) * p.slices;
  W4TilePrepareArgs r{};
  r.x = x;
  r.ldx = ldx;
  r.x_f16 = x_dtype == B200Q_F16;
  r.x_vec = x_vec;
  r.M = static_cast<int>(M);
  r.K = static_cast<int>(K);
  r.x16 = reinterpret_cast<__half*>(base + o.x);
  r.x_pow = reinterpret_cast<float*>(base + o.x_pow);
  r.scales = scales;
  r.scale_dtype = scale_dtype;
  r.zeros = zeros;
  r.N = static_cast<int>(N);
  r.KG = static_cast<int>(K / G);
  r.groups = static_cast<int>(slots * (256 / G));
  r.ldn = static_cast<int>(cdiv(N, 128) * 128);
  r.sz = reinterpret_cast<uint2*>(base + o.sz);
  r.w_pow = reinterpret_cast<float*>(base + o.w_pow);
  r.group_blocks = static_cast<int>(cdiv(r.groups, kW4PrepGroups));
  r.scale_blocks = r.ldn / kW4PrepRows * r.group_blocks;
  int s = launch(w4_tile_prepare_kernel, dim3(static_cast<unsigned>(r.scale_blocks + M)), 256, 0, st, r);
  if (s != B200Q_OK) return s;
  CUtensorMap tx, tw;
  if (!host::tmap_u8(&tx, r.x16, uint64_t(2 * K), uint64_t(M), uint64_t(2 * K), 128, static_cast<uint32_t>(p.tn),
                     CU_TENSOR_MAP_SWIZZLE_128B) ||
      !host::tmap_u8(&tw, w, uint64_t(K / 2), uint64_t(N), uint64_t(ldw), 128, 128, CU_TENSOR_MAP_SWIZZLE_128B))
    return B200Q_ERR_CUDA;
  W4TileArgs a{};
  a.sz = r.sz;
  a.ldn = r.ldn;
  a.w_pow = r.w_pow;
  a.x_pow = r.x_pow;
  a.part = p.slices > 1 ? reinterpret_cast<float*>(base + o.part) : nullptr;
  a.M = r.M;
  a.N = r.N;
  a.slots = static_cast<int>(slots);
  a.log_g = G == 32 ? 5 : G == 64 ? 6 : 7;
  a.slices = p.slices;
  const bool lo = scale_dtype == kBiasF32;
  if (p.tn == 64) s = lo ? launch_tile<64, true>(tx, tw, a, ep, ctas, st) : launch_tile<64, false>(tx, tw, a, ep, ctas, st);
  else if (p.tn == 128) s = lo ? launch_tile<128, true>(tx, tw, a, ep, ctas, st) : launch_tile<128, false>(tx, tw, a, ep, ctas, st);
  else s = lo ? launch_tile<256, true>(tx, tw, a, ep, ctas, st) : launch_tile<256, false>(tx, tw, a, ep, ctas, st);
  if (s != B200Q_OK || p.slices == 1) return s;
  return launch_join(a.part, p.slices, N, ep, st);
}

// The kernels of a call and the workspace they take.  The integer kernel for few tokens wants
// scales of x's type and indexes them with 31 bits, as the slice kernel does.
// (Up to 32 tokens whose x fits no slice, K above 194,176 at 32, or with 2^31 scales go on to
// the kernels for more.)
enum W4Kind { kW4Digits, kW4Slices, kW4Tiles, kW4Decoded };
struct W4Route {
  W4Kind kind;
  WdPlan wd;
  WsPlan ws;
  W4TilePlan tile;
  size_t need;
};
W4Route w4_route(int sms, int64_t M, int64_t N, int64_t K, int64_t G, bool same_type) {
  W4Route r{};
  const bool small = N * (K / G) <= kIntMax;
  if (same_type && small && wd_plan(sms, M, N, K, int(G), &r.wd)) {
    r.kind = kW4Digits;
  } else if (M <= kW4MaxSmallM && small && ws_plan(sms, M, N, K, int(G), &r.ws)) {
    r.kind = kW4Slices;
    r.need = r.ws.slices > 1 ? size_t(r.ws.slices) * M * N * 4 : 0;
  } else if (w4_tiles(M, N, K)) {
    r.kind = kW4Tiles;
    r.tile = w4_tile_plan(sms, M, N, K);
    r.need = w4_tile_work(r.tile, M, N, K, G).total;
  } else {
    r.kind = kW4Decoded;
    r.need = w4_work(M, N, K).total;
  }
  return r;
}

// PERSIST: as many CTAs as are resident at once (at most one per row).
template <typename K>
int launch_persistent(K kern, const NormArgs& a, int threads, int smem, int sms, cudaStream_t st) {
  int per_sm = 0;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem) != cudaSuccess || per_sm < 1) {
    cudaGetLastError();
    return B200Q_ERR_CUDA;
  }
  const int64_t ctas = int64_t(sms) * per_sm;
  return launch(kern, dim3(static_cast<unsigned>(a.rows < ctas ? a.rows : ctas)), threads, smem, st, a);
}
template <int DTYPE, int VW>
int launch_norm_loose(const NormArgs& a, int sms, cudaStream_t st) {
  const int threads = static_cast<int>(cdiv(cdiv(a.D, kLooseValues), 32) * 32), smem = (a.y ? 3 : 2) * a.D * 4;
  if (a.y) return a.q ? launch_persistent(block_norm_loose_kernel<DTYPE, VW, true, true>, a, threads, smem, sms, st)
                      : launch_persistent(block_norm_loose_kernel<DTYPE, VW, false, true>, a, threads, smem, sms, st);
  return a.q ? launch_persistent(block_norm_loose_kernel<DTYPE, VW, true, false>, a, threads, smem, sms, st)
             : launch_persistent(block_norm_loose_kernel<DTYPE, VW, false, false>, a, threads, smem, sms, st);
}
template <int DTYPE, bool PERSIST, int NPT, bool FULL, bool QUANT, bool AFTER>
int launch_norm_rows(const NormArgs& a, int threads, int sms, cudaStream_t st) {
  auto kern = block_norm_rows_kernel<DTYPE, PERSIST, NPT, FULL, QUANT, AFTER>;
  if (PERSIST) return launch_persistent(kern, a, threads, (AFTER ? 3 : 2) * a.D * 4, sms, st);
  return launch(kern, dim3(static_cast<unsigned>(a.rows)), threads, 0, st, a);
}
template <int DTYPE, bool PERSIST, int NPT, bool FULL>
int launch_norm_rows(const NormArgs& a, int threads, int sms, cudaStream_t st) {
  if (a.y) return a.q ? launch_norm_rows<DTYPE, PERSIST, NPT, FULL, true, true>(a, threads, sms, st)
                      : launch_norm_rows<DTYPE, PERSIST, NPT, FULL, false, true>(a, threads, sms, st);
  return a.q ? launch_norm_rows<DTYPE, PERSIST, NPT, FULL, true, false>(a, threads, sms, st)
             : launch_norm_rows<DTYPE, PERSIST, NPT, FULL, false, false>(a, threads, sms, st);
}
template <int DTYPE, bool PERSIST, int NPT>
int launch_norm_rows(const NormArgs& a, int threads, int sms, cudaStream_t st) {
  return threads * NPT * 8 == a.D ? launch_norm_rows<DTYPE, PERSIST, NPT, true>(a, threads, sms, st)
                                  : launch_norm_rows<DTYPE, PERSIST, NPT, false>(a, threads, sms, st);
}
// Aligned rows of up to 8192 values: one row per CTA and one 8-value vector per thread
// while all rows find a place at once (after + before, 296 rows of 5120: 7.7 us, 297 persistent
// 8.2), else persistent CTAs with four vectors per thread (two for short rows: fewer reductions
// per value, more CTAs per SM).  Other rows
// of up to 8192 values: persistent CTAs, by pairs or single values.  Longer ones take the
// form of 32 single values per thread.
template <int DTYPE>
int launch_norm(const NormArgs& a, bool vec, bool pairs, int sms, cudaStream_t st) {
  if (vec && a.D <= 8192) {
    const int vecs = a.D / 8;
    if (a.rows <= 2 * int64_t(sms))
      return launch_norm_rows<DTYPE, false, 1>(a, static_cast<int>(cdiv(vecs, 32) * 32), sms, st);
    // the vectors per thread that leave the fewest lanes idle
    const int npt = cdiv(vecs, 4 * 32) * 4 <= cdiv(vecs, 2 * 32) * 2 ? 4 : 2;
    const int threads = static_cast<int>(cdiv(vecs, npt * 32) * 32);
    return npt == 4 ? launch_norm_rows<DTYPE, true, 4>(a, threads, sms, st)
                    : launch_norm_rows<DTYPE, true, 2>(a, threads, sms, st);
  }
  if (a.D <= 8192) return pairs ? launch_norm_loose<DTYPE, 2>(a, sms, st) : launch_norm_loose<DTYPE, 1>(a, sms, st);
  return launch(block_norm_kernel<DTYPE, 32>, dim3(static_cast<unsigned>(a.rows)),
                static_cast<int>(cdiv(cdiv(a.D, 32), 32) * 32), 0, st, a);
}

// ------------------------------------------------------------ 8-bit cache
// Checks a cache and fills its kernel view.
bool make_cache(Kv8Cache* c, int8_t* k, int8_t* v, float* ks, float* vs, int64_t pages,
                int64_t heads, int64_t block, int64_t D, const int32_t* table, int64_t ld_table,
                int64_t max_blocks) {
  if (!k || !v || !ks || !vs || !table || pages < 1 || pages > kIntMax || heads < 1 ||
      heads > 65535 || (D != 64 && D != 128) || max_blocks < 1 || ld_table < max_blocks ||
      (block != 16 && block != 32 && block != 64 && block != 128) || max_blocks * block > kIntMax ||
      pages * heads * block > kIntMax || !aligned(k, 16) || !aligned(v, 16))
    return false;
  c->k = k;
  c->v = v;
  c->ks = ks;
  c->vs = vs;
  c->table = table;
  c->ld_table = ld_table;
  c->max_blocks = static_cast<int>(max_blocks);
  c->pages = static_cast<int>(pages);
  c->heads = static_cast<int>(heads);
  c->T = static_cast<int>(block);
  c->D = static_cast<int>(D);
  c->log_t = block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : 7;
  return true;
}

template <typename T>
int launch_append(const Kv8AppendArgs& a, cudaStream_t st) {
  // a sequence may start inside a block: one more block than S fills
  const dim3 grid(static_cast<unsigned>(cdiv(a.S + a.c.T - 1, a.c.T)), static_cast<unsigned>(a.c.heads),
                  static_cast<unsigned>(2 * a.B));
  const int vecs = a.c.T * a.c.D / 8;
  if (vecs <= kKvThreads) return launch(kv8_append_kernel<T, 1>, grid, kKvThreads, 0, st, a);
  if (vecs <= 2 * kKvThreads) return launch(kv8_append_kernel<T, 2>, grid, kKvThreads, 0, st, a);
  if (vecs <= 4 * kKvThreads) return launch(kv8_append_kernel<T, 4>, grid, kKvThreads, 0, st, a);
  return launch(kv8_append_kernel<T, 8>, grid, kKvThreads, 0, st, a);
}

// How many CTAs share a sequence's length.  Up to 16 rows a head: enough to give every
// SM two, and at most 4096 tokens each so that ragged batches balance; at least 128
// tokens each.  More rows (128- or 256-row tiles, two CTAs or one per SM): the split with the fewest
// rounds of stages.  More than one leave fp32 partials for the join kernel.  (A cluster
// of up to 16 CTAs joining over distributed shared memory was no faster: 8 heads x 2048
// tokens 7.4 us against 7.1, 8193 tokens 12.7 against 10.0.)
// Row tiles: 8 rows of 32 x 4096 tokens take 71 us on their kernel, 9 rows 79 on the 16-row one and
// 16 rows 83; a second 16-row tile would read the cache again, and 17 rows take 129 us on the
// 128-row tiles, 128 rows 144.  129 rows: 239 us with 256-row tiles.
int attn_row_tile(int64_t rows) { return rows <= 16 ? 16 : rows <= kPfRows ? kPfRows : 2 * kPfRows; }
int attn_splits(int sms, int64_t B, int64_t Hq, int64_t heads, int64_t Tq, int64_t max_len) {
  const int64_t rows = Hq / heads * Tq;
  const int64_t base = B * heads * cdiv(rows, attn_row_tile(rows));
  if (rows > 16) {
    const int64_t stages = cdiv(max_len, 64), slots = int64_t(sms) * (rows <= kPfRows ? 2 : 1);
    int best = 1;
    int64_t least = -1;
    for (int s = 1; s <= kAttnMaxSplits && (s == 1 || 4 * s <= stages); ++s) {
      // a CTA's start and end cost about four stages
      const int64_t cost = cdiv(base * s, slots) * (cdiv(stages, s) + 4);
      if (least < 0 || cost < least) {
        least = cost;
        best = s;
      }
    }
    return best;
  }
  int64_t s = cdiv(int64_t(sms) * 2, base);
  if (s < cdiv(max_len, 4096)) s = cdiv(max_len, 4096);
  const int64_t most = cdiv(max_len, 128);
  if (s > most) s = most;
  if (s > kAttnMaxSplits) s = kAttnMaxSplits;
  return s < 1 ? 1 : static_cast<int>(s);
}
size_t attn_work_bytes(int splits, int64_t rows, int64_t D) {
  return splits > 1 ? size_t(splits) * rows * (D + 2) * 4 : 0;
}
bool attn_dims(int64_t B, int64_t Hq, int64_t heads, int64_t Tq) {
  return B >= 0 && B <= 65535 && heads >= 1 && Hq >= heads && Hq % heads == 0 && Tq >= 0 &&
         Hq * Tq <= kIntMax && B * Hq * Tq <= kIntMax;
}

}  // namespace

extern "C" {

size_t b200q_w4a16_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t group, int x_dtype, int scale_dtype) {
  if (M <= 0 || N <= 0 || K <= 0 || (group != 32 && group != 64 && group != 128) || K % group != 0) return 0;
  const int sms = host::device_sms();
  return w4_route(sms ? sms : 148, M, N, K, group, scale_dtype == x_dtype + 1).need;
}
size_t b200q_w4a16_workspace_size(int64_t M, int64_t N, int64_t K) {
  size_t most = 0;
  for (int64_t group : {32, 64, 128})
    for (int scale_dtype : {B200Q_BIAS_BF16, B200Q_BIAS_F32})
      most = std::max(most, b200q_w4a16_workspace_bytes(M, N, K, group, B200Q_BF16, scale_dtype));
  return most;
}

int b200q_w4a16_linear(const void* x, int x_dtype, int64_t ldx, const uint8_t* w, int64_t ldw,
                       const void* scales, int scale_dtype, const uint8_t* zeros, int64_t group,
                       const void* bias, int bias_dtype, int act, void* out, int out_dtype,
                       int64_t ldo, int64_t M, int64_t N, int64_t K, void* workspace,
                       size_t workspace_bytes, void* stream) {
  if (M < 0 || N < 0 || K <= 0 || M > kIntMax || N > kIntMax || K > kIntMax ||
      (group != 32 && group != 64 && group != 128) || K % group != 0 ||
      (x_dtype != B200Q_BF16 && x_dtype != B200Q_F16) || scale_dtype < B200Q_BIAS_BF16 ||
      scale_dtype > B200Q_BIAS_F32 || bias_dtype < B200Q_BIAS_NONE || bias_dtype > B200Q_BIAS_F32 ||
      act < B200Q_ACT_NONE || act > B200Q_ACT_GELU_ERF || out_dtype < B200Q_BF16 ||
      out_dtype > B200Q_F32 || ldx < K || ldw < K / 2 || ldo < N || ldw % 16 != 0)
    return B200Q_ERR_INVALID;
  if (M == 0 || N == 0) return B200Q_OK;
  if (!x || !w || !scales || !out || !aligned(w, 16) || (bias_dtype != B200Q_BIAS_NONE && !bias))
    return B200Q_ERR_INVALID;
  const int sms = host::device_sms();
  if (!sms) return B200Q_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  EpiArgs ep{};
  ep.out = out;
  ep.ldo = ldo;
  ep.out_dtype = out_dtype;
  ep.bias = bias;
  ep.bias_dtype = bias_dtype;
  ep.act = act;
  ep.M = static_cast<int>(M);
  ep.N = static_cast<int>(N);
  const W4Route route = w4_route(sms, M, N, K, group, scale_dtype == x_dtype + 1);
  const size_t need = route.need;
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 256))) return B200Q_ERR_WORKSPACE;
  const bool x_vec = aligned(x, 16) && ldx % 8 == 0;
  if (route.kind == kW4Digits) {
    W4DigitArgs a{};
    a.x = x;
    a.ldx = ldx;
    a.w = w;
    a.ldw = ldw;
    a.scales = scales;
    a.zeros = zeros;
    a.M = static_cast<int>(M);
    a.N = static_cast<int>(N);
    a.K = static_cast<int>(K);
    a.x_vec = x_vec;
    a.tiles = static_cast<int>(cdiv(N, 16));
    return x_dtype == B200Q_F16 ? launch_digits<__half>(a, int(group), ep, route.wd, st)
                                : launch_digits<__nv_bfloat16>(a, int(group), ep, route.wd, st);
  }
  if (route.kind == kW4Tiles)
    return launch_w4_tile(route.tile, x, x_dtype, ldx, x_vec, w, ldw, scales, scale_dtype, zeros, group, M, N, K, ep,
                          static_cast<uint8_t*>(workspace), st);
  if (route.kind == kW4Slices) {
    W4SliceArgs a{};
    a.x = x;
    a.x_f16 = x_dtype == B200Q_F16;
    a.ldx = ldx;
    a.w = w;
    a.ldw = ldw;
    a.scales = scales;
    a.scale_dtype = scale_dtype;
    a.zeros = zeros;
    a.part = need ? static_cast<float*>(workspace) : nullptr;
    a.M = static_cast<int>(M);
    a.N = static_cast<int>(N);
    a.K = static_cast<int>(K);
    a.x_vec = x_vec;
    a.slices = route.ws.slices;
    a.parts = route.ws.parts;
    return launch_slice(a, int(group), ep, route.ws, st);
  }
  const W4Work o = w4_work(M, N, K);
  if (x_dtype == B200Q_F16 && !x_vec) return B200Q_ERR_INVALID;  // fp16 rows must be 16-byte aligned here
  uint8_t* base = static_cast<uint8_t*>(workspace);
  W4PrepareArgs a{};
  a.w = w;
  a.ldw = ldw;
  a.scales = scales;
  a.scale_dtype = scale_dtype;
  a.zeros = zeros;
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.log_g = group == 32 ? 5 : group == 64 ? 6 : 7;
  a.w16 = reinterpret_cast<__half*>(base);
  a.w_pow = reinterpret_cast<float*>(base + o.col);
  ep.col_scale = a.w_pow;
  ep.col_scale_vec = 1;
  int64_t blocks = cdiv(N, 8);
  if (x_dtype == B200Q_BF16) {
    a.x = static_cast<const __nv_bfloat16*>(x);
    a.ldx = ldx;
    a.M = static_cast<int>(M);
    a.x_vec = x_vec;
    a.x16 = reinterpret_cast<__half*>(base + o.x);
    a.x_pow = reinterpret_cast<float*>(base + o.row);
    ep.row_scale = a.x_pow;
    ep.row_scale_vec = 1;
    a.last = reinterpret_cast<float*>(base + o.last);
    ep.extra_scale = a.last;
    blocks += cdiv(M, 8);
    x = a.x16;
    ldx = K;
  }
  int s = launch(w4_prepare_kernel, dim3(static_cast<unsigned>(blocks)), 256, 0, st, a);
  if (s != B200Q_OK) return s;
  if (!w4_joins(N)) return host::gemm_f16_scaled(x, ldx, a.w16, K, M, N, K, ep, st);
  EpiArgs sums = ep;
  sums.out = base + o.out;
  sums.ldo = w4_join_ld(N);
  sums.out_dtype = kOutF32;
  sums.bias = nullptr;
  sums.bias_dtype = kBiasNone;
  sums.act = kActNone;
  s = host::gemm_f16_scaled(x, ldx, a.w16, K, M, N, K, sums, st);
  if (s != B200Q_OK) return s;
  ep.col_scale = ep.row_scale = ep.extra_scale = nullptr;
  return launch_join(static_cast<const float*>(sums.out), 1, sums.ldo, ep, st);
}

int b200q_block_norm(const void* x, int64_t ldx, const void* y, int64_t ldy, int dtype,
                     int post_kind, const void* post_w, int post_w_dtype, const void* gate,
                     int64_t ld_gate, float res_scale, int pre_kind, const void* w, int w_dtype,
                     const void* scale, int64_t ld_scale, const void* shift, int64_t ld_shift,
                     int mod_dtype, int64_t rows_per_mod, float eps, void* h, int64_t ldh,
                     void* out, int64_t ldo, int8_t* q, int64_t ldq, float* q_scale, int64_t rows,
                     int64_t D, void* stream) {
  if (rows < 0 || rows > kIntMax || D < 1 || D > B200Q_NORM_MAX_D || rows_per_mod < 1 ||
      (dtype != B200Q_BF16 && dtype != B200Q_F16) || post_kind < B200Q_NORM_NONE ||
      post_kind > B200Q_NORM_LAYER || pre_kind < B200Q_NORM_NONE || pre_kind > B200Q_NORM_LAYER ||
      ldx < D || (y && ldy < D) || (h && ldh < D) || (out && ldo < D) || (q && ldq < D) ||
      (q && !q_scale) || (out && q) || (!y && (h || gate || post_w)))
    return B200Q_ERR_INVALID;
  auto bad_dtype = [](const void* p, int t) { return p && (t < B200Q_BIAS_BF16 || t > B200Q_BIAS_F32); };
  if (bad_dtype(post_w, post_w_dtype) || bad_dtype(w, w_dtype) || bad_dtype(gate, mod_dtype) ||
      bad_dtype(scale, mod_dtype) || bad_dtype(shift, mod_dtype) || (gate && ld_gate < D) ||
      (scale && ld_scale < D) || (shift && ld_shift < D))
    return B200Q_ERR_INVALID;
  if (rows == 0) return B200Q_OK;
  if (!x || (!out && !q && !h)) return B200Q_ERR_INVALID;
  const int sms = host::device_sms();
  if (!sms) return B200Q_ERR_UNSUPPORTED;
  NormArgs a{};
  a.x = x; a.ldx = ldx; a.y = y; a.ldy = ldy;
  a.post_w = post_w; a.post_w_dtype = post_w_dtype;
  a.w = w; a.w_dtype = w_dtype;
  a.gate = gate; a.scale = scale; a.shift = shift;
  a.ld_gate = ld_gate; a.ld_scale = ld_scale; a.ld_shift = ld_shift;
  a.mod_dtype = mod_dtype;
  a.res_scale = res_scale; a.eps = eps;
  a.post_kind = post_kind; a.pre_kind = pre_kind;
  a.h = h; a.ldh = ldh; a.out = out; a.ldo = ldo; a.q = q; a.ldq = ldq; a.q_scale = q_scale;
  a.rows = static_cast<int>(rows); a.D = static_cast<int>(D);
  a.rows_per_mod = static_cast<int>(rows_per_mod < kIntMax ? rows_per_mod : kIntMax);
  // 16-byte vectors need every row of every operand on a 16-byte boundary
  auto ok = [](const void* p, int64_t ld) { return !p || (aligned(p, 16) && ld % 8 == 0); };
  const bool vec = D % 8 == 0 && ok(x, ldx) && ok(y, ldy) && ok(h, ldh) && ok(out, ldo) &&
                   ok(gate, ld_gate) && ok(scale, ld_scale) && ok(shift, ld_shift) &&
                   ok(post_w, 0) && ok(w, 0) && (!q || (aligned(q, 8) && ldq % 8 == 0));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto even = [](const void* p, int64_t ld, size_t bytes) { return !p || (aligned(p, bytes) && ld % 2 == 0); };
  const bool pairs = D % 2 == 0 && even(x, ldx, 4) && even(y, ldy, 4) && even(h, ldh, 4) && even(out, ldo, 4) &&
                     even(q, ldq, 2);
  return dtype == B200Q_F16 ? launch_norm<kBiasF16>(a, vec, pairs, sms, st)
                            : launch_norm<kBiasBF16>(a, vec, pairs, sms, st);
}

int b200q_kv8_append(const void* k, const void* v, int dtype, int64_t B, int64_t S,
                     const int64_t* k_strides, const int64_t* v_strides, int8_t* k_codes,
                     int8_t* v_codes, float* k_scale, float* v_scale, int64_t pages, int64_t heads,
                     int64_t block, int64_t D, const int32_t* table, int64_t ld_table,
                     int64_t max_blocks, const int32_t* start, const int32_t* counts,
                     void* stream) {
  Kv8AppendArgs a{};
  if (B < 0 || B > 32767 || S < 0 || S > kIntMax / 2 || (dtype != B200Q_BF16 && dtype != B200Q_F16) ||
      !k_strides || !v_strides ||
      !make_cache(&a.c, k_codes, v_codes, k_scale, v_scale, pages, heads, block, D, table, ld_table,
                  max_blocks))
    return B200Q_ERR_INVALID;
  if (B == 0 || S == 0) return B200Q_OK;
  if (!k || !v || !start || !aligned(k, 16) || !aligned(v, 16)) return B200Q_ERR_INVALID;
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0) return B200Q_ERR_INVALID;
  if (!host::device_sms()) return B200Q_ERR_UNSUPPORTED;
  a.k = k; a.v = v;
  a.kb = k_strides[0]; a.kh = k_strides[1]; a.kt = k_strides[2];
  a.vb = v_strides[0]; a.vh = v_strides[1]; a.vt = v_strides[2];
  a.start = start; a.counts = counts;
  a.B = static_cast<int>(B); a.S = static_cast<int>(S);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == B200Q_F16 ? launch_append<__half>(a, st) : launch_append<__nv_bfloat16>(a, st);
}

int b200q_kv8_gather(const int8_t* k_codes, const int8_t* v_codes, const float* k_scale,
                     const float* v_scale, int64_t pages, int64_t heads, int64_t block, int64_t D,
                     const int32_t* table, int64_t ld_table, int64_t max_blocks,
                     const int32_t* first, const int32_t* counts, void* k, void* v, int out_dtype,
                     int64_t B, int64_t S, void* stream) {
  Kv8GatherArgs a{};
  if (B < 0 || B > 32767 || S < 0 || S > kIntMax / 2 || out_dtype < B200Q_BF16 || out_dtype > B200Q_F32 ||
      !make_cache(&a.c, const_cast<int8_t*>(k_codes), const_cast<int8_t*>(v_codes),
                  const_cast<float*>(k_scale), const_cast<float*>(v_scale), pages, heads, block, D,
                  table, ld_table, max_blocks))
    return B200Q_ERR_INVALID;
  if (B == 0 || S == 0) return B200Q_OK;
  if (!k || !v || !first || !counts || !aligned(k, 16) || !aligned(v, 16)) return B200Q_ERR_INVALID;
  if (!host::device_sms()) return B200Q_ERR_UNSUPPORTED;
  a.k = k; a.v = v; a.out_dtype = out_dtype;
  a.first = first; a.counts = counts;
  a.B = static_cast<int>(B); a.S = static_cast<int>(S);
  const dim3 grid(static_cast<unsigned>(cdiv(S * (D / 8), kKvThreads * kGatherVecs)), static_cast<unsigned>(heads),
                  static_cast<unsigned>(2 * B));
  return launch(kv8_gather_kernel, grid, kKvThreads, 0, static_cast<cudaStream_t>(stream), a);
}

size_t b200q_kv8_attention_workspace_size(int64_t B, int64_t Hq, int64_t heads, int64_t Tq,
                                          int64_t D, int64_t max_len) {
  const int sms = host::device_sms();
  if (!sms || !attn_dims(B, Hq, heads, Tq) || B * Tq == 0) return 0;
  return attn_work_bytes(attn_splits(sms, B, Hq, heads, Tq, max_len), B * Hq * Tq, D);
}

int b200q_kv8_attention(const void* q, int dtype, int64_t B, int64_t Hq, int64_t Tq,
                        const int64_t* q_strides, const int8_t* k_codes, const int8_t* v_codes,
                        const float* k_scale, const float* v_scale, int64_t pages, int64_t heads,
                        int64_t block, int64_t D, const int32_t* table, int64_t ld_table,
                        int64_t max_blocks, const int32_t* lens, int64_t max_len, int causal,
                        float softmax_scale, void* out, const int64_t* out_strides, float* lse,
                        void* workspace, size_t workspace_bytes, void* stream) {
  Kv8AttnArgs a{};
  if ((dtype != B200Q_BF16 && dtype != B200Q_F16) || !attn_dims(B, Hq, heads, Tq) || !q_strides ||
      !out_strides || max_len < 0 ||
      !make_cache(&a.c, const_cast<int8_t*>(k_codes), const_cast<int8_t*>(v_codes),
                  const_cast<float*>(k_scale), const_cast<float*>(v_scale), pages, heads, block, D,
                  table, ld_table, max_blocks))
    return B200Q_ERR_INVALID;
  if (B == 0 || Tq == 0) return B200Q_OK;
  if (!q || !lens || !out || !lse || !aligned(q, 16) || !aligned(out, 16)) return B200Q_ERR_INVALID;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8 != 0 || out_strides[i] % 8 != 0) return B200Q_ERR_INVALID;
  const int sms = host::device_sms();
  if (!sms) return B200Q_ERR_UNSUPPORTED;
  const int64_t rows = B * Hq * Tq;
  const int splits = attn_splits(sms, B, Hq, heads, Tq, max_len);
  const size_t need = attn_work_bytes(splits, rows, D);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return B200Q_ERR_WORKSPACE;
  a.q = q; a.q_f16 = dtype == B200Q_F16;
  a.qb = q_strides[0]; a.qh = q_strides[1]; a.qt = q_strides[2];
  a.out = out;
  a.ob = out_strides[0]; a.oh = out_strides[1]; a.ot = out_strides[2];
  a.lse = lse;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + (need ? size_t(splits) * rows * D : 0);
  a.lens = lens;
  a.B = static_cast<int>(B); a.Hq = static_cast<int>(Hq); a.G = static_cast<int>(Hq / heads);
  a.Tq = static_cast<int>(Tq); a.causal = causal != 0;
  a.splits = splits;
  // ranked by one warp's lanes; where all CTAs start at once the order is nothing
  a.longest_first = B > 1 && B <= 32 && B * heads * cdiv(a.G * Tq, attn_row_tile(a.G * Tq)) * splits > sms;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t tiles = heads * cdiv(a.G * Tq, attn_row_tile(a.G * Tq));  // heads (<= 65535) up to 16 rows
  if (tiles * splits > kIntMax) return B200Q_ERR_UNSUPPORTED;
  const dim3 grid = a.G * Tq > 16 ? dim3(static_cast<unsigned>(tiles * splits), 1, static_cast<unsigned>(B))
                                  : dim3(static_cast<unsigned>(splits), static_cast<unsigned>(tiles), static_cast<unsigned>(B));
  // the pool as rows of D bytes; a page's rows of one head are contiguous
  const int64_t pool_rows = pages * heads * block;
  const uint32_t box = static_cast<uint32_t>(block < kAttnBox ? block : kAttnBox);
  const CUtensorMapSwizzle sw = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  CUtensorMap tk, tv;
  if (!host::tmap_u8(&tk, k_codes, D, pool_rows, D, static_cast<uint32_t>(D), box, sw) ||
      !host::tmap_u8(&tv, v_codes, D, pool_rows, D, static_cast<uint32_t>(D), box, sw))
    return B200Q_ERR_CUDA;
  int s;
  // up to 8 rows a head: integer q.K and transposed P V (see kv8_attn8_kernel); more
  // than 16: 128-row tiles on tcgen05
  if (a.G * Tq > kPfRows) {
    s = D == 128 ? launch(kv8_prefill_kernel<128, 2>, grid, pf_threads(2), pf_smem_bytes<128, 2>(), st, tk, tv, a)
                 : launch(kv8_prefill_kernel<64, 2>, grid, pf_threads(2), pf_smem_bytes<64, 2>(), st, tk, tv, a);
  } else if (a.G * Tq > 16) {
    s = D == 128 ? launch(kv8_prefill_kernel<128, 1>, grid, pf_threads(1), pf_smem_bytes<128, 1>(), st, tk, tv, a)
                 : launch(kv8_prefill_kernel<64, 1>, grid, pf_threads(1), pf_smem_bytes<64, 1>(), st, tk, tv, a);
  } else if (a.G * Tq <= 8) {
    s = D == 128 ? launch(kv8_attn8_kernel<128>, grid, kAttnThreads, attn_smem_bytes<128>(), st, tk, tv, a)
                 : launch(kv8_attn8_kernel<64>, grid, kAttnThreads, attn_smem_bytes<64>(), st, tk, tv, a);
  } else {
    s = D == 128 ? launch(kv8_attn_kernel<128>, grid, kAttnThreads, attn_smem_bytes<128>(), st, tk, tv, a)
                 : launch(kv8_attn_kernel<64>, grid, kAttnThreads, attn_smem_bytes<64>(), st, tk, tv, a);
  }
  if (s != B200Q_OK || !need) return s;
  if (splits <= 8) {
    const dim3 few(static_cast<unsigned>(cdiv(rows, 8)));
    return D == 128 ? launch(kv8_attn_join_few_kernel<128>, few, 256, 0, st, a)
                    : launch(kv8_attn_join_few_kernel<64>, few, 256, 0, st, a);
  }
  const dim3 jgrid(static_cast<unsigned>(rows));
  return D == 128 ? launch(kv8_attn_join_kernel<128>, jgrid, kJoinWarps * 32, 0, st, a)
                  : launch(kv8_attn_join_kernel<64>, jgrid, kJoinWarps * 32, 0, st, a);
}

}  // extern "C"
