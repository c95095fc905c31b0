// Product of 16-bit or 8-bit operands on the 5th-generation tensor cores with a fused epilogue:
//
//   out[m,n] = act(row_scale[m] * col_scale[n] * sum_k A[m,k] * B[n,k] + bias[n]) + residual[m,n]
//
// fp32 accumulation in tensor memory, fp32 epilogue, one rounding.  Persistent and warp-specialised:
//   warp 0      TMA producer: a stage is 128 bytes along the reduction axis of both operands
//   warp 1      tensor-memory allocation and single-thread tcgen05.mma issue
//   warps 2-9   epilogue: two warps per 32 rows, alternate units of 32 rows x 128 bytes of output
// The accumulator is double buffered in tensor memory, so the epilogue of a tile runs under the main
// loop of the next one.  A lane of the epilogue owns a row: it reads its sums from tensor memory, adds
// bias, applies the activation, and writes the rounded row piece into a swizzled 4 KB block of shared
// memory that TMA stores as whole 128-byte lines (stores straight from registers, 32 or 64 bytes a
// row, took 2 to 4 us per 64 KB and SM and were the kernel's bound).  The residual arrives in
// the same block by TMA before the lane replaces it by the result.
//
// kPair: two CTAs of a cluster (the two SMs of a TPC) work on one 256 x 256 tile with
// cta_group::2 MMAs.  Each holds its own 128 rows of A and half of B in shared memory, so a
// multiply-add reads 2/3 of the shared-memory bytes that a 128 x 128 tile of one CTA reads per operand
// row, and only half of B is fetched per CTA.  The even CTA issues the MMAs for both.
//
// Operands whose reduction axis is the slow one in memory (the weights in the input's gradient, both
// operands in the weights' gradient) are loaded as MN-major tiles: boxes of 64 columns x 64
// reduction rows, no transposed copies.
//
// Measured on a B200 (cuBLAS, plain product, beside it): 8192 x 8192 x 8192 bf16 693 us, 1586 TFLOP/s
// (1752); 8192 x 2048 -> 8192 181 us, 1517 (1608), with gelu, residual and stored z 246 us; 16384 x
// 1024 -> 1024 37 us, 932 (860); 8192 x 8192 -> 4096 e4m3 198 us, 2.8 PFLOP/s.  Tensor pipe active
// 87 % in the input's gradient; a stage of the 256 x 256 pair tile moves 128 bytes a cycle through shared
// memory, so operand traffic and MMAs are balanced, and long runs meet the power limit.
//
// Every mbarrier wait is bounded in time: on expiry the CTA raises a flag that ends all its loops,
// sets the status word, gives its copies in flight a bounded time to land, frees its tensor memory
// and returns.
#include <cuda.h>
#include <stdio.h>
#include "activation.cuh"
#include "common.cuh"
#include "dtypes.cuh"
#include "linear_epilogue.cuh"
#include "tc_ptx.cuh"

namespace gnn {
namespace {

constexpr int BM = 128;             // rows per CTA
constexpr int kATile = BM * kStageK;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 32 * (2 + kEpiWarps);
constexpr int kMaxStages = 7;
constexpr int kNumBars = 2 * kMaxStages + 4 + kEpiWarps;
constexpr int kBarBytes = (8 * kNumBars + 16 + 127) / 128 * 128;
constexpr int kUnitBytes = 32 * 128;                // 32 rows x 128 bytes of output

template <int BN, bool PAIR>
struct Geom {
  static constexpr int kBRows = PAIR ? BN / 2 : BN;  // B rows in this CTA's shared memory
  static constexpr int kStageBytes = kATile + kBRows * kStageK;
  static constexpr int kTmemCols = 2 * BN;
};

struct Params {
  int M, N;
  int total_kb, kb_per_split;       // stages along the reduction axis
  int tiles_m, tiles_n, num_tiles;  // num_tiles = tiles_m * tiles_n * splits
  int a_mn, b_mn;
  int k_elems;                      // elements of a stage along the reduction axis
  uint32_t idesc;                   // instruction descriptor without the N field
  float* planes;                    // splits > 1: fp32 partial planes [splits][M][N]
  int stages;
  int tma_out;                      // out, z, residual (or the planes) have rows that TMA can address
  LinearEpilogue ep;
  int* status;
};

struct TileCoord {
  int m0, n0, kb_begin, num_kb, z;
};
// Tiles in bands of 8 row tiles, column by column inside a band: the CTAs that run at the same time
// share rows of A and of B through L2.
template <int TM, int TN>
__device__ __forceinline__ TileCoord decode_tile(const Params& p, int tile) {
  constexpr int kBand = 8;
  const int per_split = p.tiles_m * p.tiles_n;
  TileCoord t;
  t.z = tile / per_split;
  const int i = tile - t.z * per_split;
  const int band = i / (kBand * p.tiles_n);
  const int high = min(kBand, p.tiles_m - band * kBand);
  const int j = i - band * kBand * p.tiles_n;
  const int nt = j / high;
  t.m0 = (band * kBand + j - nt * high) * TM;
  t.n0 = nt * TN;
  t.kb_begin = t.z * p.kb_per_split;
  t.num_kb = max(0, min(p.kb_per_split, p.total_kb - t.kb_begin));
  return t;
}

// Eight columns of kRows rows at a time: residual, bias and scales are requested early, and the
// activation is one branch for all 8 * kRows values.
template <class T, int kRows>
struct Finish8 {
  static constexpr int V = 16 / (int)sizeof(T), Q = 8 / V;
  Pack<T, V> residual[kRows][Q];
  float bias[8], scale[8], row_scale[kRows];

  // rows row0 + step * i; in(i): the row exists
  template <class In>
  __device__ __forceinline__ void request(const LinearEpilogue& ep, int64_t row0, int step, int col, int N, In&& in) {
    if (ep.residual) {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (in(i)) {
          const T* const at = static_cast<const T*>(ep.residual) + (row0 + step * i) * N + col;
#pragma unroll
          for (int q = 0; q < Q; ++q) residual[i][q] = load_pack(reinterpret_cast<const Pack<T, V>*>(at) + q);
        }
    }
  }
  template <class In>
  __device__ __forceinline__ void columns(const LinearEpilogue& ep, int64_t row0, int step, int col, bool ok, In&& in) {
#pragma unroll
    for (int j = 0; j < 8; ++j) bias[j] = 0.f;
    if (ep.bias && ok) load8(static_cast<const T*>(ep.bias) + col, bias);
    if (ep.col_scale) {
      if (ok) load8(ep.col_scale + col, scale);
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (in(i)) row_scale[i] = __ldg(ep.row_scale + row0 + step * i);
    }
  }
  template <class In>
  __device__ __forceinline__ void finish(const LinearEpilogue& ep, int64_t row0, int step, int col, int N, In&& in,
                                         float (&v)[kRows * 8]) {
    if (ep.col_scale) {
#pragma unroll
      for (int i = 0; i < kRows * 8; ++i) v[i] *= row_scale[i / 8] * scale[i % 8];
    }
#pragma unroll
    for (int i = 0; i < kRows * 8; ++i) v[i] += bias[i % 8];
    if (ep.z) {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (in(i)) store_row(static_cast<T*>(ep.z) + (row0 + step * i) * N + col, v, i);
    }
    apply_act<sizeof(T) == 4>(v, ep.act, ep.slope);
    if (ep.residual) {
#pragma unroll
      for (int i = 0; i < kRows * 8; ++i) v[i] += to_f32(residual[i / 8][i % 8 / V].v[i % V]);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (in(i)) store_row(static_cast<T*>(ep.out) + (row0 + step * i) * N + col, v, i);
  }
  __device__ __forceinline__ static void store_row(T* at, const float (&v)[kRows * 8], int i) {
    float o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = v[i * 8 + j];
    store8(at, o);
  }
};

// Sixteen consecutive columns of one output row in a unit's block: the 16-byte units of row r are
// exchanged by r mod 8 (the pattern of TMA's 128-byte swizzle), so 8 lanes on 8 rows meet 8 banks.
template <class O>
struct RowPiece {
  static constexpr int V = 16 / (int)sizeof(O), kUnits = 16 / V;  // 16-byte units of 16 columns
  __device__ __forceinline__ static uint8_t* at(uint8_t* block, int lane, int piece, int u) {
    return block + lane * 128 + (((piece * kUnits + u) ^ (lane & 7)) << 4);
  }
  __device__ __forceinline__ static void put(uint8_t* block, int lane, int piece, const float (&v)[16]) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      Pack<O, V> o;
      o.round_from(v + u * V);
      store_pack(reinterpret_cast<Pack<O, V>*>(at(block, lane, piece, u)), o);
    }
  }
  __device__ __forceinline__ static void add(uint8_t* block, int lane, int piece, float (&v)[16]) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const Pack<O, V> o = load_pack(reinterpret_cast<const Pack<O, V>*>(at(block, lane, piece, u)));
#pragma unroll
      for (int j = 0; j < V; ++j) v[u * V + j] += to_f32(o.v[j]);
    }
  }
};

template <int BN, bool PAIR, bool FP8, class T>
__global__ void __launch_bounds__(kThreads, 1)
linear_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_z,
                 const __grid_constant__ CUtensorMap map_res, const Params p) {
  using G = Geom<BN, PAIR>;
  constexpr int TM = PAIR ? 2 * BM : BM;
  extern __shared__ uint8_t smem_raw[];
  const int stages = p.stages;
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;  // swizzle atoms need 1024-byte alignment
  uint8_t* const base_ptr = smem_raw + (base - raw_addr);
  const uint32_t bar_off = stages * G::kStageBytes + kEpiWarps * kUnitBytes * (p.ep.z ? 2 : 1);
  const uint32_t bars = base + bar_off;
  auto full_bar = [&](int s) { return bars + 8u * s; };                             // TMA -> MMA
  auto empty_bar = [&](int s) { return bars + 8u * (kMaxStages + s); };             // MMA -> TMA
  auto acc_full_bar = [&](int b) { return bars + 8u * (2 * kMaxStages + b); };      // MMA -> epilogue
  auto acc_empty_bar = [&](int b) { return bars + 8u * (2 * kMaxStages + 2 + b); }; // epilogue -> MMA
  auto res_bar = [&](int w) { return bars + 8u * (2 * kMaxStages + 4 + w); };       // residual -> its epilogue warp
  const uint32_t tmem_slot = bars + 8u * kNumBars;

  __shared__ volatile int s_failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  const int unit = PAIR ? blockIdx.x >> 1 : blockIdx.x, units = PAIR ? gridDim.x >> 1 : gridDim.x;

  if (threadIdx.x == 0) {
    s_failed = 0;
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full_bar(b), 1);
      mbar_init(acc_empty_bar(b), kEpiWarps * (PAIR ? 2 : 1));
    }
    for (int w = 0; w < kEpiWarps; ++w) mbar_init(res_bar(w), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(G::kTmemCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(G::kTmemCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the other CTA's barriers exist
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(base_ptr + bar_off + 8 * kNumBars);

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    if (lane == 0) {
      int s = 0;
      uint32_t phase = 1;  // a fresh barrier lets the wait for parity 1 through
      for (int tile = unit; tile < p.num_tiles && !s_failed; tile += units) {
        const TileCoord t = decode_tile<TM, BN>(p, tile);
        const int a_row = t.m0 + (int)rank * BM, b_row = t.n0 + (int)rank * G::kBRows;
        for (int kb = 0; kb < t.num_kb; ++kb) {
          if (!mbar_wait(empty_bar(s), phase, &s_failed)) { s_failed = 1; break; }
          const uint32_t st = base + s * G::kStageBytes;
          const int k0 = (t.kb_begin + kb) * p.k_elems;
          if (rank == 0) mbar_expect_tx(full_bar(s), G::kStageBytes * (PAIR ? 2 : 1));
          if (p.a_mn) {
#pragma unroll
            for (int g = 0; g < BM / 64; ++g) tma_load<PAIR>(st + g * 8192, &map_a, a_row + 64 * g, k0, full_bar(s));
          } else {
            tma_load<PAIR>(st, &map_a, k0, a_row, full_bar(s));
          }
          if (p.b_mn) {
#pragma unroll
            for (int g = 0; g < G::kBRows / 64; ++g)
              tma_load<PAIR>(st + kATile + g * 8192, &map_b, b_row + 64 * g, k0, full_bar(s));
          } else {
            tma_load<PAIR>(st + kATile, &map_b, k0, b_row, full_bar(s));
          }
          if (++s == stages) { s = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issue
    if (lane == 0 && rank == 0) {
      const uint64_t a_step = p.a_mn ? (2048 >> 4) : (32 >> 4);  // descriptor advance per K slice
      const uint64_t b_step = p.b_mn ? (2048 >> 4) : (32 >> 4);
      const uint32_t idesc = p.idesc | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(TM >> 4) << 24);
      int s = 0;
      uint32_t phase = 0, count = 0;
      bool ok = true;
      for (int tile = unit; tile < p.num_tiles && ok && !s_failed; tile += units, ++count) {
        const TileCoord t = decode_tile<TM, BN>(p, tile);
        const int buf = count & 1;
        if (!mbar_wait(acc_empty_bar(buf), ((count >> 1) & 1) ^ 1, &s_failed)) { s_failed = 1; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t acc = tmem_base + (uint32_t)(buf * BN);
        for (int kb = 0; kb < t.num_kb; ++kb) {
          if (!mbar_wait(full_bar(s), phase, &s_failed)) { s_failed = 1; ok = false; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t st = base + s * G::kStageBytes;
          const uint64_t da = operand_desc(st, p.a_mn), db = operand_desc(st + kATile, p.b_mn);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma<PAIR, FP8>(acc, da + a_step * k, db + b_step * k, idesc, (kb | k) != 0);
          umma_commit<PAIR>(empty_bar(s));  // the stage is free once these MMAs have read it
          if (++s == stages) { s = 0; phase ^= 1; }
        }
        if (ok) umma_commit<PAIR>(acc_full_bar(buf));
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue
    const int w = warp - 2;
    const int lg = warp & 3;   // this warp may touch tensor-memory lanes [32*lg, 32*lg + 32)
    const int part = w >> 2;   // units part, part + 2, ... of its rows
    uint8_t* const block = base_ptr + stages * G::kStageBytes + w * kUnitBytes;
    uint8_t* const z_block = block + kEpiWarps * kUnitBytes;
    const bool with_res = p.tma_out && p.ep.residual && !p.planes;
    uint32_t res_phase = 0, count = 0;
    bool res_due = false;  // a residual copy is under way (lane 0's view)

    for (int tile = unit; tile < p.num_tiles && !s_failed; tile += units, ++count) {
      const TileCoord t = decode_tile<TM, BN>(p, tile);
      const int buf = count & 1;
      const int top = t.m0 + (int)rank * BM + lg * 32;  // first row of this warp
      const int row = top + lane;

      // The units of this warp's rows, of output type O (fp32 for planes).
      auto run = [&](auto tag, auto is_plane) -> bool {
        using O = decltype(tag);
        using Piece = RowPiece<O>;
        constexpr bool kPlanes = decltype(is_plane)::value;
        constexpr int kCols = 128 / (int)sizeof(O), kPieces = kCols / 16;
        auto want_residual = [&](int col0) {  // the block is free: its last store has been read
          if (lane == 0) {
            mbar_expect_tx(res_bar(w), kUnitBytes);
            tma_load_local(base + stages * G::kStageBytes + w * kUnitBytes, &map_res, col0, top, res_bar(w));
            res_due = true;
          }
        };
        const bool mine = top < p.M && part * kCols < BN && t.n0 + part * kCols < p.N;
        if (mine && !kPlanes && with_res) {  // the first residual is under way while the product finishes
          if (lane == 0) bulk_wait_read();
          want_residual(t.n0 + part * kCols);
        }
        const float rs = !kPlanes && p.ep.col_scale && row < p.M ? __ldg(p.ep.row_scale + row) : 1.f;
        if (!warp_wait(acc_full_bar(buf), (count >> 1) & 1, &s_failed)) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (!mine) return true;
        const uint32_t lane_base = tmem_base + ((uint32_t)(lg * 32) << 16) + (uint32_t)(buf * BN);
#pragma unroll 1
        for (int u = part; u < BN / kCols; u += 2) {
          const int col0 = t.n0 + u * kCols;
          if (col0 >= p.N) break;
          if (!kPlanes && with_res) {
            if (!warp_wait(res_bar(w), res_phase, &s_failed)) return false;
            res_phase ^= 1;
            if (lane == 0) res_due = false;
          } else {
            if (lane == 0) bulk_wait_read();
            __syncwarp();
          }
#pragma unroll 1
          for (int q = 0; q < kPieces; ++q) {
            uint32_t r[16];
            tmem_load16(lane_base + (uint32_t)(u * kCols + q * 16), r);
            const int col = col0 + q * 16;
            float v[16], b[16];
            const bool in = col + 16 <= p.N;
            if (!kPlanes && p.ep.bias) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float f[8];
                if (in) {
                  load8(static_cast<const T*>(p.ep.bias) + col + 8 * h, f);
                } else {
#pragma unroll
                  for (int j = 0; j < 8; ++j)
                    f[j] = col + 8 * h + j < p.N ? to_f32(static_cast<const T*>(p.ep.bias)[col + 8 * h + j]) : 0.f;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) b[8 * h + j] = f[j];
              }
            }
            tmem_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = t.num_kb ? __uint_as_float(r[j]) : 0.f;  // an empty range adds nothing
            if constexpr (!kPlanes) {
              if constexpr (FP8) {
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] *= rs * (in || col + j < p.N ? __ldg(p.ep.col_scale + col + j) : 0.f);
              }
              if (p.ep.bias) {
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] += b[j];
              }
              if (p.ep.z) Piece::put(z_block, lane, q, v);
              apply_act<sizeof(O) == 4>(v, p.ep.act, p.ep.slope);
              if (with_res) Piece::add(block, lane, q, v);
            }
            Piece::put(block, lane, q, v);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            const uint32_t src = base + stages * G::kStageBytes + w * kUnitBytes;
            if constexpr (kPlanes) {
              tma_store_3d(&map_out, src, col0, top, t.z);
            } else {
              tma_store_2d(&map_out, src, col0, top);
              if (p.ep.z) tma_store_2d(&map_z, src + kEpiWarps * kUnitBytes, col0, top);
            }
            bulk_commit();
          }
          if (!kPlanes && with_res && u + 2 < BN / kCols && col0 + 2 * kCols < p.N) {
            if (lane == 0) bulk_wait_read();
            want_residual(col0 + 2 * kCols);
          }
        }
        return true;
      };

      if (p.tma_out) {
        const bool ok = p.planes ? run(float{}, std::true_type{}) : run(T{}, std::false_type{});
        if (!ok) { s_failed = 1; break; }
      } else {
        // rows that are not whole 16-byte units: 32 x 32 blocks through shared memory, then a column per
        // lane, whose residual is requested before the sums are fetched
        if (!warp_wait(acc_full_bar(buf), (count >> 1) & 1, &s_failed)) { s_failed = 1; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const float my_rs = FP8 && !p.planes && row < p.M ? __ldg(p.ep.row_scale + row) : 1.f;
        const int rows = min(32, p.M - top);
#pragma unroll 1
        for (int c = part; c < BN / 32; c += 2) {
          const int col0 = t.n0 + c * 32, col = col0 + lane;
          if (col0 >= p.N || rows <= 0) break;
          const bool in = col < p.N;
          const int64_t at = (int64_t)top * p.N + col;
          const bool with_r = p.ep.residual && !p.planes;
          T res[32];
          if (with_r) {
            const T* const src = static_cast<const T*>(p.ep.residual) + (in ? at : 0);
#pragma unroll
            for (int i = 0; i < 32; ++i) res[i] = src[(int64_t)(in ? min(i, rows - 1) : 0) * p.N];
          }
          const float bias = in && p.ep.bias && !p.planes ? to_f32(static_cast<const T*>(p.ep.bias)[col]) : 0.f;
          const float cs = FP8 && in && !p.planes ? __ldg(p.ep.col_scale + col) : 1.f;
#pragma unroll 1
          for (int q = 0; q < 2; ++q) {
            uint32_t r[16];
            tmem_load16(tmem_base + ((uint32_t)(lg * 32) << 16) + (uint32_t)(buf * BN + c * 32 + q * 16), r);
            tmem_wait();
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = t.num_kb ? __uint_as_float(r[j]) : 0.f;
            RowPiece<float>::put(block, lane, q, v);
          }
          __syncwarp();
#pragma unroll
          for (int r0 = 0; r0 < 32; r0 += 8) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              v[i] = *reinterpret_cast<const float*>(block + (r0 + i) * 128 + (((lane >> 2) ^ i) << 4) + (lane & 3) * 4);
              if constexpr (FP8) v[i] *= __shfl_sync(kFull, my_rs, r0 + i) * cs;
              v[i] += bias;
            }
            if (p.planes) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (in && r0 + i < rows) p.planes[(size_t)t.z * p.M * p.N + at + (int64_t)(r0 + i) * p.N] = v[i];
              continue;
            }
            if (p.ep.z) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (in && r0 + i < rows) static_cast<T*>(p.ep.z)[at + (int64_t)(r0 + i) * p.N] = from_f32<T>(v[i]);
            }
            apply_act<sizeof(T) == 4>(v, p.ep.act, p.ep.slope);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (with_r) v[i] += to_f32(res[r0 + i]);
              if (in && r0 + i < rows) static_cast<T*>(p.ep.out)[at + (int64_t)(r0 + i) * p.N] = from_f32<T>(v[i]);
            }
          }
          __syncwarp();  // the block is rewritten by the next chunk
        }
      }
      // the buffer may be overwritten once every epilogue warp has read it
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) mbar_arrive_at(acc_empty_bar(buf), 0);
        else mbar_arrive(acc_empty_bar(buf));
      }
    }
    if (lane == 0) {
      bulk_wait_read();  // the stores have left shared memory
      if (s_failed && res_due) mbar_wait(res_bar(w), res_phase, nullptr, kDrainCycles);
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (s_failed) {
    // something expired: give the copies still in flight a bounded time to land before the shared
    // memory is released
    if (threadIdx.x == 0) {
      *p.status = 1;
      for (int s = 0; s < stages; ++s) {
        mbar_wait(full_bar(s), 0, nullptr, kDrainCycles);
        mbar_wait(full_bar(s), 1, nullptr, kDrainCycles);
      }
    }
    __syncthreads();
  }
  if constexpr (PAIR) cluster_sync();  // neither CTA leaves while the other may still signal it
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if constexpr (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(G::kTmemCols) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(G::kTmemCols) : "memory");
  }
}

// Sums the fp32 planes of a split product in order and finishes the row pieces.
template <class T>
__global__ void __launch_bounds__(256) split_epilogue_kernel(const float* __restrict__ planes, int parts, int64_t M, int N, int octs,
                                                             int vec_ok, const LinearEpilogue ep) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t row = i / octs;
  if (row >= M) return;
  const int col = (int)(i - row * octs) * 8;
  const size_t plane = (size_t)M * N;
  const float* const at = planes + row * N + col;
  if (vec_ok) {
    Finish8<T, 1> fin;
    auto in = [](int) { return true; };
    fin.request(ep, row, 0, col, N, in);
    fin.columns(ep, row, 0, col, true, in);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
#pragma unroll 4
    for (int z = 0; z < parts; ++z) {
      float f[8];
      load8(at + z * plane, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += f[j];
    }
    fin.finish(ep, row, 0, col, N, in, v);
  } else {
#pragma unroll 1
    for (int j = 0; j < 8 && col + j < N; ++j) {
      float v = 0.f;
#pragma unroll 4
      for (int z = 0; z < parts; ++z) v += at[z * plane + j];
      finish_one<T>(ep, row, col + j, N, v);
    }
  }
}

// Map over an output-shaped array [planes][M][N] with a box of 32 rows x 128 bytes.
bool encode_out(CUtensorMap* m, const void* ptr, int type, int64_t planes, int64_t M, int64_t N) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const int elt = dtype_bytes(type);
  const CUtensorMapDataType dt = type == GNN_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : type == GNN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  cuuint64_t dims[3] = {(cuuint64_t)N, (cuuint64_t)M, (cuuint64_t)(planes ? planes : 1)};
  cuuint64_t strides[2] = {(cuuint64_t)N * elt, (cuuint64_t)M * N * elt};
  cuuint32_t box[3] = {(cuuint32_t)(128 / elt), 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(m, dt, planes ? 3 : 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan {
  int bn, pair, splits;
  int64_t tiles_m, tiles_n;
};
constexpr int kSms = 148;

// Tile and split of the reduction axis for a shape: the candidate with the least estimated time.
// A stage costs its shared-memory traffic (every operand byte is written by TMA and read by the MMAs,
// 128 bytes a cycle) or its MMAs, whichever is more; a tile costs about kTileCycles on top that a wave
// cannot hide, a split a second pass over fp32 planes.
Plan plan_for(int64_t M, int64_t N, int64_t K, int in_type) {
  const int64_t kb = (K * (in_type == GNN_E4M3 ? 1 : 2) + kStageK - 1) / kStageK;
  struct { int bn, pair; double stage; } const shapes[] = {
      {256, 1, 512}, {128, 1, 384}, {128, 0, 512}, {64, 0, 384}};
  constexpr double kTileCycles = 5000, kSplitCycles = 6000, kPlaneBytesPerCycle = 3000;
  const int64_t least = (kb + max_chain(in_type) - 1) / max_chain(in_type);
  Plan best{};
  double best_cost = 0;
  for (const auto& c : shapes) {
    if (c.pair ? M <= BM : M > BM && N > 64) continue;  // a pair's second half would be empty; a pair reads less
    const int64_t tm = c.pair ? 2 * BM : BM, units = c.pair ? kSms / 2 : kSms;
    const int64_t tiles_m = (M + tm - 1) / tm, tiles_n = (N + c.bn - 1) / c.bn, tiles = tiles_m * tiles_n;
    for (int64_t s = 1; s <= 64; s *= 2) {
      if (s > 1 && (kb / s < 4 || tiles * s > 2 * units) && s > least) break;
      if (s < least && s * 2 <= 64) continue;
      const double waves = (double)((tiles * s + units - 1) / units), stages = (double)((kb + s - 1) / s);
      const double cost = waves * (stages * c.stage + kTileCycles) +
                          (s > 1 ? kSplitCycles + 8.0 * s * M * N / kPlaneBytesPerCycle : 0);
      if (best_cost == 0 || cost < best_cost) {
        best_cost = cost;
        best = Plan{c.bn, c.pair, (int)(s < least ? least : s), tiles_m, tiles_n};
      }
    }
  }
  return best;
}

struct Maps {
  CUtensorMap a, b, out, z, res;
};

template <int BN, bool PAIR, bool FP8, class T>
int launch_instance(const Maps& m, Params p, int grid, cudaStream_t stream) {
  using G = Geom<BN, PAIR>;
  auto kernel = linear_tc_kernel<BN, PAIR, FP8, T>;
  const int fixed = 1024 + kBarBytes + kEpiWarps * kUnitBytes * (p.ep.z ? 2 : 1);
  p.stages = (kSmemLimit - 64 - fixed) / G::kStageBytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  const int smem = fixed + p.stages * G::kStageBytes;
  static SmemGrant grant;
  grant.allow(kernel, kSmemLimit - 64);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR ? 2 : 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, m.a, m.b, m.out, m.z, m.res, p) == cudaSuccess ? 0 : 1;
}

template <bool FP8, class T>
int launch_shape(const Plan& pl, const Maps& m, const Params& p, int grid, cudaStream_t stream) {
  if (pl.pair && pl.bn == 256) return launch_instance<256, true, FP8, T>(m, p, grid, stream);
  if (pl.pair) return launch_instance<128, true, FP8, T>(m, p, grid, stream);
  if (pl.bn == 128) return launch_instance<128, false, FP8, T>(m, p, grid, stream);
  return launch_instance<64, false, FP8, T>(m, p, grid, stream);
}

// Whole 16-byte accesses of every array of the output's shape.
bool epilogue_vec_ok(const LinearEpilogue& ep, int64_t N, const float* planes) {
  const uintptr_t all = (uintptr_t)ep.out | (uintptr_t)ep.z | (uintptr_t)ep.residual | (uintptr_t)ep.bias |
                        (uintptr_t)ep.col_scale | (uintptr_t)planes;
  return N % 8 == 0 && all % 16 == 0;
}

}  // namespace

size_t linear_tc_workspace(int64_t M, int64_t N, int64_t K, int in_type) {
  const Plan p = plan_for(M, N, K, in_type);
  return p.splits > 1 ? (size_t)p.splits * M * N * sizeof(float) + 256 : 0;
}

int launch_split_epilogue(const float* planes, int parts, int64_t M, int64_t N, const LinearEpilogue& ep, cudaStream_t stream) {
  const int octs = (int)((N + 7) / 8);
  const int64_t grid = (M * octs + 255) / 256;
  const int vec = epilogue_vec_ok(ep, N, planes);
  if (ep.out_type == GNN_F32) split_epilogue_kernel<float><<<(unsigned)grid, 256, 0, stream>>>(planes, parts, M, (int)N, octs, vec, ep);
  else if (ep.out_type == GNN_BF16) split_epilogue_kernel<__nv_bfloat16><<<(unsigned)grid, 256, 0, stream>>>(planes, parts, M, (int)N, octs, vec, ep);
  else split_epilogue_kernel<__half><<<(unsigned)grid, 256, 0, stream>>>(planes, parts, M, (int)N, octs, vec, ep);
  return GNN_OK;
}

int launch_linear_tc(const TcOperand& a, const TcOperand& b, int in_type, int64_t M, int64_t N, int64_t K,
                     const LinearEpilogue& ep, void* workspace, size_t workspace_bytes, int* status, cudaStream_t stream,
                     const char* what) {
  const Plan pl = plan_for(M, N, K, in_type);
  char msg[200];
  if (pl.splits > 1 && (!workspace || workspace_bytes < linear_tc_workspace(M, N, K, in_type))) {
    snprintf(msg, sizeof msg, "%s: workspace too small", what);
    set_last_error(msg);
    return GNN_ERR_WORKSPACE;
  }
  const int64_t tiles = pl.tiles_m * pl.tiles_n * pl.splits;
  if (tiles > INT32_MAX) {
    snprintf(msg, sizeof msg, "%s: too many output tiles", what);
    set_last_error(msg);
    return GNN_ERR_LIMIT;
  }
  Maps m = {};
  float* const planes = pl.splits > 1 ? (float*)(((uintptr_t)workspace + 255) & ~(uintptr_t)255) : nullptr;
  // the epilogue goes through TMA where rows are a multiple of 16 bytes apart and start on such a boundary
  const uintptr_t arrays = planes ? (uintptr_t)planes
                                  : (uintptr_t)ep.out | (uintptr_t)ep.z | (uintptr_t)ep.residual | (uintptr_t)ep.bias;
  const bool tma_out = N * (planes ? 4 : dtype_bytes(ep.out_type)) % 16 == 0 && arrays % 16 == 0;
  bool encoded = encode_operand(&m.a, a, in_type, M, K, BM) && encode_operand(&m.b, b, in_type, N, K, pl.pair ? pl.bn / 2 : pl.bn);
  if (encoded && tma_out && planes) {
    encoded = encode_out(&m.out, planes, GNN_F32, pl.splits, M, N);
  } else if (encoded && tma_out) {
    encoded = encode_out(&m.out, ep.out, ep.out_type, 0, M, N);
    if (ep.z) encoded = encoded && encode_out(&m.z, ep.z, ep.out_type, 0, M, N);
    if (ep.residual) encoded = encoded && encode_out(&m.res, ep.residual, ep.out_type, 0, M, N);
  }
  if (!encoded) {
    snprintf(msg, sizeof msg, "%s: cuTensorMapEncodeTiled failed", what);
    set_last_error(msg);
    return GNN_ERR_CUDA;
  }
  const bool fp8 = in_type == GNN_E4M3;
  Params p = {};
  p.M = (int)M;
  p.N = (int)N;
  p.k_elems = fp8 ? kStageK : kStageK / 2;
  p.total_kb = (int)((K + p.k_elems - 1) / p.k_elems);
  p.kb_per_split = (p.total_kb + pl.splits - 1) / pl.splits;
  p.tiles_m = (int)pl.tiles_m;
  p.tiles_n = (int)pl.tiles_n;
  p.num_tiles = (int)tiles;
  p.a_mn = a.mn_major;
  p.b_mn = b.mn_major;
  // D = F32 (1 at bits 4-5), A / B type at bits 7-9 / 10-12 (kind f16: 0 half, 1 bfloat16; kind
  // f8f6f4: 0 e4m3), bit 15 / 16 = A / B is MN-major; N/8 and M/16 are added by the kernel
  const uint32_t type = in_type == GNN_BF16 ? 1u : 0u;
  p.idesc = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)a.mn_major << 15) | ((uint32_t)b.mn_major << 16);
  p.planes = planes;
  p.tma_out = tma_out;
  p.ep = ep;
  if (planes) p.ep.z = nullptr;  // the second kernel writes it
  p.status = status;
  const int64_t units = pl.pair ? kSms / 2 : kSms;
  const int grid = (int)(tiles < units ? tiles : units) * (pl.pair ? 2 : 1);
  int rc;
  if (!fp8) {  // 16-bit operands give results of their own type
    rc = ep.out_type == GNN_BF16 ? launch_shape<false, __nv_bfloat16>(pl, m, p, grid, stream)
                                 : launch_shape<false, __half>(pl, m, p, grid, stream);
  } else {
    rc = ep.out_type == GNN_F32    ? launch_shape<true, float>(pl, m, p, grid, stream)
         : ep.out_type == GNN_BF16 ? launch_shape<true, __nv_bfloat16>(pl, m, p, grid, stream)
                                   : launch_shape<true, __half>(pl, m, p, grid, stream);
  }
  if (rc == 0 && pl.splits > 1) launch_split_epilogue(p.planes, pl.splits, M, N, ep, stream);
  return check_launch(what);
}

}  // namespace gnn
