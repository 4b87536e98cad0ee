// C ABI of libpolylora_b200.so: argument checks, TMA tensor maps, launch
// configuration and dispatch between the tensor-core (bf16/fp16) and CUDA-core
// kernels.  One translation unit so the device status word is shared.
#include <cudaTypedefs.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <string>

#include "common.cuh"
#include "segments.cuh"
#include "sgmv_simt.cuh"
#include "sgmv_grid.cuh"
#include "host_rows.cuh"
#include "sgmv_stream.cuh"
#include "paged.cuh"
#include "logits.cuh"
#include "peft_pack.h"

using namespace plora;

// Scratch of plora_sgmv_a_fwd_noalloc: segment scratch + slot table for one
// batch, resident on every device that loads the library.  Host code must not
// use this symbol as a pointer; it is a host-side stand-in for the device
// array, whose address comes from cudaGetSymbolAddress below.
static __device__ __align__(256) unsigned char g_noalloc_scratch[PLORA_NOALLOC_SCRATCH_BYTES];

namespace {

thread_local std::string g_last_error;

int fail(int status, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return status;
}

int cuda_fail(cudaError_t e, const char* what) {
  return fail(PLORA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

#define PLORA_CUDA(call, what)             \
  do {                                     \
    cudaError_t _e = (call);               \
    if (_e != cudaSuccess) return cuda_fail(_e, what); \
  } while (0)

constexpr int kMaxDevices = 64;

// Shared-memory bytes of the per-slot table staged by the token-split kernels.
size_t tab_bytes(int32_t ns) { return (size_t)slot_tab_bytes(ns); }

struct DeviceInfo {
  int sm_count = 0;
  bool attrs_set = false;
};
DeviceInfo g_dev[kMaxDevices];
std::mutex g_dev_mu;

// Batches of at most this many tokens per SM run the slot-grid kernels
// (sgmv_grid.cuh): their slots have few tokens each, so giving every (slot,
// weight part) a CTA beats giving each CTA a share of the tokens (which makes
// every CTA stream the whole LoRA weights of each slot it touches).
std::atomic<int64_t> g_wsplit_tokens_per_sm{16};

// Rank-16 calls of many tokens run the stream kernels (sgmv_stream.cuh) when
// this is non-zero; 0 keeps them on the windowed mma kernels.  2 (the default)
// also runs plora_sgmv_shrink_expand as the fused stream kernel, 1 as the two.
std::atomic<int32_t> g_stream_kernels{2};

// A CTA's share of the token list must fit the stream kernels' shared-memory
// copy of its token ids.  Shares are cost-balanced (stream_share): one holds at
// most ceil((tokens + slot_cost * active slots) / SMs) + 1 tokens.
bool stream_share_ok(int64_t num_tokens, int64_t num_slots, int64_t slot_cost, const DeviceInfo* di) {
  const int64_t virt = num_tokens + slot_cost * num_slots;
  return (virt + di->sm_count - 1) / di->sm_count + 1 <= kStreamMaxShare;
}
bool stream_shrink_ok(int64_t R, int64_t K, int64_t num_tokens, int64_t num_slots, const DeviceInfo* di) {
  return g_stream_kernels.load(std::memory_order_relaxed) != 0 && R == kStreamRank && K % 512 == 0 &&
         K <= kStreamMaxDim && stream_share_ok(num_tokens, num_slots, kShrinkSlotCost, di);
}
bool stream_expand_ok(int64_t R, int64_t N, int64_t num_tokens, int64_t num_slots, const DeviceInfo* di) {
  return g_stream_kernels.load(std::memory_order_relaxed) != 0 && R == kStreamRank && N % 512 == 0 &&
         N <= kStreamMaxDim && stream_share_ok(num_tokens, num_slots, 0, di);  // equal token shares
}

bool use_weight_split(int64_t num_tokens, const DeviceInfo* di) {
  return num_tokens <= g_wsplit_tokens_per_sm.load(std::memory_order_relaxed) * di->sm_count;
}

int device_info(DeviceInfo** out) {
  int dev = 0;
  PLORA_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(PLORA_ERR_UNSUPPORTED, "device ordinal %d", dev);
  std::lock_guard<std::mutex> lk(g_dev_mu);
  DeviceInfo& d = g_dev[dev];
  if (!d.attrs_set) {
    PLORA_CUDA(cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, dev),
               "cudaDeviceGetAttribute");
    int major = 0, minor = 0;
    PLORA_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev), "cc");
    PLORA_CUDA(cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev), "cc");
    if (major != 10 || minor != 0)
      return fail(PLORA_ERR_UNSUPPORTED, "device %d is sm_%d%d; this build targets sm_100a", dev,
                  major, minor);
#define SET_SMEM(kern, bytes)                                                                  \
  PLORA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,           \
                                  (int)((bytes) + tab_bytes(kFastPathMaxSlots))),              \
             #kern);
#define SET_SMEM_BOTH(name, RPV, bytes)   \
  SET_SMEM((name<RPV, true>), bytes)      \
  SET_SMEM((name<RPV, false>), bytes)
    SET_SMEM_BOTH(sgmv_shrink_mma_kernel, 16, ShrinkMmaCfg<16>::kSmemBytes)
    SET_SMEM_BOTH(sgmv_shrink_mma_kernel, 32, ShrinkMmaCfg<32>::kSmemBytes)
    SET_SMEM_BOTH(sgmv_shrink_mma_kernel, 64, ShrinkMmaCfg<64>::kSmemBytes)
    SET_SMEM_BOTH(sgmv_expand_mma_kernel, 16, ExpandMmaCfg<16>::kSmemBytes)
    SET_SMEM_BOTH(sgmv_expand_mma_kernel, 32, ExpandMmaCfg<32>::kSmemBytes)
    SET_SMEM_BOTH(sgmv_expand_mma_kernel, 64, ExpandMmaCfg<64>::kSmemBytes)
#undef SET_SMEM_BOTH
#undef SET_SMEM
#define SET_GRID(kern, bytes)                                                                  \
  PLORA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,           \
                                  (int)(bytes)),                                               \
             #kern);
#define SET_GRID_ALL(RPV)                                                                      \
  SET_GRID((sgmv_expand_grid_kernel<RPV, true>), ExpandGridCfg<RPV>::kSmemBytes)               \
  SET_GRID((sgmv_expand_grid_kernel<RPV, false>), ExpandGridCfg<RPV>::kSmemBytes)              \
  SET_GRID((sgmv_shrink_grid_kernel<RPV, true>), ShrinkGridCfg<RPV>::kSmemBytes)               \
  SET_GRID((sgmv_shrink_grid_kernel<RPV, false>), ShrinkGridCfg<RPV>::kSmemBytes)              \
  PLORA_CUDA(cudaFuncSetAttribute((sgmv_shrink_grid_kernel<RPV, true>),                        \
                                  cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "cluster"); \
  PLORA_CUDA(cudaFuncSetAttribute((sgmv_shrink_grid_kernel<RPV, false>),                       \
                                  cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "cluster");
    SET_GRID_ALL(16)
    SET_GRID_ALL(32)
    SET_GRID_ALL(64)
#undef SET_GRID_ALL
    SET_GRID((sgmv_shrink_stream_kernel<true, false>), kStreamSmemLimit)
    SET_GRID((sgmv_shrink_stream_kernel<false, false>), kStreamSmemLimit)
    SET_GRID((sgmv_shrink_stream_kernel<true, true>), kStreamSmemLimit)
    SET_GRID((sgmv_shrink_stream_kernel<false, true>), kStreamSmemLimit)
    SET_GRID((sgmv_expand_stream_kernel<true>), kStreamSmemLimit)
    SET_GRID((sgmv_expand_stream_kernel<false>), kStreamSmemLimit)
    SET_GRID(seg_scan_place_kernel, (kSegScanPlaceMaxInts + kSegMaxSlots + 1) * 4)
#define SET_ATTN(DP, NT)                                                       \
  SET_GRID((attn_mma_kernel<true, DP, NT, true>), (AttnMmaCfg<DP, NT>::kSmemBytes))   \
  SET_GRID((attn_mma_kernel<false, DP, NT, true>), (AttnMmaCfg<DP, NT>::kSmemBytes))  \
  SET_GRID((attn_mma_kernel<true, DP, NT, false>), (AttnMmaCfg<DP, NT>::kSmemBytes))  \
  SET_GRID((attn_mma_kernel<false, DP, NT, false>), (AttnMmaCfg<DP, NT>::kSmemBytes))
    SET_ATTN(64, 1)
    SET_ATTN(64, 2)
    SET_ATTN(64, 4)
    SET_ATTN(128, 1)
    SET_ATTN(128, 2)
    SET_ATTN(128, 4)
    SET_ATTN(256, 1)
    SET_ATTN(256, 2)
#undef SET_ATTN
#define SET_SIMT(DP, H) SET_GRID((attn_simt_kernel<DP, H>), (AttnSimtCfg<DP, H>::kSmemBytes))
#define SET_SIMT_ALL(DP) SET_SIMT(DP, 1) SET_SIMT(DP, 2) SET_SIMT(DP, 4) SET_SIMT(DP, 8)
    SET_SIMT_ALL(64)
    SET_SIMT_ALL(128)
    SET_SIMT_ALL(256)
#undef SET_SIMT_ALL
#undef SET_SIMT
    constexpr int kRulesSmem = kRulesMostSmem + kRulesMaxBiases * 12;
#define SET_RULES(T)                                     \
  SET_GRID((logit_find_kernel<T, int32_t>), kRulesSmem) \
  SET_GRID((logit_find_kernel<T, int64_t>), kRulesSmem) \
  SET_MOST_SMEM(logit_copy_kernel<T>)
    // the copy uses no shared memory, the rules beside it do
#define SET_MOST_SMEM(kern)                                                                         \
  PLORA_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout,             \
                                  (int)cudaSharedmemCarveoutMaxShared),                             \
             "cudaFuncSetAttribute(carveout)");
    SET_RULES(float)
    SET_RULES(__half)
    SET_RULES(__nv_bfloat16)
#undef SET_MOST_SMEM
#undef SET_RULES
#undef SET_GRID
    // the row copies use no shared memory; an SM running them keeps its largest
    // shared-memory carveout, so the segment-table kernels of the next rows of
    // a host pipeline fit beside them instead of waiting for the SM to drain
    PLORA_CUDA(cudaFuncSetAttribute(token_rows_copy_kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                    (int)cudaSharedmemCarveoutMaxShared),
               "cudaFuncSetAttribute(carveout)");
    d.attrs_set = true;
  }
  *out = &d;
  return PLORA_OK;
}

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// LoRA-A (num_slots, K, R) viewed as 5-D (R, e:2, m:4, cc:4, block) with
// row k = 32 block + 8 m + 2 cc + e, so that a box lands each 32-row block
// in (cc, m, e) order: shared-memory row position 8 cc + 2 m + e.  Slots are
// folded into the block index (K % 32 == 0); the box covers `blocks` blocks.
int make_map_lora_a_blocks(CUtensorMap* map, const void* base, int dtype, uint64_t R, uint64_t K,
                           uint64_t num_slots, uint32_t blocks, CUtensorMapSwizzle swz) {
  auto enc = tensor_map_encoder();
  if (!enc) return fail(PLORA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const uint64_t row = R * 2;
  const cuuint64_t dims[5] = {R, 2, 4, 4, num_slots * (K / 32)};
  const cuuint64_t strides[4] = {row, 8 * row, 2 * row, 32 * row};
  const cuuint32_t box[5] = {(cuuint32_t)R, 2, 4, 4, blocks};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUtensorMapDataType dt = dtype == PLORA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUresult r = enc(map, dt, 5, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, swz, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(PLORA_ERR_CUDA, "cuTensorMapEncodeTiled (LoRA-A blocks) failed (%d)", (int)r);
  return PLORA_OK;
}

// LoRA-B (num_slots, R, N) viewed as 4-D (64 columns, R, N / 64 chunks, slot):
// a box lands `chunks` 64-column chunks of all R rows, chunk-major, each chunk
// R rows of 128 bytes with the 128-byte swizzle.  Requires N % 64 == 0.
int make_map_lora_b_chunks(CUtensorMap* map, const void* base, int dtype, uint64_t R, uint64_t N,
                           uint64_t num_slots, uint32_t chunks) {
  auto enc = tensor_map_encoder();
  if (!enc) return fail(PLORA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[4] = {64, R, N / 64, num_slots};
  const cuuint64_t strides[3] = {N * 2, 128, R * N * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)R, chunks, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType dt = dtype == PLORA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUresult r = enc(map, dt, 4, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(PLORA_ERR_CUDA, "cuTensorMapEncodeTiled (LoRA-B chunks) failed (%d)", (int)r);
  return PLORA_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

size_t elem_size(int dtype) { return dtype == PLORA_DTYPE_F32 ? 4 : 2; }

bool valid_dtype(int dtype) {
  return dtype == PLORA_DTYPE_F32 || dtype == PLORA_DTYPE_F16 || dtype == PLORA_DTYPE_BF16;
}

int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, what);
  return PLORA_OK;
}

// Workspace of the *_fwd entry points: segment scratch, slot_start, token_index.
struct FwdWorkspace {
  SegWorkspace seg;
  int32_t* slot_start;
  int32_t* token_index;
};

// num_rows x max_seq token ids fit in int32 (checked before any product is formed).
bool token_count_ok(int64_t num_rows, int64_t max_seq) {
  if (num_rows < 0 || max_seq < 0) return false;
  return max_seq == 0 || num_rows <= (int64_t)INT32_MAX / max_seq;
}

size_t fwd_workspace_bytes(int64_t num_rows, int64_t max_seq, int32_t num_slots) {
  return seg_workspace_bytes(num_rows, num_slots) + align256((size_t)(num_slots + 1) * 4) +
         align256((size_t)(num_rows * max_seq) * 4);
}

// Launches `kernel` with programmatic stream serialisation when `pdl` is set:
// the kernel may then start while its predecessor in the stream finishes and
// must call griddep_wait() before reading anything that predecessor writes.
// With cluster_x > 0 the grid is launched as clusters of cluster_x CTAs along x.
template <typename... KArgs, typename... Args>
cudaError_t launch_kernel(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                          cudaStream_t stream, bool pdl, int cluster_x, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  if (cluster_x > 0) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)cluster_x;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

int build_segments(const int64_t* wi, const int32_t* seq_lens, const int32_t* ranks,
                   int64_t num_rows, int64_t max_seq, int32_t num_slots, int32_t* slot_start,
                   int32_t* token_index, void* ws, size_t ws_bytes, cudaStream_t stream) {
  if (num_slots < 1 || num_slots > kSegMaxSlots)
    return fail(PLORA_ERR_UNSUPPORTED, "num_slots %d outside [1, %d]", num_slots, kSegMaxSlots);
  if (num_rows < 0 || max_seq < 0)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "negative num_rows/max_seq");
  if (!token_count_ok(num_rows, max_seq))
    return fail(PLORA_ERR_UNSUPPORTED, "num_rows*max_seq exceeds int32 token ids");
  if (!slot_start) return fail(PLORA_ERR_INVALID_ARGUMENT, "slot_start is null");
  if (num_rows == 0 || max_seq == 0) {
    PLORA_CUDA(cudaMemsetAsync(slot_start, 0, (size_t)(num_slots + 1) * 4, stream), "memset");
    return PLORA_OK;
  }
  if (!wi || !seq_lens || !ranks || !token_index)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "null segment input");
  const size_t need = seg_workspace_bytes(num_rows, num_slots);
  if (!ws || ws_bytes < need)
    return fail(PLORA_ERR_WORKSPACE, "segment workspace %zu < %zu bytes", ws_bytes, need);
  if (num_rows <= kSegSmallRows && num_slots <= kSegSmallSlots && num_rows * max_seq <= kSegSmallTokens) {
    PLORA_CUDA(launch_kernel(seg_small_kernel, dim3(1), dim3(1024), 0, stream, true, 0, wi, seq_lens, ranks,
                             (int32_t)num_rows, max_seq, num_slots, slot_start, token_index),
               "launch seg_small_kernel");
    return check_launch("seg_small_kernel");
  }
  SegWorkspace w = seg_workspace_carve(ws, num_rows, num_slots);
  const int64_t blocks = (num_rows + kSegRowsPerBlock - 1) / kSegRowsPerBlock;
  if (blocks > INT32_MAX) return fail(PLORA_ERR_UNSUPPORTED, "too many rows");
  // programmatic launches: each kernel waits for its predecessor before touching memory
  PLORA_CUDA(launch_kernel(seg_count_kernel, dim3((unsigned)blocks), dim3(kSegRowsPerBlock), (size_t)num_slots * 4,
                           stream, true, 0, wi, seq_lens, ranks, num_rows, max_seq, num_slots, w),
             "launch seg_count_kernel");
  int st = check_launch("seg_count_kernel");
  if (st) return st;
  if (blocks * num_slots <= kSegScanPlaceMaxInts) {  // scan and placement in one launch
    DeviceInfo* di = nullptr;
    if ((st = device_info(&di))) return st;
    const int64_t grid = std::min<int64_t>(di->sm_count, (num_rows + 31) / 32);
    PLORA_CUDA(launch_kernel(seg_scan_place_kernel, dim3((unsigned)grid), dim3(1024),
                             (size_t)(blocks * num_slots + num_slots + 1) * 4, stream, true, 0, num_rows, max_seq,
                             seq_lens, (int32_t)blocks, num_slots, w, slot_start, token_index),
               "launch seg_scan_place_kernel");
    return check_launch("seg_scan_place_kernel");
  }
  PLORA_CUDA(launch_kernel(seg_scan_kernel, dim3(1), dim3(1024), (size_t)num_slots * 4, stream, true, 0,
                           (int32_t)blocks, num_slots, w, slot_start),
             "launch seg_scan_kernel");
  if ((st = check_launch("seg_scan_kernel"))) return st;
  PLORA_CUDA(launch_kernel(seg_place_kernel, dim3((unsigned)((num_rows + 7) / 8)), dim3(256), 0, stream, true, 0,
                           num_rows, max_seq, seq_lens, (int32_t)blocks, w, slot_start, token_index),
             "launch seg_place_kernel");
  return check_launch("seg_place_kernel");
}

// Tensor-core path eligibility (16-bit types, rank tile 16/32/64, 16-byte rows).
bool tc_rank_ok(int64_t R) { return R == 16 || R == 32 || R == 64; }


// K parts of the grid-split shrink: parts of >= 2048 rows (a multiple of 32),
// at most 8 (a portable cluster).  On B200 at config-4 decode (256 tokens over
// 128 slots) that measured fastest: K = 14336 in 7 parts took 45.3 us against
// 49.7 in 8 and 65.6 in 16 (16-CTA clusters fit only ~16 at once); K = 4096 in
// 2 parts 24.8 us against 26.7 in 8.
void grid_k_parts(int64_t K, int* parts, int* part_rows) {
  int kp = (int)std::min<int64_t>(8, std::max<int64_t>(1, (K + 2047) / 2048));
  const int rows = (int)(((K + kp - 1) / kp + 31) / 32 * 32);
  *part_rows = rows;
  *parts = (int)((K + rows - 1) / rows);
}


int shrink_impl(const void* x, const void* a, void* tmp, const int32_t* ranks, SegTable seg,
                int64_t num_tokens, int64_t K, int64_t R, int32_t stack_num, int32_t dtype,
                cudaStream_t stream) {
  DeviceInfo* di = nullptr;
  int st = device_info(&di);
  if (st) return st;
  ShrinkArgs args;
  args.x = static_cast<const uint8_t*>(x);
  args.a = static_cast<const uint8_t*>(a);
  args.tmp = static_cast<uint8_t*>(tmp);
  args.ranks = ranks;
  args.seg = seg;
  args.K = (int32_t)K;
  args.R = (int32_t)R;
  args.stack_num = stack_num;
  const bool tc = dtype != PLORA_DTYPE_F32 && tc_rank_ok(R) && K % 32 == 0 &&
                  seg.num_slots <= kFastPathMaxSlots && aligned16(x) &&
                  aligned16(a) && aligned16(tmp);
  if (tc) {
    const bool bf = dtype == PLORA_DTYPE_BF16;
    if (use_weight_split(num_tokens, di)) {  // few tokens per slot: grid split
      int kp = 0, kp_rows = 0;
      grid_k_parts(K, &kp, &kp_rows);
      // rows: slots plus later 16-token tiles (few K parts, rows within a grid dimension), else slots
      const int64_t tile_rows = grid_tile_rows(num_tokens, seg.num_slots);
      const bool by_tile = kp <= kTileMaxKParts && tile_rows <= 65535;
      const dim3 grid((unsigned)kp, (unsigned)(by_tile ? tile_rows : seg.num_slots));
      // the kernel reads its inputs only after griddep_wait(): always launched programmatically
#define LAUNCH_SHRINK_GRID(RPV)                                                                    \
  PLORA_CUDA(launch_kernel(bf ? sgmv_shrink_grid_kernel<RPV, true> : sgmv_shrink_grid_kernel<RPV, false>, \
                           grid, dim3(kGridThreads), ShrinkGridCfg<RPV>::kSmemBytes, stream, true, kp, \
                           args, kp_rows, by_tile, (int)grid_later_rows(num_tokens)),              \
             "launch sgmv_shrink_grid_kernel");
      if (R == 16) {
        LAUNCH_SHRINK_GRID(16)
      } else if (R == 32) {
        LAUNCH_SHRINK_GRID(32)
      } else {
        LAUNCH_SHRINK_GRID(64)
      }
#undef LAUNCH_SHRINK_GRID
      return check_launch("sgmv_shrink_grid_kernel");
    }
    if (stream_shrink_ok(R, K, num_tokens, seg.num_slots, di)) {  // rank 16: rows through a bulk-copy ring, A in registers
      const StreamPlan plan = shrink_stream_plan(K, seg.num_slots);
      if (plan.nst >= 2) {
        // the kernel reads its inputs only after griddep_wait(): always launched programmatically
        PLORA_CUDA(launch_kernel(bf ? sgmv_shrink_stream_kernel<true, false> : sgmv_shrink_stream_kernel<false, false>,
                                 dim3(di->sm_count), dim3(kShrinkThreads), plan.smem_bytes, stream, true, 0,
                                 args, plan, ExpandArgs{}, FusedPlan{}),
                   "launch sgmv_shrink_stream_kernel");
        return check_launch("sgmv_shrink_stream_kernel");
      }
    }
    CUtensorMap map8, map1;
    const CUtensorMapSwizzle swz = R == 16   ? CU_TENSOR_MAP_SWIZZLE_32B
                                   : R == 32 ? CU_TENSOR_MAP_SWIZZLE_64B
                                             : CU_TENSOR_MAP_SWIZZLE_128B;
    if ((st = make_map_lora_a_blocks(&map8, a, dtype, (uint64_t)R, (uint64_t)K,
                                     (uint64_t)seg.num_slots, kWinBoxRows / 32, swz)) ||
        (st = make_map_lora_a_blocks(&map1, a, dtype, (uint64_t)R, (uint64_t)K,
                                     (uint64_t)seg.num_slots, 1, swz)))
      return st;
    const dim3 grid(di->sm_count), block(kMmaThreads);
    const size_t tb = tab_bytes(seg.num_slots);
    // the kernel reads its inputs only after griddep_wait(): always launched programmatically
#define LAUNCH_SHRINK(RPV)                                                                         \
  PLORA_CUDA(launch_kernel(bf ? sgmv_shrink_mma_kernel<RPV, true> : sgmv_shrink_mma_kernel<RPV, false>, \
                           grid, block, ShrinkMmaCfg<RPV>::kSmemBytes + tb, stream, true, 0, map8, map1, args), \
             "launch sgmv_shrink_mma_kernel");
    if (R == 16) {
      LAUNCH_SHRINK(16)
    } else if (R == 32) {
      LAUNCH_SHRINK(32)
    } else {
      LAUNCH_SHRINK(64)
    }
#undef LAUNCH_SHRINK
    return check_launch("sgmv_shrink_mma_kernel");
  }
  if (R > kSimtMaxRank) return fail(PLORA_ERR_UNSUPPORTED, "max_rank %lld > %d", (long long)R, kSimtMaxRank);
  const dim3 grid(di->sm_count * 8), block(kSimtThreads);
  if (dtype == PLORA_DTYPE_F32)
    sgmv_shrink_simt_kernel<float><<<grid, block, 0, stream>>>(args, seg.num_slots);
  else if (dtype == PLORA_DTYPE_BF16)
    sgmv_shrink_simt_kernel<__nv_bfloat16><<<grid, block, 0, stream>>>(args, seg.num_slots);
  else
    sgmv_shrink_simt_kernel<__half><<<grid, block, 0, stream>>>(args, seg.num_slots);
  return check_launch("sgmv_shrink_simt_kernel");
}

int expand_impl(const void* tmp, const void* b, void* y, const int32_t* ranks, const float* scales,
                SegTable seg, int64_t num_tokens, int64_t R, int64_t N, int32_t dtype,
                cudaStream_t stream, bool after_shrink = false) {
  DeviceInfo* di = nullptr;
  int st = device_info(&di);
  if (st) return st;
  ExpandArgs args;
  args.tmp = static_cast<const uint8_t*>(tmp);
  args.b = static_cast<const uint8_t*>(b);
  args.y = static_cast<uint8_t*>(y);
  args.ranks = ranks;
  args.scales = scales;
  args.seg = seg;
  args.R = (int32_t)R;
  args.N = (int32_t)N;
  const bool tc = dtype != PLORA_DTYPE_F32 && tc_rank_ok(R) && N % 64 == 0 &&
                  seg.num_slots <= kFastPathMaxSlots && aligned16(tmp) &&
                  aligned16(b) && aligned16(y);
  if (tc) {
    const bool bf = dtype == PLORA_DTYPE_BF16;
    if (use_weight_split(num_tokens, di)) {  // few tokens per slot: grid split
      // rows: slots plus later 16-token tiles (few column chunks, rows within a grid dimension), else slots
      const int64_t chunks = (N + kGridCols - 1) / kGridCols;
      const int64_t tile_rows = grid_tile_rows(num_tokens, seg.num_slots);
      const bool by_tile = chunks <= kTileMaxColChunks && tile_rows <= 65535;
      const dim3 grid((unsigned)chunks, (unsigned)(by_tile ? tile_rows : seg.num_slots));
      // programmatic only right after this library's shrink: tmp is read after griddep_wait()
#define LAUNCH_EXPAND_GRID(RPV)                                                                    \
  PLORA_CUDA(launch_kernel(bf ? sgmv_expand_grid_kernel<RPV, true> : sgmv_expand_grid_kernel<RPV, false>, \
                           grid, dim3(kGridThreads), ExpandGridCfg<RPV>::kSmemBytes, stream,       \
                           after_shrink, 0, args, by_tile, (int)grid_later_rows(num_tokens)),       \
             "launch sgmv_expand_grid_kernel");
      if (R == 16) {
        LAUNCH_EXPAND_GRID(16)
      } else if (R == 32) {
        LAUNCH_EXPAND_GRID(32)
      } else {
        LAUNCH_EXPAND_GRID(64)
      }
#undef LAUNCH_EXPAND_GRID
      return check_launch("sgmv_expand_grid_kernel");
    }
    if (stream_expand_ok(R, N, num_tokens, seg.num_slots, di)) {  // rank 16: rows through a bulk-copy ring, B in registers
      const StreamPlan plan = expand_stream_plan(N, seg.num_slots);
      if (plan.smem_bytes <= (uint32_t)kStreamSmemLimit) {
        // programmatic only right after this library's shrink (after_shrink): the kernel
        // reads the segment table and LoRA-B before griddep_wait(), tmp after it; y is
        // only added to, after tmp
        PLORA_CUDA(launch_kernel(bf ? sgmv_expand_stream_kernel<true> : sgmv_expand_stream_kernel<false>,
                                 dim3(di->sm_count), dim3(kStreamThreads), plan.smem_bytes, stream,
                                 after_shrink, 0, args, plan),
                   "launch sgmv_expand_stream_kernel");
        return check_launch("sgmv_expand_stream_kernel");
      }
    }
    CUtensorMap mapn, map1;
    const uint32_t box = R == 16 ? ExpandMmaCfg<16>::kBoxChunks
                         : R == 32 ? ExpandMmaCfg<32>::kBoxChunks
                                   : ExpandMmaCfg<64>::kBoxChunks;
    if ((st = make_map_lora_b_chunks(&mapn, b, dtype, (uint64_t)R, (uint64_t)N,
                                     (uint64_t)seg.num_slots, box)) ||
        (st = make_map_lora_b_chunks(&map1, b, dtype, (uint64_t)R, (uint64_t)N,
                                     (uint64_t)seg.num_slots, 1)))
      return st;
    const dim3 grid(di->sm_count), block(kMmaThreads);
    const size_t tb = tab_bytes(seg.num_slots);
    // programmatic only right after this library's shrink (after_shrink): the kernel reads
    // the segment table, LoRA-B and y before griddep_wait(), tmp after it
#define LAUNCH_EXPAND(RPV)                                                                         \
  PLORA_CUDA(launch_kernel(bf ? sgmv_expand_mma_kernel<RPV, true> : sgmv_expand_mma_kernel<RPV, false>, \
                           grid, block, ExpandMmaCfg<RPV>::kSmemBytes + tb, stream, after_shrink, 0, mapn, \
                           map1, args),                                                            \
             "launch sgmv_expand_mma_kernel");
    if (R == 16) {
      LAUNCH_EXPAND(16)
    } else if (R == 32) {
      LAUNCH_EXPAND(32)
    } else {
      LAUNCH_EXPAND(64)
    }
#undef LAUNCH_EXPAND
    return check_launch("sgmv_expand_mma_kernel");
  }
  if (R > kSimtMaxRank) return fail(PLORA_ERR_UNSUPPORTED, "max_rank %lld > %d", (long long)R, kSimtMaxRank);
  const dim3 grid(di->sm_count * 8), block(kSimtThreads);
  if (dtype == PLORA_DTYPE_F32)
    sgmv_expand_simt_kernel<float><<<grid, block, 0, stream>>>(args, seg.num_slots);
  else if (dtype == PLORA_DTYPE_BF16)
    sgmv_expand_simt_kernel<__nv_bfloat16><<<grid, block, 0, stream>>>(args, seg.num_slots);
  else
    sgmv_expand_simt_kernel<__half><<<grid, block, 0, stream>>>(args, seg.num_slots);
  return check_launch("sgmv_expand_simt_kernel");
}

int check_common(int32_t dtype, int32_t num_slots, int64_t max_rank) {
  if (!valid_dtype(dtype)) return fail(PLORA_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  if (num_slots < 1 || num_slots > kSegMaxSlots)
    return fail(PLORA_ERR_UNSUPPORTED, "num_slots %d outside [1, %d]", num_slots, kSegMaxSlots);
  if (max_rank < 1) return fail(PLORA_ERR_INVALID_ARGUMENT, "max_rank must be >= 1");
  return PLORA_OK;
}

FwdWorkspace carve_fwd(void* ws, int64_t num_rows, int64_t max_seq, int32_t num_slots) {
  FwdWorkspace f;
  char* p = static_cast<char*>(ws);
  f.seg = seg_workspace_carve(p, num_rows, num_slots);
  p += seg_workspace_bytes(num_rows, num_slots);
  f.slot_start = reinterpret_cast<int32_t*>(p);
  p += align256((size_t)(num_slots + 1) * 4);
  f.token_index = reinterpret_cast<int32_t*>(p);
  return f;
}

// Device address of `bytes` (> 0) bytes of host memory that a kernel may read
// and write over PCIe: page-locked and mapped at both ends, as one range.
int mapped_host_range(const void* p, int64_t bytes, const char* what, const uint8_t** dev) {
  cudaPointerAttributes a = {}, b = {};
  const void* last = static_cast<const uint8_t*>(p) + (bytes - 1);
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess || cudaPointerGetAttributes(&b, last) != cudaSuccess) {
    cudaGetLastError();
    return fail(PLORA_ERR_INVALID_ARGUMENT, "%s: pointer attributes unavailable", what);
  }
  if (a.type != cudaMemoryTypeHost || b.type != cudaMemoryTypeHost || !a.devicePointer || !b.devicePointer)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "%s must be page-locked, mapped host memory", what);
  const uint8_t* d0 = static_cast<const uint8_t*>(a.devicePointer);
  if (static_cast<const uint8_t*>(b.devicePointer) - d0 != bytes - 1)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "%s is not one mapped range", what);
  *dev = d0;
  return PLORA_OK;
}

int device_range(const void* p, int64_t bytes, const char* what) {
  cudaPointerAttributes a = {}, b = {};
  const void* last = static_cast<const uint8_t*>(p) + (bytes - 1);
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess || cudaPointerGetAttributes(&b, last) != cudaSuccess) {
    cudaGetLastError();
    return fail(PLORA_ERR_INVALID_ARGUMENT, "%s: pointer attributes unavailable", what);
  }
  const bool ok = (a.type == cudaMemoryTypeDevice || a.type == cudaMemoryTypeManaged) && a.type == b.type;
  if (!ok) return fail(PLORA_ERR_INVALID_ARGUMENT, "%s must be device memory", what);
  return PLORA_OK;
}

// Both directions of the token-row copy: arguments checked on the host, then
// one programmatic launch of token_rows_copy_kernel.
int token_rows_impl(const void* host_rows, void* device_rows, bool to_host, int64_t row_bytes, int64_t num_tokens,
                    const int32_t* slot_start, const int32_t* token_index, int32_t num_slots, void* stream) {
  g_last_error.clear();
  if (row_bytes < 16 || row_bytes % 16 || num_tokens < 0)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "row_bytes must be a positive multiple of 16, num_tokens >= 0");
  if (num_slots < 1 || num_slots > kSegMaxSlots)
    return fail(PLORA_ERR_UNSUPPORTED, "num_slots %d outside [1, %d]", num_slots, kSegMaxSlots);
  if (num_tokens > (int64_t)INT32_MAX) return fail(PLORA_ERR_UNSUPPORTED, "num_tokens exceeds int32 token ids");
  if (row_bytes > INT64_MAX / std::max<int64_t>(num_tokens, 1))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "num_tokens * row_bytes overflows");
  if (num_tokens == 0) return PLORA_OK;
  if (!host_rows || !device_rows || !slot_start || !token_index)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "null pointer");
  if (reinterpret_cast<uintptr_t>(host_rows) % 16 || reinterpret_cast<uintptr_t>(device_rows) % 16)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "row buffers must be 16-byte aligned");
  const int64_t bytes = num_tokens * row_bytes;
  const uint8_t* host_dev = nullptr;
  int st = mapped_host_range(host_rows, bytes, "host_rows", &host_dev);
  if (st) return st;
  st = device_range(device_rows, bytes, "device_rows");
  if (st) return st;
  DeviceInfo* di = nullptr;
  st = device_info(&di);
  if (st) return st;
  const uint8_t* dev_rows = static_cast<const uint8_t*>(device_rows);
  const uint8_t* src = to_host ? dev_rows : host_dev;
  uint8_t* dst = const_cast<uint8_t*>(to_host ? host_dev : dev_rows);
  // a plain launch: the rows' producers typically finish on another stream (events)
  PLORA_CUDA(launch_kernel(token_rows_copy_kernel, dim3((unsigned)(2 * di->sm_count)), dim3(kRowsThreads), 0,
                           static_cast<cudaStream_t>(stream), false, 0, src, dst, row_bytes, num_tokens, slot_start,
                           token_index, num_slots),
             "launch token_rows_copy_kernel");
  return PLORA_OK;
}

// ---------------------------------------------------------------- paged cache
// Whether two byte ranges share memory.
bool ranges_meet(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const __int128 x = (__int128)reinterpret_cast<uintptr_t>(a), y = (__int128)reinterpret_cast<uintptr_t>(b);
  return a_bytes > 0 && b_bytes > 0 && x < y + b_bytes && y < x + a_bytes;
}
// Whether rows of `width` elements at two addresses share memory without being
// the same rows.  Rows of one stride may interleave.
bool rows_meet(const void* a, int64_t a_stride, const void* b, int64_t b_stride, int64_t rows, int64_t width, int64_t el) {
  if (a == b && (a_stride == b_stride || rows == 1)) return false;
  if (!ranges_meet(a, ((rows - 1) * a_stride + width) * el, b, ((rows - 1) * b_stride + width) * el)) return false;
  if (a_stride != b_stride || rows == 1) return true;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  const int64_t off = (int64_t)((x < y ? y - x : x - y) % (uint64_t)(a_stride * el));
  return off < width * el || off > (a_stride - width) * el;
}
// SMs of a B200: the attention grid, so that its workspace does not depend on the device.
constexpr int kAttnGrid = 148;
constexpr int64_t kPagedMaxRows = 1 << 20;

// The attention kernel of a call: padded head size, query heads of its block (in
// eights for the tensor cores, 0: CUDA cores, `simt` heads) and warps of a CTA.
// Blocks are as large as registers allow, for a second block reads the cache again.
struct AttnPlan {
  int dp, eights, simt, blocks, block_heads, warps, segments;
  int direct;  // CTAs of an item's cluster; 0: by the list
  size_t before_offset, cut_offset, ml_offset, part_offset, bytes;
};
AttnPlan attn_plan(int64_t rows, int32_t heads, int32_t kv_heads, int32_t dim, int64_t capacity, int64_t window, int dtype) {
  AttnPlan a;
  const int group = heads / kv_heads;
  a.dp = dim <= 64 ? 64 : (dim <= 128 ? 128 : 256);
  const int most = dtype == PLORA_DTYPE_F32 ? 8 : (a.dp == 256 ? 16 : 32);
  a.blocks = (group + most - 1) / most;
  a.block_heads = (group + a.blocks - 1) / a.blocks;
  a.blocks = (group + a.block_heads - 1) / a.block_heads;
  a.eights = a.simt = 0;
  if (dtype == PLORA_DTYPE_F32) {
    a.simt = a.block_heads <= 2 ? a.block_heads : (a.block_heads <= 4 ? 4 : 8);
    a.warps = a.dp == 64 ? AttnSimtCfg<64, 8>::kWarps : (a.dp == 128 ? AttnSimtCfg<128, 8>::kWarps : AttnSimtCfg<256, 8>::kWarps);
  } else {
    a.eights = a.block_heads <= 8 ? 1 : (a.block_heads <= 16 ? 2 : 4);
#define PLORA_WARPS(DP, NT) \
  if (a.dp == DP && a.eights == NT) a.warps = AttnMmaCfg<DP, NT>::kWarps;
    PLORA_WARPS(64, 1) PLORA_WARPS(64, 2) PLORA_WARPS(64, 4)
    PLORA_WARPS(128, 1) PLORA_WARPS(128, 2) PLORA_WARPS(128, 4)
    PLORA_WARPS(256, 1) PLORA_WARPS(256, 2)
#undef PLORA_WARPS
  }
  // Without a list where the SMs hold all items at once with few tiles a warp, as
  // far as the page table's width tells: the lengths are on the device.  One row
  // of 200 tokens: 5 us against 10.
  const int64_t tokens = window > 0 && window < capacity ? std::min(capacity, window + kAttnTile - 1) : capacity;
  const int64_t tiles = (tokens + kAttnTile - 1) / kAttnTile, items = rows * kv_heads * a.blocks;
  // Clusters of 1, 2, ... CTAs, one CTA an SM, that the GPU holds at once (what
  // cudaOccupancyMaxActiveClusters says there, a few left out): a cluster lies in one GPC.
  constexpr int kClusters[kAttnClusterCtas] = {kAttnGrid, 74, 44, 32, 25, 21, 15, 15};
  a.direct = 0;
  for (int ctas = 1; ctas <= kAttnClusterCtas && items > 0 && !a.direct; ++ctas)  // the fewest that have enough warps
    if (items <= kClusters[ctas - 1] && tiles <= ctas * a.warps * kAttnDirect) a.direct = ctas;
  for (int ctas = a.direct; a.direct && ctas <= kAttnClusterCtas; ++ctas)  // and more, down to a tile a warp
    if (items <= kClusters[ctas - 1] && tiles > (ctas - 1) * a.warps) a.direct = ctas;
  a.bytes = 0;
  if (a.direct) return a;
  const size_t segments = (size_t)kAttnGrid * a.warps + attn_asked_max(kAttnGrid * a.warps, a.block_heads);
  const size_t parts = segments * 2 * a.block_heads;
  a.before_offset = 256;
  a.segments = (int)segments;
  a.cut_offset = a.before_offset + align256((size_t)rows * 8);
  a.ml_offset = a.cut_offset + align256(segments * 16);
  a.part_offset = a.ml_offset + align256(parts * 8);
  a.bytes = a.part_offset + align256(parts * dim * 4);
  return a;
}

// Arguments that both paged entry points share.
int paged_view(PagedView* c, const plora_paged_cache& a, int64_t heads) {
  const int64_t head_dim = a.head_dim, page_size = a.page_size, kv_heads = a.kv_heads;
  if (a.dtype < 0 || a.dtype > INT32_MAX || !valid_dtype((int)a.dtype))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "unknown dtype %lld", (long long)a.dtype);
  if (a.rows < 0 || kv_heads < 1 || heads < 0 || head_dim < 1 || page_size < 1 || a.num_pages < 1 || a.max_pages < 1)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "rows, heads, head_dim, page_size or page counts not positive");
  if (heads % kv_heads)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "%lld heads over %lld kv heads", (long long)heads, (long long)kv_heads);
  if (head_dim % 8 || head_dim > 256)
    return fail(PLORA_ERR_UNSUPPORTED, "head_dim %lld is no multiple of 8 up to 256", (long long)head_dim);
  if (a.rows > kPagedMaxRows || heads > 65535 || kv_heads > 65535)
    return fail(PLORA_ERR_UNSUPPORTED, "%lld rows, %lld heads", (long long)a.rows, (long long)heads);
  if (page_size > INT32_MAX || a.num_pages > INT32_MAX || a.max_pages > INT32_MAX / page_size)
    return fail(PLORA_ERR_UNSUPPORTED, "page_size, num_pages, or positions of max_pages pages, beyond int32");
  const int64_t page_elems = kv_heads * head_dim;  // kv_heads <= 65535, head_dim <= 256
  if (page_elems > INT32_MAX / page_size) return fail(PLORA_ERR_UNSUPPORTED, "elements of a page beyond int32");
  if (a.k_page_stride < page_elems * page_size || a.v_page_stride < page_elems * page_size ||
      a.table_stride < a.max_pages)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "page or page-table stride below its extent");
  const int64_t vec = 16 / (int64_t)elem_size((int)a.dtype);
  if (a.k_page_stride % vec || a.v_page_stride % vec || !aligned16(a.k_cache) || !aligned16(a.v_cache))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "cache pages must be 16-byte aligned");
  if (a.num_pages > INT64_MAX / 16 / std::max(a.k_page_stride, a.v_page_stride))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "cache size overflows");
  if (a.rows > 0 && (!a.k_cache || !a.v_cache || !a.page_table)) return fail(PLORA_ERR_INVALID_ARGUMENT, "null pointer");
  c->k = a.k_cache;
  c->v = a.v_cache;
  c->table = a.page_table;
  c->table_stride = a.table_stride;
  c->k_page = a.k_page_stride;
  c->v_page = a.v_page_stride;
  c->capacity = a.max_pages * page_size;
  c->num_pages = (int32_t)a.num_pages;
  c->kv_heads = (int32_t)kv_heads;
  c->page_size = (int32_t)page_size;
  c->dim = (int32_t)head_dim;
  c->page.set((uint32_t)page_size);
  return PLORA_OK;
}

template <typename T>
cudaError_t launch_append(const AppendParams& p, bool vec, unsigned grid, cudaStream_t s) {
  return vec ? launch_kernel(paged_append_kernel<T, true>, dim3(grid), dim3(kAppendThreads), 0, s, true, 0, p)
             : launch_kernel(paged_append_kernel<T, false>, dim3(grid), dim3(kAppendThreads), 0, s, true, 0, p);
}

// A 16-bit cache viewed as (64 elements, slot, 64-element block, kv head, page);
// a box is a tile: 16 slots of one head of one page, block by block.
int make_map_cache(CUtensorMap* map, const void* base, int dtype, const PagedView& c, int64_t page_stride) {
  auto enc = tensor_map_encoder();
  if (!enc) return fail(PLORA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t d = c.dim;
  const cuuint64_t dims[5] = {64, (cuuint64_t)c.page_size, d / 64, (cuuint64_t)c.kv_heads, (cuuint64_t)c.num_pages};
  const cuuint64_t strides[4] = {d * 2, 128, (cuuint64_t)c.page_size * d * 2, (cuuint64_t)page_stride * 2};
  const cuuint32_t box[5] = {64, kAttnTile, (cuuint32_t)(d / 64), 1, 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUtensorMapDataType dt = dtype == PLORA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                           : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUresult r = enc(map, dt, 5, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(PLORA_ERR_CUDA, "cuTensorMapEncodeTiled (cache) failed (%d)", (int)r);
  return PLORA_OK;
}

// TMA copies whole tiles of whole pages, 64 elements at a time.
bool attn_by_tma(const PagedView& c, const AttnPlan& a) {
  const int64_t most = (1ll << 39) - 1;  // elements: strides below 2^40 bytes
  return a.eights > 0 && c.dim == a.dp && c.page_size % kAttnTile == 0 && c.k_page <= most && c.v_page <= most;
}

cudaError_t launch_attn(const AttnParams& p, const AttnPlan& a, int dtype, bool tma, const CUtensorMap& mk,
                        const CUtensorMap& mv, cudaStream_t s) {
  cudaError_t e = cudaErrorInvalidValue;
  if (!p.direct) {
    e = launch_kernel(attn_plan_kernel, dim3(1), dim3(kAttnPlanThreads), 0, s, true, 0, p, kAttnGrid * a.warps);
    if (e != cudaSuccess) return e;
    e = cudaErrorInvalidValue;
  }
  const dim3 ctas(p.direct ? (unsigned)(p.rows * p.c.kv_heads * p.blocks * p.direct) : kAttnGrid);
#define PLORA_SIMT(DP, H)                                                                                  \
  if (a.simt == H && a.dp == DP)                                                                           \
    e = launch_kernel(attn_simt_kernel<DP, H>, ctas, dim3(a.warps * 32), AttnSimtCfg<DP, H>::kSmemBytes,   \
                      s, true, p.direct, p);
#define PLORA_SIMT_ALL(DP) PLORA_SIMT(DP, 1) PLORA_SIMT(DP, 2) PLORA_SIMT(DP, 4) PLORA_SIMT(DP, 8)
#define PLORA_MMA(BF16, DP, NT, TMA)                                                                      \
  if (a.eights == NT && a.dp == DP && BF16 == (dtype == PLORA_DTYPE_BF16) && TMA == tma)                  \
    e = launch_kernel(attn_mma_kernel<BF16, DP, NT, TMA>, ctas, dim3(a.warps * 32),                       \
                      AttnMmaCfg<DP, NT>::kSmemBytes, s, true, p.direct, p, mk, mv);
#define PLORA_MMA_BOTH(DP, NT) \
  PLORA_MMA(true, DP, NT, true) PLORA_MMA(false, DP, NT, true) PLORA_MMA(true, DP, NT, false) PLORA_MMA(false, DP, NT, false)
  PLORA_SIMT_ALL(64) PLORA_SIMT_ALL(128) PLORA_SIMT_ALL(256)
  PLORA_MMA_BOTH(64, 1) PLORA_MMA_BOTH(64, 2) PLORA_MMA_BOTH(64, 4)
  PLORA_MMA_BOTH(128, 1) PLORA_MMA_BOTH(128, 2) PLORA_MMA_BOTH(128, 4)
  PLORA_MMA_BOTH(256, 1) PLORA_MMA_BOTH(256, 2)
#undef PLORA_MMA_BOTH
#undef PLORA_MMA
#undef PLORA_SIMT_ALL
#undef PLORA_SIMT
  if (e != cudaSuccess || p.direct) return e;
  const dim3 grid(kJoinGrid), block(kJoinWarps * 32);
  return dtype == PLORA_DTYPE_F32   ? launch_kernel(attn_join_kernel<float>, grid, block, 0, s, true, 0, p)
         : dtype == PLORA_DTYPE_F16 ? launch_kernel(attn_join_kernel<__half>, grid, block, 0, s, true, 0, p)
                                    : launch_kernel(attn_join_kernel<__nv_bfloat16>, grid, block, 0, s, true, 0, p);
}

// The call's kernels: which run, how the finding cuts a row's vocabulary, and the
// workspace that lists of rules need.
struct RulesPlan {
  bool copy, find, lists, fused;
  int part, parts;
  size_t smem, listed_offset, bytes;
};
RulesPlan rules_plan(int64_t rows, int64_t vocab, int64_t history, int64_t biases, bool copy) {
  RulesPlan a = {};
  const int64_t entries = history + biases;
  a.copy = copy;
  a.find = entries > 0;
  // as small a part as keeps all CTAs beside the copy (rows of kRulesLeastPart or less
  // are not cut), and one whose tables leave room for a second CTA
  const int64_t cuts = std::max<int64_t>(kRulesBesideCtas / std::max<int64_t>(rows, 1), 1);
  const int64_t share = std::max<int64_t>(((vocab + cuts - 1) / cuts + 31) & ~31ll, kRulesLeastPart);
  a.part = (int)std::min({std::max<int64_t>(vocab, 1), share, (int64_t)kRulesMostPart});
  while (a.part > 1024 && rules_smem_bytes(a.part, entries, 0) > kRulesMostSmem) a.part = (a.part / 2 + 31) & ~31;
  a.parts = (int)((vocab + a.part - 1) / a.part);
  a.smem = (size_t)rules_smem_bytes(a.part, entries, (int)biases);
  // one finding CTA fits on an SM beside the copy
  a.lists = a.find && copy && rows * a.parts > kRulesBesideCtas;
  // Small parts are copied by the CTAs that find their rules: a launch less.  Two kernels
  // and one: 1 x 128256 bf16 15.6 and 13.4 us a call (host), 5.0 and 5.6 on the device;
  // 64 x 128256, parts of 64128, 15.7 and 14.3, 8.9 and 14.3.
  a.fused = a.find && copy && !a.lists && a.part <= kRulesLeastPart;
  if (a.lists) {
    a.listed_offset = align256((size_t)(rows * a.parts) * rules_ruled(a.part, entries) * sizeof(RulesEntry));
    a.bytes = a.listed_offset + align256((size_t)(rows * a.parts) * 4);
  }
  return a;
}

template <typename T>
cudaError_t launch_rules(RulesParams& p, const RulesPlan& a, bool wide, int64_t rows, cudaStream_t s) {
  const dim3 block(kRulesThreads);
  cudaError_t e = cudaSuccess;
  auto copy = [&] {
    const int64_t strips = (p.vocab * sizeof(T) + kRulesStrip * 16 - 1) / (kRulesStrip * 16);
    const dim3 grid((unsigned)((strips * 32 + kRulesThreads - 1) / kRulesThreads), (unsigned)rows);
    e = launch_kernel(logit_copy_kernel<T>, grid, block, 0, s, true, 0, p);
  };
  p.copies = a.fused;
  p.beside = a.copy && !a.lists && !a.fused;
  if (p.beside) {
    copy();
    if (e != cudaSuccess) return e;
  }
  if (!a.find) return e;
  const dim3 grid((unsigned)a.parts, (unsigned)rows);
  e = wide ? launch_kernel(logit_find_kernel<T, int64_t>, grid, block, a.smem, s, true, 0, p)
           : launch_kernel(logit_find_kernel<T, int32_t>, grid, block, a.smem, s, true, 0, p);
  if (e != cudaSuccess || !a.lists) return e;
  copy();
  if (e != cudaSuccess) return e;
  return launch_kernel(logit_apply_kernel<T>, dim3(4, (unsigned)rows), block, 0, s, true, 0, p);
}

}  // namespace

extern "C" {

const char* plora_version(void) { return "polylora_b200 0.1.0 (sm_100a)"; }

const char* plora_status_string(int status) {
  switch (status) {
    case PLORA_OK: return "ok";
    case PLORA_ERR_INVALID_ARGUMENT: return "invalid argument";
    case PLORA_ERR_UNSUPPORTED: return "unsupported";
    case PLORA_ERR_CUDA: return "CUDA error";
    case PLORA_ERR_WORKSPACE: return "workspace too small";
    case PLORA_ERR_DEVICE: return "device status raised";
    default: return "unknown status";
  }
}

const char* plora_last_error(void) { return g_last_error.c_str(); }

int64_t plora_weight_split_tokens_per_sm(int64_t value) {
  return value >= 0 ? g_wsplit_tokens_per_sm.exchange(value) : g_wsplit_tokens_per_sm.load();
}

int32_t plora_stream_kernels(int32_t value) {
  return value >= 0 ? g_stream_kernels.exchange(value > 2 ? 2 : value) : g_stream_kernels.load();
}

int plora_set_wait_limit_ns(uint64_t limit_ns, uint64_t* previous) {
  g_last_error.clear();
  uint64_t old = 0;
  PLORA_CUDA(cudaDeviceSynchronize(), "cudaDeviceSynchronize");
  PLORA_CUDA(cudaMemcpyFromSymbol(&old, g_wait_limit_ns, sizeof(old)), "read wait limit");
  PLORA_CUDA(cudaMemcpyToSymbol(g_wait_limit_ns, &limit_ns, sizeof(limit_ns)), "set wait limit");
  if (previous) *previous = old;
  return PLORA_OK;
}

int plora_device_status(int32_t* status_out, int32_t clear) {
  int v = 0;
  PLORA_CUDA(cudaDeviceSynchronize(), "cudaDeviceSynchronize");
  PLORA_CUDA(cudaMemcpyFromSymbol(&v, g_device_status, sizeof(int)), "read device status");
  if (clear) {
    const int zero = 0;
    PLORA_CUDA(cudaMemcpyToSymbol(g_device_status, &zero, sizeof(int)), "clear device status");
  }
  if (status_out) *status_out = v;
  return v ? fail(PLORA_ERR_DEVICE, "device status 0x%x", v) : PLORA_OK;
}

size_t plora_workspace_size(int64_t num_rows, int64_t max_seq, int32_t num_slots) {
  if (!token_count_ok(num_rows, max_seq) || num_slots < 1 || num_slots > kSegMaxSlots) return 0;
  return fwd_workspace_bytes(num_rows, max_seq, num_slots);
}

int plora_build_segments(const int64_t* weight_indices, const int32_t* seq_lens,
                         const int32_t* lora_ranks, int64_t num_rows, int64_t max_seq,
                         int32_t num_slots, int32_t* slot_start, int32_t* token_index,
                         void* workspace, size_t workspace_size, void* stream) {
  g_last_error.clear();
  return build_segments(weight_indices, seq_lens, lora_ranks, num_rows, max_seq, num_slots,
                        slot_start, token_index, workspace, workspace_size,
                        static_cast<cudaStream_t>(stream));
}

int plora_gather_token_rows(const void* host_rows, void* device_rows, int64_t row_bytes, int64_t num_tokens,
                            const int32_t* slot_start, const int32_t* token_index, int32_t num_slots,
                            void* stream) {
  return token_rows_impl(host_rows, device_rows, false, row_bytes, num_tokens, slot_start, token_index, num_slots,
                         stream);
}

int plora_scatter_token_rows(const void* device_rows, void* host_rows, int64_t row_bytes, int64_t num_tokens,
                             const int32_t* slot_start, const int32_t* token_index, int32_t num_slots,
                             void* stream) {
  return token_rows_impl(host_rows, const_cast<void*>(device_rows), true, row_bytes, num_tokens, slot_start,
                         token_index, num_slots, stream);
}

int plora_check_right_padded(const void* mask, int32_t mask_elem_bytes, int32_t mask_is_float,
                             const int64_t* seq_lens, int64_t rows, int64_t width, void* stream) {
  g_last_error.clear();
  const bool size_ok = mask_elem_bytes == 1 || mask_elem_bytes == 2 || mask_elem_bytes == 4 || mask_elem_bytes == 8;
  if (rows < 0 || width < 0 || !size_ok || (mask_is_float && mask_elem_bytes == 1))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "mask shape or element type");
  if (rows > INT32_MAX) return fail(PLORA_ERR_UNSUPPORTED, "more than 2^31-1 mask rows");
  if (rows == 0 || width == 0) return PLORA_OK;
  if (!mask || !seq_lens) return fail(PLORA_ERR_INVALID_ARGUMENT, "null pointer");
  if (reinterpret_cast<uintptr_t>(mask) % mask_elem_bytes)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "mask not aligned to its element size");
  mask_padding_kernel<<<(unsigned)rows, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(mask), mask_elem_bytes, mask_is_float ? 1 : 0, seq_lens, width);
  return check_launch("mask_padding_kernel");
}

int plora_flat_schedule(const int32_t* seq_lens, const int32_t* n_eff, int64_t num_rows,
                        int32_t block_m, int32_t block_n, int32_t* cum_tiles,
                        int32_t* num_n_tiles, void* stream) {
  g_last_error.clear();
  if (num_rows < 0 || block_m < 1 || block_n < 1 || !cum_tiles)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "flat schedule arguments");
  if (num_rows > 0 && (!seq_lens || !n_eff || !num_n_tiles))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "null flat schedule input");
  flat_schedule_kernel<<<1, 1024, 0, static_cast<cudaStream_t>(stream)>>>(
      seq_lens, n_eff, num_rows, block_m, block_n, cum_tiles, num_n_tiles);
  return check_launch("flat_schedule_kernel");
}

int plora_sgmv_shrink(const void* x, const void* lora_a, void* tmp, const int32_t* lora_ranks,
                      const int32_t* slot_start, const int32_t* token_index, int64_t num_tokens,
                      int64_t in_features, int64_t max_rank, int32_t num_slots, int32_t stack_num,
                      int32_t dtype, void* stream) {
  g_last_error.clear();
  int st = check_common(dtype, num_slots, max_rank);
  if (st) return st;
  if (in_features < 1 || in_features > INT32_MAX || stack_num < 1)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "in_features/stack_num");
  if (num_tokens == 0) return PLORA_OK;
  if (!x || !lora_a || !tmp || !lora_ranks || !slot_start || !token_index)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "null pointer");
  SegTable seg{slot_start, token_index, num_slots};
  if (num_tokens > (int64_t)INT32_MAX)
    return fail(PLORA_ERR_UNSUPPORTED, "num_tokens exceeds int32 token ids");
  return shrink_impl(x, lora_a, tmp, lora_ranks, seg, num_tokens, in_features, max_rank, stack_num,
                     dtype, static_cast<cudaStream_t>(stream));
}

int plora_sgmv_expand(const void* tmp, const void* lora_b, void* y, const int32_t* lora_ranks,
                      const float* scalings, const int32_t* slot_start, const int32_t* token_index,
                      int64_t num_tokens, int64_t max_rank, int64_t out_features,
                      int32_t num_slots, int32_t dtype, void* stream) {
  g_last_error.clear();
  int st = check_common(dtype, num_slots, max_rank);
  if (st) return st;
  if (out_features < 1 || out_features > INT32_MAX)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "out_features");
  if (num_tokens == 0) return PLORA_OK;
  if (!tmp || !lora_b || !y || !lora_ranks || !scalings || !slot_start || !token_index)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "null pointer");
  SegTable seg{slot_start, token_index, num_slots};
  return expand_impl(tmp, lora_b, y, lora_ranks, scalings, seg, num_tokens, max_rank, out_features,
                     dtype, static_cast<cudaStream_t>(stream));
}

// The fused stream kernel for plora_sgmv_shrink_expand: rank 16, 16-bit types,
// K and N multiples of 512 up to 4096, many tokens, and an expand phase that
// fits the shrink's shared memory.  *launched = false leaves the call to the
// two kernels.
int fused_impl(const void* x, const void* a, void* tmp, const void* b, void* y, const int32_t* ranks,
               const float* scales, SegTable seg, int64_t num_tokens, int64_t K, int64_t R, int64_t N, int32_t dtype,
               cudaStream_t stream, bool* launched) {
  *launched = false;
  if (g_stream_kernels.load(std::memory_order_relaxed) != 2 || dtype == PLORA_DTYPE_F32 || R != kStreamRank ||
      seg.num_slots > kFastPathMaxSlots || !aligned16(x) || !aligned16(a) || !aligned16(tmp) || !aligned16(b) ||
      !aligned16(y) || N % 512 != 0 || N > kStreamMaxDim)
    return PLORA_OK;
  DeviceInfo* di = nullptr;
  int st = device_info(&di);
  if (st) return st;
  if (use_weight_split(num_tokens, di) || !stream_shrink_ok(R, K, num_tokens, seg.num_slots, di)) return PLORA_OK;
  StreamPlan plan;
  FusedPlan fp;
  if (!fused_stream_plan(K, N, seg.num_slots, plan, fp)) return PLORA_OK;
  ShrinkArgs sa;
  sa.x = static_cast<const uint8_t*>(x);
  sa.a = static_cast<const uint8_t*>(a);
  sa.tmp = static_cast<uint8_t*>(tmp);
  sa.ranks = ranks;
  sa.seg = seg;
  sa.K = (int32_t)K;
  sa.R = (int32_t)R;
  sa.stack_num = 1;
  ExpandArgs ea;
  ea.tmp = static_cast<const uint8_t*>(tmp);
  ea.b = static_cast<const uint8_t*>(b);
  ea.y = static_cast<uint8_t*>(y);
  ea.ranks = ranks;
  ea.scales = scales;
  ea.seg = seg;
  ea.R = (int32_t)R;
  ea.N = (int32_t)N;
  const bool bf = dtype == PLORA_DTYPE_BF16;
  // programmatic like the shrink: it reads its inputs only after griddep_wait()
  PLORA_CUDA(launch_kernel(bf ? sgmv_shrink_stream_kernel<true, true> : sgmv_shrink_stream_kernel<false, true>,
                           dim3(di->sm_count), dim3(kShrinkThreads), plan.smem_bytes, stream, true, 0, sa, plan,
                           ea, fp),
             "launch fused sgmv_shrink_stream_kernel");
  *launched = true;
  return check_launch("fused sgmv_shrink_stream_kernel");
}

int plora_sgmv_shrink_expand(const void* x, const void* lora_a, void* tmp, const void* lora_b,
                             void* y, const int32_t* lora_ranks, const float* scalings,
                             const int32_t* slot_start, const int32_t* token_index,
                             int64_t num_tokens, int64_t in_features, int64_t max_rank,
                             int64_t out_features, int32_t num_slots, int32_t dtype,
                             void* stream) {
  g_last_error.clear();
  int st = check_common(dtype, num_slots, max_rank);
  if (st) return st;
  if (in_features < 1 || in_features > INT32_MAX || out_features < 1 || out_features > INT32_MAX)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "in_features/out_features");
  if (num_tokens == 0) return PLORA_OK;
  if (!x || !lora_a || !tmp || !lora_b || !y || !lora_ranks || !scalings || !slot_start ||
      !token_index)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "null pointer");
  if (num_tokens > (int64_t)INT32_MAX)
    return fail(PLORA_ERR_UNSUPPORTED, "num_tokens exceeds int32 token ids");
  SegTable seg{slot_start, token_index, num_slots};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  bool fused = false;
  if ((st = fused_impl(x, lora_a, tmp, lora_b, y, lora_ranks, scalings, seg, num_tokens, in_features, max_rank,
                       out_features, dtype, s, &fused)) || fused)
    return st;
  if ((st = shrink_impl(x, lora_a, tmp, lora_ranks, seg, num_tokens, in_features, max_rank, 1,
                        dtype, s)))
    return st;
  return expand_impl(tmp, lora_b, y, lora_ranks, scalings, seg, num_tokens, max_rank, out_features,
                     dtype, s, /*after_shrink=*/true);
}

int plora_sgmv_a_fwd(const void* x, const void* lora_a, void* tmp, const int32_t* seq_lens,
                     const int64_t* weight_indices, const int32_t* lora_ranks, int64_t num_rows,
                     int64_t max_seq, int64_t in_features, int64_t max_rank, int32_t num_slots,
                     int32_t stack_num, int32_t dtype, void* workspace, size_t workspace_size,
                     void* stream) {
  g_last_error.clear();
  int st = check_common(dtype, num_slots, max_rank);
  if (st) return st;
  if (!token_count_ok(num_rows, max_seq))
    return fail(PLORA_ERR_UNSUPPORTED, "num_rows %lld x max_seq %lld: negative or beyond int32 token ids",
                (long long)num_rows, (long long)max_seq);
  if (num_rows == 0 || max_seq == 0) return PLORA_OK;  // sgmv.py:159-160
  const size_t need = fwd_workspace_bytes(num_rows, max_seq, num_slots);
  if (!workspace || workspace_size < need)
    return fail(PLORA_ERR_WORKSPACE, "workspace %zu < %zu bytes", workspace_size, need);
  FwdWorkspace w = carve_fwd(workspace, num_rows, max_seq, num_slots);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if ((st = build_segments(weight_indices, seq_lens, lora_ranks, num_rows, max_seq, num_slots,
                           w.slot_start, w.token_index, workspace, workspace_size, s)))
    return st;
  return plora_sgmv_shrink(x, lora_a, tmp, lora_ranks, w.slot_start, w.token_index,
                           num_rows * max_seq, in_features, max_rank, num_slots, stack_num, dtype,
                           stream);
}

int plora_sgmv_b_fwd(const void* tmp, const void* lora_b, void* y, const int32_t* seq_lens,
                     const int64_t* weight_indices, const int32_t* lora_ranks,
                     const float* scalings, int64_t num_rows, int64_t max_seq, int64_t max_rank,
                     int64_t out_features, int32_t num_slots, int32_t dtype, void* workspace,
                     size_t workspace_size, void* stream) {
  g_last_error.clear();
  int st = check_common(dtype, num_slots, max_rank);
  if (st) return st;
  if (!token_count_ok(num_rows, max_seq))
    return fail(PLORA_ERR_UNSUPPORTED, "num_rows %lld x max_seq %lld: negative or beyond int32 token ids",
                (long long)num_rows, (long long)max_seq);
  if (num_rows == 0 || max_seq == 0) return PLORA_OK;  // sgmv.py:314-315
  const size_t need = fwd_workspace_bytes(num_rows, max_seq, num_slots);
  if (!workspace || workspace_size < need)
    return fail(PLORA_ERR_WORKSPACE, "workspace %zu < %zu bytes", workspace_size, need);
  FwdWorkspace w = carve_fwd(workspace, num_rows, max_seq, num_slots);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if ((st = build_segments(weight_indices, seq_lens, lora_ranks, num_rows, max_seq, num_slots,
                           w.slot_start, w.token_index, workspace, workspace_size, s)))
    return st;
  return plora_sgmv_expand(tmp, lora_b, y, lora_ranks, scalings, w.slot_start, w.token_index,
                           num_rows * max_seq, max_rank, out_features, num_slots, dtype, stream);
}

int plora_slot_fill(const plora_slot_module* modules, int32_t num_modules, int32_t slot,
                    int32_t num_slots, int64_t max_rank, int32_t dtype, const void* host_image,
                    size_t image_bytes, void* staging, size_t staging_bytes, void* stream) {
  g_last_error.clear();
  if (!valid_dtype(dtype)) return fail(PLORA_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  if (num_modules < 0 || slot < 0 || slot >= num_slots || max_rank < 1)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "slot %d of %d, %d modules", slot, num_slots,
                num_modules);
  if (num_modules == 0) return PLORA_OK;
  if (!modules || !host_image || !staging)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "null pointer");
  if (image_bytes < (size_t)num_modules * sizeof(plora_slot_record))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "image smaller than its records");
  if (staging_bytes < image_bytes)
    return fail(PLORA_ERR_WORKSPACE, "staging %zu < image %zu bytes", staging_bytes, image_bytes);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  PLORA_CUDA(cudaMemcpyAsync(staging, host_image, image_bytes, cudaMemcpyHostToDevice, s),
             "slot image copy");
  const dim3 grid(64, (unsigned)num_modules), block(256);
  const uint8_t* img = static_cast<const uint8_t*>(staging);
  const int64_t nbytes = (int64_t)image_bytes;
  if (elem_size(dtype) == 4)
    slot_fill_kernel<float><<<grid, block, 0, s>>>(modules, num_modules, slot, max_rank, img, nbytes);
  else if (dtype == PLORA_DTYPE_BF16)
    slot_fill_kernel<__nv_bfloat16><<<grid, block, 0, s>>>(modules, num_modules, slot, max_rank, img, nbytes);
  else
    slot_fill_kernel<__half><<<grid, block, 0, s>>>(modules, num_modules, slot, max_rank, img, nbytes);
  return check_launch("slot_fill_kernel");
}

int plora_paged_append(const plora_paged_append_args* args, void* stream) {
  g_last_error.clear();
  if (!args) return fail(PLORA_ERR_INVALID_ARGUMENT, "null arguments");
  const plora_paged_cache& c = args->cache;
  const void *q = args->q, *k = args->k, *v = args->v;
  const int64_t pairs = args->pairs, max_new = args->max_new, rows = c.rows;
  AppendParams p = {};
  int st = paged_view(&p.c, c, q ? c.heads : 0);
  if (st) return st;
  if (max_new < 0 || pairs < 0 || pairs > c.head_dim / 2)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "max_new negative, or %lld rotated pairs in a head of %lld",
                (long long)pairs, (long long)c.head_dim);
  const int dtype = (int)c.dtype, head_dim = (int)c.head_dim, kv_heads = (int)c.kv_heads;
  if (!token_count_ok(rows, max_new)) return fail(PLORA_ERR_UNSUPPORTED, "rows * max_new beyond int32");
  if (rows == 0 || max_new == 0) return PLORA_OK;
  if (!k || !v || !args->past_lens || (q && !args->q_out) || (pairs && !args->phases))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "null pointer");
  const int64_t vec = 16 / (int64_t)elem_size(dtype);
  const int64_t strides[9] = {q ? args->q_row_stride : 0, q ? args->q_token_stride : 0, q ? args->q_head_stride : 0,
                              args->k_row_stride, args->k_token_stride, args->k_head_stride,
                              args->v_row_stride, args->v_token_stride, args->v_head_stride};
  for (int64_t x : strides)
    if (x < 0 || x % vec) return fail(PLORA_ERR_INVALID_ARGUMENT, "token strides must be multiples of 16 bytes");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(args->q_out) ||
      !aligned16(args->k_out))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "token pointers must be 16-byte aligned");
  // halves of one buffer's pages interleave; keys and values in one place would not both last
  const int64_t page_elems = c.kv_heads * c.page_size * c.head_dim, el = (int64_t)elem_size(dtype);
  if (c.k_cache == c.v_cache ||
      rows_meet(c.k_cache, c.k_page_stride, c.v_cache, c.v_page_stride, c.num_pages, page_elems, el))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "k_cache and v_cache share memory");
  DeviceInfo* di = nullptr;
  if ((st = device_info(&di))) return st;
  p.q = q, p.k = k, p.v = v, p.q_out = args->q_out, p.k_out = args->k_out;
  p.q_row = strides[0], p.q_tok = strides[1], p.q_head = strides[2];
  p.k_row = strides[3], p.k_tok = strides[4], p.k_head = strides[5];
  p.v_row = strides[6], p.v_tok = strides[7], p.v_head = strides[8];
  p.past = args->past_lens, p.news = args->new_lens;
  p.phases = reinterpret_cast<const uint64_t*>(args->phases);
  p.q_heads = q ? (int32_t)c.heads : 0;
  p.pairs = (int32_t)pairs, p.interleaved = args->interleaved != 0, p.scale = (float)args->rotary_scale;
  p.max_new = (int32_t)max_new, p.tokens = (int32_t)(rows * max_new);
  // one token a CTA until that fills the SMs
  p.cta_tokens = p.tokens <= 8 * di->sm_count ? 1 : kAppendTokens;
  const int n = (int)vec, per_head = (head_dim / n + 1) / 2;
  p.by_new.set((uint32_t)max_new);
  p.by_head.set((uint32_t)per_head);
  p.by_item.set((uint32_t)(per_head * (p.q_heads + 2 * kv_heads)));
  const bool whole = p.interleaved ? 2 * pairs % n == 0 : pairs % n == 0;
  const unsigned grid = (unsigned)((p.tokens + p.cta_tokens - 1) / p.cta_tokens);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = dtype == PLORA_DTYPE_F32   ? launch_append<float>(p, whole, grid, s)
                  : dtype == PLORA_DTYPE_F16 ? launch_append<__half>(p, whole, grid, s)
                                             : launch_append<__nv_bfloat16>(p, whole, grid, s);
  PLORA_CUDA(e, "launch paged_append_kernel");
  return PLORA_OK;
}

size_t plora_paged_attention_workspace(int64_t rows, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                       int32_t page_size, int64_t max_pages, int64_t window, int32_t dtype) {
  if (!valid_dtype(dtype) || rows < 0 || rows > kPagedMaxRows || kv_heads < 1 || heads < 1 || heads % kv_heads ||
      heads > 65535 || head_dim < 1 || head_dim > 256 || head_dim % 8 || page_size < 1 || max_pages < 1 ||
      max_pages > INT32_MAX / page_size || window < 0)
    return 0;
  return attn_plan(rows, heads, kv_heads, head_dim, max_pages * page_size, window, dtype).bytes;
}

int plora_paged_attention(const plora_paged_attention_args* args, void* stream) {
  g_last_error.clear();
  if (!args) return fail(PLORA_ERR_INVALID_ARGUMENT, "null arguments");
  const plora_paged_cache& c = args->cache;
  const int64_t rows = c.rows, window = args->window;
  const void* q = args->q;
  AttnParams p = {};
  int st = paged_view(&p.c, c, c.heads);
  if (st) return st;
  const int dtype = (int)c.dtype, heads = (int)c.heads, kv_heads = (int)c.kv_heads, head_dim = (int)c.head_dim;
  if (heads < 1) return fail(PLORA_ERR_INVALID_ARGUMENT, "no heads");
  if (window < 0) return fail(PLORA_ERR_INVALID_ARGUMENT, "window %lld is negative", (long long)window);
  if (rows == 0) return PLORA_OK;
  if (!q || !args->seq_lens || !args->out) return fail(PLORA_ERR_INVALID_ARGUMENT, "null pointer");
  const int64_t vec = 16 / (int64_t)elem_size(dtype);
  if (args->q_row_stride < 0 || args->q_head_stride < 0 || args->q_row_stride % vec || args->q_head_stride % vec ||
      !aligned16(q) || !aligned16(args->out))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "q and out must be 16-byte aligned, with q's strides multiples of 16 bytes");
  const AttnPlan a = attn_plan(rows, heads, kv_heads, head_dim, p.c.capacity, window, dtype);
  if (a.bytes && (!args->workspace || args->workspace_size < (int64_t)a.bytes))
    return fail(PLORA_ERR_WORKSPACE, "attention workspace %lld < %zu bytes", (long long)args->workspace_size, a.bytes);
  if (reinterpret_cast<uintptr_t>(args->workspace) % 256)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
  if (args->q_row_stride > INT64_MAX / 16 / rows || args->q_head_stride > INT64_MAX / 16 / heads)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "size of q overflows");
  const int64_t el = (int64_t)elem_size(dtype);
  // in place each query is read before its output is written, and by no other item
  const bool in_place = q == args->out && (heads == 1 || args->q_head_stride == head_dim) &&
                        (rows == 1 || args->q_row_stride == (int64_t)heads * head_dim);
  if (!in_place && ranges_meet(q, ((rows - 1) * args->q_row_stride + (heads - 1) * args->q_head_stride + head_dim) * el,
                               args->out, rows * heads * head_dim * el))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "out shares memory with q and is not q");
  DeviceInfo* di = nullptr;
  if ((st = device_info(&di))) return st;
  p.q = q, p.out = args->out, p.seq_lens = args->seq_lens;
  p.q_row = args->q_row_stride, p.q_head = args->q_head_stride;
  p.rows = (int32_t)rows, p.group = heads / kv_heads, p.blocks = a.blocks, p.block_heads = a.block_heads;
  p.window = (int32_t)std::min<int64_t>(window, INT32_MAX);
  p.scale_log2 = (float)(args->scale * 1.4426950408889634);  // log2(e)
  uint8_t* ws = static_cast<uint8_t*>(args->workspace);
  p.work = reinterpret_cast<AttnWork*>(ws);
  p.before = reinterpret_cast<int64_t*>(ws + a.before_offset);
  p.cut = reinterpret_cast<int4*>(ws + a.cut_offset);
  p.cut_room = a.segments;
  p.part_ml = reinterpret_cast<float2*>(ws + a.ml_offset);
  p.part_o = reinterpret_cast<float*>(ws + a.part_offset);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  p.direct = a.direct;
  CUtensorMap mk = {}, mv = {};
  const bool tma = attn_by_tma(p.c, a);
  if (tma && ((st = make_map_cache(&mk, c.k_cache, dtype, p.c, c.k_page_stride)) ||
              (st = make_map_cache(&mv, c.v_cache, dtype, p.c, c.v_page_stride))))
    return st;
  PLORA_CUDA(launch_attn(p, a, dtype, tma, mk, mv, s), "launch paged attention");
  return PLORA_OK;
}

size_t plora_logit_rules_workspace(int64_t rows, int64_t vocab, int64_t history, int64_t biases) {
  if (rows < 0 || rows > 65535 || vocab < 0 || vocab > (1 << 30) || history < 0 || history > (1 << 30) - 1 ||
      biases < 0 || biases > kRulesMaxBiases)
    return 0;
  return rules_plan(rows, vocab, history, biases, true).bytes;
}

int plora_logit_rules(const plora_logit_rules_args* args, void* stream) {
  g_last_error.clear();
  if (!args) return fail(PLORA_ERR_INVALID_ARGUMENT, "null arguments");
  const void *logits = args->logits, *tokens = args->tokens, *bias_tokens = args->bias_tokens;
  void *out = args->out, *workspace = args->workspace;
  const int64_t rows = args->rows, vocab = args->vocab, history = args->history, biases = args->biases;
  const int64_t logits_stride = args->logits_stride, out_stride = args->out_stride;
  if (args->dtype < 0 || args->dtype > INT32_MAX || !valid_dtype((int)args->dtype))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "unknown dtype %lld", (long long)args->dtype);
  const int dtype = (int)args->dtype;
  if (rows < 0 || vocab < 0 || history < 0 || biases < 0)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "negative rows, vocab, history or biases");
  if (args->token_bytes != 4 && args->token_bytes != 8)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "token ids of %lld bytes", (long long)args->token_bytes);
  if (rows > 65535 || vocab > (1 << 30) || history > (1 << 30) - 1 || biases > kRulesMaxBiases)
    return fail(PLORA_ERR_UNSUPPORTED, "rows > 65535, vocab or history beyond 2^30, or more than %d biases a row",
                kRulesMaxBiases);
  if (rows == 0 || vocab == 0) return PLORA_OK;
  if (!logits || !out || (history && !tokens) || (biases && (!bias_tokens || !args->bias_values)))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "null pointer");
  if (logits_stride < vocab || out_stride < vocab || (history && args->tokens_stride < 0) ||
      (biases && (args->bias_tokens_stride < 0 || args->bias_values_stride < 0)) ||
      (args->allowed && args->allowed_stride < 0))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "row strides below the vocabulary, or negative");
  const RulesPlan a = rules_plan(rows, vocab, history, biases, logits != out || logits_stride != out_stride || args->allowed);
  if (a.bytes && (!workspace || args->workspace_size < (int64_t)a.bytes))
    return fail(PLORA_ERR_WORKSPACE, "logit rules workspace %lld < %zu bytes", (long long)args->workspace_size, a.bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
  const uintptr_t el = elem_size(dtype) - 1;
  if ((reinterpret_cast<uintptr_t>(logits) & el) || (reinterpret_cast<uintptr_t>(out) & el))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "logits or out not aligned to its type");
  if (logits_stride > INT64_MAX / 16 / rows || out_stride > INT64_MAX / 16 / rows)
    return fail(PLORA_ERR_INVALID_ARGUMENT, "size of logits or out overflows");
  if (rows_meet(logits, logits_stride, out, out_stride, rows, vocab, (int64_t)elem_size(dtype)))
    return fail(PLORA_ERR_INVALID_ARGUMENT, "out shares memory with logits and is not logits");
  DeviceInfo* di = nullptr;
  int st = device_info(&di);
  if (st) return st;
  RulesParams p = {};
  p.x = logits, p.y = out, p.x_row = logits_stride, p.y_row = out_stride, p.vocab = vocab;
  p.tokens = tokens, p.token_row = args->tokens_stride, p.history = (int32_t)history;
  p.token_lens = args->token_lens, p.prompt_lens = args->prompt_lens;
  p.repetition = args->repetition, p.presence = args->presence, p.frequency = args->frequency;
  p.bias_tokens = bias_tokens, p.bias_row = args->bias_tokens_stride;
  p.bias_values = args->bias_values, p.value_row = args->bias_values_stride, p.biases = (int32_t)biases;
  p.allowed = reinterpret_cast<const uint32_t*>(args->allowed), p.mask_row = args->allowed_stride;
  p.part = a.part;
  if (a.lists) {
    p.list = static_cast<RulesEntry*>(workspace);
    p.listed = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + a.listed_offset);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = args->token_bytes == 8;
  cudaError_t e = dtype == PLORA_DTYPE_F32   ? launch_rules<float>(p, a, wide, rows, s)
                  : dtype == PLORA_DTYPE_F16 ? launch_rules<__half>(p, a, wide, rows, s)
                                             : launch_rules<__nv_bfloat16>(p, a, wide, rows, s);
  PLORA_CUDA(e, "launch logit rules");
  return PLORA_OK;
}

// Device address of g_noalloc_scratch, looked up once per device and CUDA
// context with that device current (the first plora_sgmv_a_fwd_noalloc call
// there).  The cache is keyed on the context's unique id: after
// cudaDeviceReset the module is loaded again in a new context, and the array
// may live at another address.
namespace {
struct NoallocScratch {
  unsigned long long ctx_id = 0;
  void* ptr = nullptr;
};
NoallocScratch g_noalloc[kMaxDevices];
std::mutex g_noalloc_mu;

// Unique id of the calling thread's current CUDA context (0 if unavailable).
unsigned long long current_context_id() {
  using GetCurrent = CUresult (*)(CUcontext*);
  using GetId = CUresult (*)(CUcontext, unsigned long long*);
  static GetCurrent get_current = nullptr;
  static GetId get_id = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuCtxGetCurrent", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      get_current = reinterpret_cast<GetCurrent>(p);
    if (cudaGetDriverEntryPoint("cuCtxGetId", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      get_id = reinterpret_cast<GetId>(p);
  });
  CUcontext ctx = nullptr;
  unsigned long long id = 0;
  if (!get_current || !get_id || get_current(&ctx) != CUDA_SUCCESS || !ctx || get_id(ctx, &id) != CUDA_SUCCESS)
    return 0;
  return id;
}

int noalloc_scratch(void** out) {
  int dev = 0;
  PLORA_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(PLORA_ERR_UNSUPPORTED, "device ordinal %d", dev);
  std::lock_guard<std::mutex> lk(g_noalloc_mu);
  NoallocScratch& e = g_noalloc[dev];
  const unsigned long long id = current_context_id();  // 0 before the runtime set one up
  if (!e.ptr || id == 0 || e.ctx_id != id) {
    void* p = nullptr;
    // also makes the runtime's context for `dev` current on this thread
    PLORA_CUDA(cudaGetSymbolAddress(&p, g_noalloc_scratch), "cudaGetSymbolAddress(noalloc scratch)");
    e.ptr = p;
    e.ctx_id = current_context_id();
  }
  *out = e.ptr;
  return PLORA_OK;
}
}  // namespace

extern "C" int plora_sgmv_a_fwd_noalloc(const void* x, const void* lora_a, void* tmp,
                                        const int32_t* seq_lens, const int64_t* weight_indices,
                                        const int32_t* lora_ranks, int64_t num_rows,
                                        int64_t max_seq, int64_t in_features, int64_t max_rank,
                                        int32_t num_slots, int32_t stack_num, int32_t dtype,
                                        void* stream) {
  g_last_error.clear();
  int st = check_common(dtype, num_slots, max_rank);
  if (st) return st;
  if (num_rows < 0 || max_seq < 0) return fail(PLORA_ERR_INVALID_ARGUMENT, "negative num_rows/max_seq");
  if (!token_count_ok(num_rows, max_seq))
    return fail(PLORA_ERR_UNSUPPORTED, "num_rows %lld x max_seq %lld exceeds int32 token ids",
                (long long)num_rows, (long long)max_seq);
  if (num_rows == 0 || max_seq == 0) return PLORA_OK;
  const size_t need = fwd_workspace_bytes(num_rows, max_seq, num_slots);
  if (need > (size_t)PLORA_NOALLOC_SCRATCH_BYTES)
    return fail(PLORA_ERR_UNSUPPORTED,
                "batch needs %zu bytes of scratch; the static scratch of plora_sgmv_a_fwd_noalloc "
                "holds %u bytes (use plora_sgmv_a_fwd with a workspace)",
                need, (unsigned)PLORA_NOALLOC_SCRATCH_BYTES);
  void* scratch = nullptr;
  if ((st = noalloc_scratch(&scratch))) return st;
  FwdWorkspace w = carve_fwd(scratch, num_rows, max_seq, num_slots);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if ((st = build_segments(weight_indices, seq_lens, lora_ranks, num_rows, max_seq, num_slots,
                           w.slot_start, w.token_index, scratch, need, s)))
    return st;
  return plora_sgmv_shrink(x, lora_a, tmp, lora_ranks, w.slot_start, w.token_index,
                           num_rows * max_seq, in_features, max_rank, num_slots, stack_num, dtype,
                           stream);
}

}  // extern "C"
