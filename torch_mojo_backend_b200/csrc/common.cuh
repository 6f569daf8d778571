// Shared declarations between the host entry points (api.cu) and the kernel translation
// units.  Everything here is internal to the library; the public surface is include/b200fa.h.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200fa {

// A validated (B, H, S, D) view: base pointer plus element strides (D stride is 1).
struct View4 {
  void* ptr;
  int64_t sb, sh, ss;
};

// Dropout: element (b, h, i, j) of the attention matrix is kept when its byte of a
// Philox4x32-10 stream keyed by `seed` is >= `threshold` (see philox.cuh); kept probabilities
// are multiplied by `inv_keep` = 1 / (1 - p).  threshold == 0 means no dropout.
struct DropoutParams {
  uint64_t seed;
  uint64_t offset;
  uint32_t threshold;  // 0..255: bytes below it are dropped
  float inv_keep;
};

struct FwdParams {
  View4 q, k, v, out;
  float* lse;        // (B, Hq, Sq) fp32 contiguous
  int B, Hq, Hkv, Sq, Sk, D;
  int causal;        // 0: no mask; otherwise query row i sees key column j iff j <= i + causal_off
  int causal_off;    // 0 (top-left aligned diagonal) or Sk - Sq (bottom-right aligned)
  int window, sinks; // window > 0 (causal only): row i sees the last `window` of those keys and the first `sinks`; 0: all of them
  float scale;       // softmax scale
  float scale_log2;  // scale * log2(e)
  uint32_t* status;  // optional device status word
  int64_t whole_heads;    // batch * query heads of the problem this one is a piece of (its own, if it is whole)
  int tiles_per_cta;      // forward kernel shape: 0 = chosen by the launcher, 1 or 2 = forced
  long long wait_budget;  // SM cycles any single internal wait may take before the kernel gives up
  DropoutParams drop;
};

struct BwdParams {
  View4 q, k, v, out, dout, dq, dk, dv;
  const float* lse;  // (B, Hq, S) fp32 contiguous (natural log)
  float* dpsum;      // workspace: (B, Hq, Spad) rowsum(dO * O)   (the tensor-core route stores both
  float* lse_log2;   // workspace: (B, Hq, Spad) lse * log2(e)     statistics negated, the SIMT route as is)
  int B, Hq, Hkv, S, Sk, Spad, D;   // S: query rows (Spad: padded to 128); Sk: key rows
  int causal;
  int causal_off;
  int window, sinks;   // as in FwdParams
  int sink_chunks;     // blocks that share the query rows of a K/V tile with sinks in it (1: none do)
  float* sink_part;    // workspace, if sink_chunks > 1: their dV and dK, (B, Hkv, tiles with sinks, sink_chunks, 2, 128, D)
  float scale;
  float scale_log2;
  uint32_t* status;
  long long wait_budget;
  int parts;  // bit 0 preprocess, bit 1 dK/dV kernel, bit 2 dQ kernel (7 = the whole backward)
  DropoutParams drop;
};

// Split-KV forward for short query blocks (decode): partial (max, sum, O) per key split.
struct SplitKvParams {
  View4 q, k, v, out;
  float* lse;
  float* part_o;    // workspace: (B, Hq, Sq, nsplit, D) fp32
  float* part_ml;   // workspace: (B, Hq, Sq, nsplit, 2) fp32: running max (log2 domain), row sum
  unsigned* counters;   // workspace: (B, Hkv) splits finished so far, zeroed before the launch
  int B, Hq, Hkv, Sq, Sk, D;
  int causal, causal_off;
  int nsplit, split_len;   // keys per split (a multiple of 64)
  float scale, scale_log2;
};

// The blocks of `kRows` keys that query rows at positions p_first .. p_last visit under a window: those with one of the first
// `sinks` keys, then the ones from the window of p_first on.  Rows at p_first with a smaller p_last visit a prefix of the list.
struct KeyBlocks {
  int n_sink;   // leading blocks 0 .. n_sink - 1
  int first;    // block that follows them
  int n;        // blocks in all; 0: no row sees a key
  __host__ __device__ __forceinline__ int at(int i) const { return i < n_sink ? i : first + (i - n_sink); }
};
template <int kRows>
__host__ __device__ __forceinline__ KeyBlocks window_blocks(int p_first, int p_last, int Sk, int window, int sinks) {
  const int last = p_last < Sk - 1 ? p_last : Sk - 1;   // last key that any of the rows sees
  KeyBlocks r = {0, 0, 0};
  if (last < 0) return r;
  const int begin = p_first - window + 1;
  const int first = begin > 0 ? begin / kRows : 0;
  const int n_sink = ((sinks < last + 1 ? sinks : last + 1) + kRows - 1) / kRows;
  if (first <= n_sink) {   // no gap
    r.n = last / kRows + 1;
    return r;
  }
  r.n_sink = n_sink;
  r.first = first;
  r.n = n_sink + (last / kRows >= first ? last / kRows - first + 1 : 0);
  return r;
}

constexpr int kSplitkvCluster = 16;   // splits of a KV head that may merge as a cluster

// A validated paged cache of B sequences (see paged.cu).
struct PagedCache {
  void *k, *v;                  // (pages, Hkv, page, D) 16-bit elements or D / 2 bytes of codes
  void *k_scales, *v_scales;    // 4 bits: (pages, Hkv, page, D / 32, 2)
  const int32_t* table;         // (B, table_stride)
  const int32_t* lengths;       // (B): tokens in the cache, the new ones included
  const int32_t* new_lengths;   // (B) or null: all of a call's S tokens are new
  int64_t table_stride;
  int B, Hkv, D, bits;
  int shift;                    // log2 of the page size
  int pages, capacity;          // of the pool; tokens that a row of the table has pages for
  uint32_t* status;
};
struct AppendParams {
  PagedCache c;
  View4 q, k, v, q_out;         // (B, H, S, D); q and q_out only if Hq > 0
  const float *cos, *sin;       // (positions, rotary / 2)
  int Hq, S, rotary, positions, interleaved;
  int clear;                    // rows of q_out that no new token has become zero, or NaN by a bad index
};
struct GatherParams {
  PagedCache c;
  View4 k, v;                   // (B, Hkv, S, D)
  int S;
};
struct AttendParams {
  PagedCache c;
  View4 q, out;                 // (B, Hq, S, D)
  float* lse;                   // (B, Hq, S)
  int Hq, S, window, sinks;     // window 0: none
  int peers, teams, group;      // set by the launcher: blocks of a cluster, clusters that share a unit, query heads of a KV head
  float* parts;                 // workspace, if teams > 1: rows and (max, sum) of every team (merge in paged.cu)
  long long wait_budget;        // SM cycles that a wait for a copy may take
  float scale_log2;
  uint32_t one_f16, one_bf16;   // kOneF16, kOneBf16 (paged.cu)
};

// mask of a tensor-core kernel: every key, the causal diagonal, or the diagonal with a window and sinks
constexpr int kAll = 0, kCausalMask = 1, kWindowMask = 2;

// dtype tags shared with the C header
constexpr int kF32 = 0, kBF16 = 1, kF16 = 2;

// Launchers implemented in the kernel translation units.  Each returns a cudaError_t and
// adds the number of kernels it enqueued to *launches.
cudaError_t launch_fwd_sm100(const FwdParams& p, int dtype, cudaStream_t stream, int* launches);
int fwd_splits(const FwdParams& p);   // CTAs that share a query unit's K/V blocks in launch_fwd_sm100 (host only)
cudaError_t launch_fwd_simt(const FwdParams& p, int dtype, cudaStream_t stream, int* launches);
cudaError_t launch_fwd_fp32(const FwdParams& p, cudaStream_t stream, int* launches);   // fp32 on the tensor cores
cudaError_t launch_bwd_fp32(const BwdParams& p, cudaStream_t stream, int* launches);   // ... head dim 64
cudaError_t launch_fwd_splitkv(const SplitKvParams& p, int dtype, cudaStream_t stream, int* launches);
cudaError_t launch_bwd_sm100(const BwdParams& p, int dtype, cudaStream_t stream, int* launches);
cudaError_t launch_bwd_simt(const BwdParams& p, int dtype, cudaStream_t stream, int* launches);
// sink_chunks of the tensor-core and the SIMT backward, and the key rows of a tile of theirs (host only; sizes, window and sinks are read)
int bwd_sink_chunks(const BwdParams& p, int* tile_rows);
int simt_sink_chunks(const BwdParams& p, int* tile_rows);
// How many blocks share the steps of a key tile with sinks in it.  Every query row behind such a tile sees it, so its block runs a step
// for every tile of query rows where the others run a window's; with few heads it would outlast all of them.  A share is at most
// a quarter of what each of `slots` blocks has to do in all, and at least `least` steps (it leaves two fp32 tiles to be added up).
inline int sink_chunks_for(int64_t pairs, int64_t tiles, int64_t sink_tiles, int64_t sink_steps, int64_t other_steps, int64_t slots, int64_t least) {
  if (sink_tiles == 0) return 1;
  const int64_t all = pairs * (sink_tiles * sink_steps + (tiles - sink_tiles) * other_steps);
  int64_t chunks = (4 * slots * sink_steps + all - 1) / all;
  if (chunks > sink_steps / least) chunks = sink_steps / least;
  return static_cast<int>(chunks < 1 ? 1 : chunks > 64 ? 64 : chunks);
}
cudaError_t launch_paged_append(const AppendParams& p, int dtype, cudaStream_t stream, int* launches);
cudaError_t launch_paged_gather(const GatherParams& p, int dtype, cudaStream_t stream, int* launches);
// `keys`: the most that a query row can see, as far as the host knows; `part_bytes` at p.parts
cudaError_t launch_paged_attention(const AttendParams& p, int dtype, int64_t keys, size_t part_bytes, cudaStream_t stream, int* launches);
// How such a call's keys are shared on the current device: blocks of a cluster, clusters of a unit, warps of a block (p: c, Hq, S)
cudaError_t paged_shares(const AttendParams& p, int dtype, int64_t keys, size_t part_bytes, int* peers, int* teams, int* warps);
// Bytes of a team's part, and how many teams (clusters that share a unit) are worth a workspace for a call that sees `keys` keys
size_t paged_part_bytes(int64_t batch, int64_t heads_q, int64_t heads_kv, int64_t S, int64_t D);
int paged_teams(int64_t batch, int64_t heads_q, int64_t heads_kv, int64_t S, int64_t keys);
// A one-warp kernel whose only job is to wait, with `budget` SM cycles, on a barrier nobody
// arrives at: exercises the bounded-wait give-up path without touching the attention kernels.
cudaError_t launch_wait_timeout_selftest(uint32_t* status, long long budget, cudaStream_t stream, int* launches);

// In the dK/dV kernels, by the threads that read the row statistics: waits for the kernel that wrote them and lets the dQ
// kernel start.  The dQ kernel does not wait for that one itself: it starts when every block has been here, and the fence
// orders what this thread has been shown ahead of that.  It reads the statistics from L2 (__ldcg), never through an L1
// line that may be older.
__device__ __forceinline__ void let_the_dq_kernel_start() {
  cudaGridDependencySynchronize();
  __threadfence();
  cudaTriggerProgrammaticLaunchCompletion();
}

// A launch that, if `early`, may start as soon as every block of the kernel ahead of it on the stream has allowed it.
template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kern)(Params...), dim3 grid, int threads, int smem, cudaStream_t stream, bool early, Args... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Encodes a 4-D tiled tensor map over a (B,H,S,D) view of 16-bit elements with a
// {64 x box_rows x 1 x 1} box and 128-byte swizzle.  Returns false if the driver entry
// point is unavailable or the encode fails.
bool encode_map_16bit(CUtensorMap* map, const View4& t, int B, int H, int S, int D, int box_rows, bool bf16);

}  // namespace b200fa
