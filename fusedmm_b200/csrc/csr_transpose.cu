// csr_transpose.cu -- the transposed pattern of a CSR (include/fusedmm_b200.h, fusedmm_b200_csr_transpose): for every column
// the rows of its edges in the order of the edges.  A backward pass over the columns gathers through it, so no sum needs an
// atomic and its order is the same on every run.
//
// A stable radix sort of the edges by column, 8 bits a pass, least significant digit first; edges whose column id is
// outside [0, n) get the key n and stay behind the last column.  A pass is three launches: the digit counts of every tile
// of edges, their running sums (one block per digit), and the move.  Inside a tile a warp owns a run of consecutive edges
// and ranks them 32 at a time: lanes with the same digit find each other with match.any, the earlier lanes and the warp's
// count so far give the place.  Bytes of an edge: 16 in the first pass (32-bit ids), 20 in each other, 24 for rows and positions at
// the end: 2^23 edges of 2^19 columns take 451 us, and these bytes need 103.
#include "../../include/fusedmm_b200.h"
#include "attn_common.cuh"
#include "attn_host.h"

namespace fmm {
namespace attn {

constexpr int TR_THREADS = 256, TR_WARPS = TR_THREADS / 32;
// Edges of a tile: TR_THREADS * TR_ROUNDS (524288 edges: 57 us a transposition with 16 rounds, 44 with 4; 2^23 edges: 564 and 453).
constexpr int TR_ROUNDS = 4;
constexpr int TR_DIGITS = 256;

__device__ __forceinline__ long long load_int(const void *p, int is64, long long i)
{
   return is64 ? __ldg(static_cast<const long long *>(p) + i) : static_cast<long long>(__ldg(static_cast<const int *>(p) + i));
}

struct SortParams {
   const void *colidx, *rowptr;  // first pass: keys come from colidx, edge ids are the positions
   int idx64, ptr64;
   long long m, n, nnz, tiles;
   const unsigned *key_in, *edge_in;
   unsigned *key_out, *edge_out;
   unsigned *counts;  // [digit][tile]
   unsigned *totals;  // [digit]
   int shift;
};

// the edges the row pointers cover are a run [first, last); what colidx holds around it belongs to no row
__device__ __forceinline__ unsigned first_key(const SortParams &p, long long e)
{
   const long long first = load_int(p.rowptr, p.ptr64, 0), last = load_int(p.rowptr, p.ptr64, p.m);
   const long long c = e >= first && e < last ? load_int(p.colidx, p.idx64, e) : -1;
   return c >= 0 && c < p.n ? static_cast<unsigned>(c) : static_cast<unsigned>(p.n);
}

template <bool FIRST>
__global__ void __launch_bounds__(TR_THREADS) sort_count_kernel(const SortParams p)
{
   __shared__ unsigned count[TR_DIGITS];
   count[threadIdx.x] = 0;
   __syncthreads();
   const long long base = static_cast<long long>(blockIdx.x) * TR_THREADS * TR_ROUNDS;
   for (int r = 0; r < TR_ROUNDS; r++) {
      const long long e = base + r * TR_THREADS + threadIdx.x;
      if (e >= p.nnz) break;
      const unsigned key = FIRST ? first_key(p, e) : p.key_in[e];
      atomicAdd(&count[(key >> p.shift) & (TR_DIGITS - 1)], 1u);
   }
   __syncthreads();
   p.counts[threadIdx.x * p.tiles + blockIdx.x] = count[threadIdx.x];
}

// counts[digit][*] -> exclusive running sums over the tiles; totals[digit]
__global__ void __launch_bounds__(TR_THREADS) sort_scan_kernel(const SortParams p)
{
   __shared__ unsigned warp_sum[TR_WARPS];
   unsigned *c = p.counts + blockIdx.x * p.tiles;
   const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
   unsigned carry = 0;
   for (long long base = 0; base < p.tiles; base += TR_THREADS) {
      const long long t = base + threadIdx.x;
      const unsigned v = t < p.tiles ? c[t] : 0u;
      unsigned s = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
         const unsigned o = __shfl_up_sync(FULL, s, d);
         if (lane >= d) s += o;
      }
      if (lane == 31) warp_sum[w] = s;
      __syncthreads();
      unsigned before = carry, all = 0;
      for (int i = 0; i < TR_WARPS; i++) {
         if (i < w) before += warp_sum[i];
         all += warp_sum[i];
      }
      if (t < p.tiles) c[t] = before + s - v;
      carry += all;
      __syncthreads();
   }
   if (threadIdx.x == 0) p.totals[blockIdx.x] = carry;
}

template <bool FIRST>
__global__ void __launch_bounds__(TR_THREADS) sort_move_kernel(const SortParams p)
{
   __shared__ unsigned place[TR_WARPS][TR_DIGITS];  // first the warp's counts, then where its next edge of the digit goes
   __shared__ unsigned warp_sum[TR_WARPS];
   const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
   for (int i = 0; i < TR_WARPS; i++) place[i][threadIdx.x] = 0;
   __syncthreads();
   const long long base = (static_cast<long long>(blockIdx.x) * TR_THREADS + w * 32) * TR_ROUNDS;
   unsigned key[TR_ROUNDS], rank[TR_ROUNDS];
   const unsigned lower = (1u << lane) - 1;
#pragma unroll
   for (int r = 0; r < TR_ROUNDS; r++) {
      const long long e = base + r * 32 + lane;
      const bool live = e < p.nnz;
      key[r] = !live ? 0u : FIRST ? first_key(p, e) : p.key_in[e];
      const unsigned digit = live ? (key[r] >> p.shift) & (TR_DIGITS - 1) : TR_DIGITS + 1;
      const unsigned same = __match_any_sync(FULL, digit);
      const unsigned before = live ? place[w][digit] : 0u;
      rank[r] = before + __popc(same & lower);
      __syncwarp();
      if (live && (same & lower) == 0) place[w][digit] = before + __popc(same);
      __syncwarp();
   }
   __syncthreads();
   // thread d: where the digit d starts, in all and for this tile, then for each warp of the tile
   const unsigned total = p.totals[threadIdx.x];
   unsigned s = total;
#pragma unroll
   for (int d = 1; d < 32; d <<= 1) {
      const unsigned o = __shfl_up_sync(FULL, s, d);
      if (lane >= d) s += o;
   }
   if (lane == 31) warp_sum[w] = s;
   __syncthreads();
   unsigned at = s - total + p.counts[threadIdx.x * p.tiles + blockIdx.x];
   for (int i = 0; i < w; i++) at += warp_sum[i];
   for (int i = 0; i < TR_WARPS; i++) {
      const unsigned c = place[i][threadIdx.x];
      place[i][threadIdx.x] = at;
      at += c;
   }
   __syncthreads();
#pragma unroll
   for (int r = 0; r < TR_ROUNDS; r++) {
      const long long e = base + r * 32 + lane;
      if (e >= p.nnz) continue;
      const unsigned to = place[w][(key[r] >> p.shift) & (TR_DIGITS - 1)] + rank[r];
      p.key_out[to] = key[r];
      p.edge_out[to] = FIRST ? static_cast<unsigned>(e) : p.edge_in[e];
   }
}

// first position in the sorted keys that is not below v
__device__ __forceinline__ long long key_lower_bound(const unsigned *keys, long long count, unsigned v)
{
   long long lo = 0, hi = count;
   while (lo < hi) {
      const long long mid = (lo + hi) >> 1;
      if (keys[mid] < v) lo = mid + 1;
      else hi = mid;
   }
   return lo;
}

// t_rowptr[c] = first sorted edge of a column not below c
__global__ void __launch_bounds__(256) transpose_ptr_kernel(const unsigned *keys, long long nnz, long long n, void *t_rowptr, int ptr64)
{
   const long long c = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
   if (c > n) return;
   const long long t = key_lower_bound(keys, nnz, static_cast<unsigned>(c));
   if (ptr64) static_cast<long long *>(t_rowptr)[c] = t;
   else static_cast<int *>(t_rowptr)[c] = static_cast<int>(t);
}

// the row of every edge: a warp per row writes the row's index over its edges
__global__ void __launch_bounds__(256) edge_rows_kernel(const void *rowptr, int ptr64, long long m, long long nnz, int *row_of)
{
   const long long u = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 5;
   if (u >= m) return;
   const long long b = load_int(rowptr, ptr64, u), e = load_int(rowptr, ptr64, u + 1);
   for (long long i = (b < 0 ? 0 : b) + (threadIdx.x & 31); i < e && i < nnz; i += 32) row_of[i] = static_cast<int>(u);
}

__global__ void __launch_bounds__(256) transpose_rows_kernel(const unsigned *edge, const int *row_of, long long nnz, int *t_row, int *t_edge)
{
   const long long t = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
   if (t >= nnz) return;
   const unsigned e = edge[t];
   t_row[t] = row_of[e];
   if (t_edge) t_edge[t] = static_cast<int>(e);
}

namespace {

long long round256(long long b) { return (b + 255) / 256 * 256; }
long long sort_tiles(long long nnz) { return (nnz + TR_THREADS * TR_ROUNDS - 1) / (TR_THREADS * TR_ROUNDS); }

void sort_pass(const SortParams &p, cudaStream_t st)
{
   const unsigned grid = static_cast<unsigned>(p.tiles);
   if (p.shift == 0) sort_count_kernel<true><<<grid, TR_THREADS, 0, st>>>(p);
   else sort_count_kernel<false><<<grid, TR_THREADS, 0, st>>>(p);
   sort_scan_kernel<<<TR_DIGITS, TR_THREADS, 0, st>>>(p);
   if (p.shift == 0) sort_move_kernel<true><<<grid, TR_THREADS, 0, st>>>(p);
   else sort_move_kernel<false><<<grid, TR_THREADS, 0, st>>>(p);
}

}  // namespace
}  // namespace attn
}  // namespace fmm

using namespace fmm::attn;

extern "C" {

int64_t fusedmm_b200_csr_transpose_workspace(int64_t m, int64_t n, int64_t nnz)
{
   if (m < 0 || n < 0 || nnz < 0) return FUSEDMM_B200_ERR_ARG;
   if (m >= 0x7fffffffLL || n >= 0x7fffffffLL || nnz >= 0x7fffffffLL) return FUSEDMM_B200_ERR_LIMIT;
   return 5 * round256(nnz * 4) + round256(sort_tiles(nnz) * TR_DIGITS * 4) + round256(TR_DIGITS * 4);
}

int fusedmm_b200_csr_transpose(int32_t ptr_bits, int32_t idx_bits, int64_t m, int64_t n, int64_t nnz, const void *rowptr,
                               const void *colidx, void *t_rowptr, int32_t *t_row, int32_t *t_edge, void *workspace,
                               int64_t workspace_bytes, void *stream)
{
   if ((ptr_bits != 32 && ptr_bits != 64) || (idx_bits != 32 && idx_bits != 64)) return FUSEDMM_B200_ERR_ARG;
   const int64_t need = fusedmm_b200_csr_transpose_workspace(m, n, nnz);
   if (need < 0) return static_cast<int>(need);
   if (!t_rowptr || !rowptr || (nnz > 0 && (!colidx || !t_row || !workspace))) return FUSEDMM_B200_ERR_ARG;
   if (nnz > 0 && (workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256)) return FUSEDMM_B200_ERR_ARG;
   if (!on_device({rowptr, t_rowptr, nnz > 0 ? colidx : nullptr, nnz > 0 ? t_row : nullptr, nnz > 0 ? t_edge : nullptr,
                   nnz > 0 ? workspace : nullptr}))
      return FUSEDMM_B200_ERR_ARG;
   cudaStream_t st = static_cast<cudaStream_t>(stream);
   if (nnz == 0) {
      if (cudaMemsetAsync(t_rowptr, 0, (n + 1) * (ptr_bits / 8), st) != cudaSuccess) return cuda_status();
      return finish_call(stream);
   }
   char *ws = static_cast<char *>(workspace);
   const long long arr = round256(nnz * 4), tiles = sort_tiles(nnz);
   unsigned *key[2] = {reinterpret_cast<unsigned *>(ws), reinterpret_cast<unsigned *>(ws + arr)};
   unsigned *edge[2] = {reinterpret_cast<unsigned *>(ws + 2 * arr), reinterpret_cast<unsigned *>(ws + 3 * arr)};
   int *row_of = reinterpret_cast<int *>(ws + 4 * arr);
   SortParams p = {};
   p.colidx = colidx; p.rowptr = rowptr; p.idx64 = idx_bits == 64; p.ptr64 = ptr_bits == 64;
   p.m = m; p.n = n; p.nnz = nnz; p.tiles = tiles;
   p.counts = reinterpret_cast<unsigned *>(ws + 5 * arr);
   p.totals = reinterpret_cast<unsigned *>(ws + 5 * arr + round256(tiles * TR_DIGITS * 4));
   int now = 0;
   for (int shift = 0; shift == 0 || (n >> shift) != 0; shift += 8) {  // keys are 0 .. n
      p.shift = shift;
      p.key_in = key[now]; p.edge_in = edge[now];
      p.key_out = key[now ^ 1]; p.edge_out = edge[now ^ 1];
      sort_pass(p, st);
      now ^= 1;
   }
   // edges outside every row keep row 0; they are behind t_rowptr[n] and no reader reaches them
   if (cudaMemsetAsync(row_of, 0, nnz * 4, st) != cudaSuccess) return cuda_status();
   if (m > 0) edge_rows_kernel<<<static_cast<unsigned>((m + 7) / 8), 256, 0, st>>>(rowptr, p.ptr64, m, nnz, row_of);
   transpose_ptr_kernel<<<static_cast<unsigned>((n + 256) / 256), 256, 0, st>>>(key[now], nnz, n, t_rowptr, p.ptr64);
   transpose_rows_kernel<<<static_cast<unsigned>((nnz + 255) / 256), 256, 0, st>>>(edge[now], row_of, nnz, t_row, t_edge);
   return finish_call(stream);
}

}  // extern "C"
