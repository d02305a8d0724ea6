// diff_attn_capi.cu -- the entry points of differential attention (include/fusedmm_b200.h): argument checks, the choice of
// the walk's shape, scratch layout.  The kernels are in diff_attn.cuh.
#include "attn_host.h"
#include "diff_attn.cuh"

#include <climits>
#include <mutex>
#include <set>
#include <utility>

namespace fmm {
namespace attn {

constexpr int LAM_BLOCKS = 256;

bool allow_shared(const void *kernel, int bytes)
{
   if (bytes <= 48 << 10) return true;
   static std::mutex mu;
   static std::set<std::pair<const void *, int>> *done = new std::set<std::pair<const void *, int>>;
   int dev = 0;
   if (cudaGetDevice(&dev) != cudaSuccess) return false;
   std::lock_guard<std::mutex> lock(mu);
   if (done->count({kernel, dev})) return true;
   if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
   done->insert({kernel, dev});
   return true;
}

// dlam[h] = sum over the rows: each block a run of rows, then one block the blocks' sums
__global__ void __launch_bounds__(256) lam_sum_kernel(const float *in, long long rows, int heads, float *out, long long each)
{
   __shared__ float part[8][33];
   const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
   const long long r0 = blockIdx.x * each, r1 = r0 + each < rows ? r0 + each : rows;
   for (int h0 = 0; h0 < heads; h0 += 32) {
      const int h = h0 + lane;
      float s = 0.0f;
      if (h < heads)
         for (long long r = r0 + w; r < r1; r += 8) s += in[r * heads + h];
      part[w][lane] = s;
      __syncthreads();
      if (w == 0 && h < heads) {
         float t = 0.0f;
         for (int i = 0; i < 8; i++) t += part[i][lane];
         out[static_cast<long long>(blockIdx.x) * heads + h] = t;
      }
      __syncthreads();
   }
}

// the bias of the edges in the order of the transposed pattern
__global__ void __launch_bounds__(256) permute_bias_kernel(const float *bias, const int *t_edge, long long nnz, const void *t_rowptr,
                                                           int ptr64, long long n, float *out)
{
   const long long t = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
   if (t >= nnz || t >= load_index(t_rowptr, ptr64, n)) return;  // behind the last column t_edge names no edge of a column
   const int e = __ldg(t_edge + t);
   out[t] = e >= 0 && e < nnz ? __ldg(bias + e) : -INFINITY;
}

namespace {

enum Walk { FORWARD, ROWS, COLUMNS };

struct Shape {
   WalkShape walk;
   int units = 0, unit_blocks = 0, slot_heads = 0, unit_kv = 1, unit_heads = 1, head_blocks = 1;
   long long piece = 0, row_limit = 0, pieces = 0, part_bytes = 0;
   long long scratch_bytes() const { return (pieces * 2 * units * part_bytes + 255) / 256 * 256 + (pieces * 8 + 255) / 256 * 256; }
};

constexpr long long SCRATCH_LIMIT = 128LL << 20;

Shape choose_shape(Walk w, int dtype, bool vector, long long rows, long long edges, int heads, int kv_heads, int d, int dv, int sms)
{
   Shape s;
   const int width = dtype == DT_F32 ? 4 : 8;
   const int nk = 2 * ((d + width - 1) / width), nvv = (dv + width - 1) / width, need = nk > nvv ? nk : nvv;
   const int group = heads / kv_heads;
   int lane_floats;
   if (dtype == DT_BF16 || (dtype == DT_F16 && w == FORWARD)) {
      s.walk.width = need <= 4 ? 16 : need <= 8 ? 32 : need <= 16 ? 64 : 128;
      s.walk.form = !vector ? PIECES : d == s.walk.width && dv == 2 * d ? EXACT : RAGGED;
      // a product has columns for four heads of each map: query heads of one kv head first, then neighbouring kv heads
      s.unit_kv = 1;
      if (w == COLUMNS) {
         s.unit_heads = group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
      } else {
         s.head_blocks = (group + 3) / 4;
         s.unit_heads = (group + s.head_blocks - 1) / s.head_blocks;
      }
      if (s.unit_heads == group)
         while (s.unit_kv * 2 * s.unit_heads <= 4 && kv_heads % (s.unit_kv * 2) == 0) s.unit_kv *= 2;
      s.units = kv_heads / s.unit_kv * s.head_blocks;
      s.slot_heads = 1;
      lane_floats = w == FORWARD ? s.walk.width / 2 + 4 : w == ROWS ? s.walk.width / 2 + 2 : s.walk.width;
      s.part_bytes = static_cast<long long>(lane_floats) * 32 * 4;
   } else {
      s.walk.g = need <= 8 ? 4 : need <= 16 ? 8 : need <= 32 ? 16 : 32;
      s.walk.nv = need <= 4 ? 1 : 2;
      const int vectors = s.walk.g * s.walk.nv;
      s.walk.form = !vector ? PIECES : nk == vectors && nvv == vectors ? EXACT : RAGGED;
      const int most = w == COLUMNS || s.walk.form != EXACT ? 1 : dtype == DT_F32 ? 4 : 2;
      s.walk.qb = most >= 4 && group % 4 == 0 ? 4 : most >= 2 && group % 2 == 0 ? 2 : 1;
      s.units = w == COLUMNS ? kv_heads : heads / s.walk.qb;
      s.slot_heads = 1;
      while (2 * s.slot_heads <= 32 / s.walk.g && s.units % (2 * s.slot_heads) == 0) s.slot_heads *= 2;
      lane_floats = w == COLUMNS ? 2 * s.walk.nv * width : s.walk.qb * (2 * s.walk.nv * width + 2);
      s.part_bytes = static_cast<long long>(lane_floats) * s.walk.g * 4;
   }
   s.unit_blocks = s.units / s.slot_heads;
   const long long items = edges + ROW_ITEMS * rows, mean = edges / rows;
   const bool few = rows * s.unit_blocks < 8LL * sms;
   s.walk.together = mean >= 256 || (few && mean >= 64);
   const long long lo = s.walk.together ? 256 : 128, hi = s.walk.together ? 8192 : 1024;
   const long long jobs = static_cast<long long>(sms) * (s.walk.together ? 12 : 128);
   s.piece = (items * s.unit_blocks + jobs - 1) / jobs;
   s.piece = s.piece < lo ? lo : s.piece > hi ? hi : s.piece;
   for (;; s.piece *= 2) {
      s.pieces = (items + s.piece - 1) / s.piece;
      if (s.pieces * 2 * s.units * s.part_bytes <= SCRATCH_LIMIT && s.pieces * s.unit_blocks < INT_MAX / 2) break;
   }
   s.row_limit = s.walk.together ? s.piece : s.piece > 512 ? s.piece : 512;
   return s;
}

void apply(AttnParams &p, const Shape &s, char *scratch)
{
   p.units = s.units; p.unit_blocks = s.unit_blocks; p.slot_heads = s.slot_heads;
   p.unit_kv = s.unit_kv; p.unit_heads = s.unit_heads; p.head_blocks = s.head_blocks;
   p.piece = s.piece; p.row_limit = s.row_limit; p.pieces = s.pieces;
   p.join_pieces = s.pieces * s.unit_blocks <= 8192 ? 1 : 8;  // few pieces: their long rows side by side
   p.partial = reinterpret_cast<float *>(scratch);
   p.long_row = reinterpret_cast<long long *>(scratch + (s.pieces * 2 * s.units * s.part_bytes + 255) / 256 * 256);
}

int launch(Walk w, int dtype, const Shape &s, AttnParams &p, cudaStream_t st)
{
   const long long b = dtype == DT_F32 ? 4 : 2;
   const bool columns = w == COLUMNS;
   p.a_stride = static_cast<unsigned>((columns ? p.ldq : p.ldk) * b);
   p.b_stride = static_cast<unsigned>((columns ? p.ldo : p.ldv) * b);
   p.a_head = (columns ? p.hsq : p.hsk) * b;
   p.b_head = (columns ? p.hso : p.hsv) * b;
   p.a_width = p.d;
   p.b_width = p.dv;
   p.subs = columns ? p.group / s.unit_heads : 1;
   p.kv_log2 = columns ? s.unit_heads >> 1 : 0;  // 1, 2, 4 -> 0, 1, 2
   int r = -1;
   if (w == FORWARD) r = dtype == DT_F32 ? walk_forward_f32(s.walk, p, st) : dtype == DT_BF16 ? walk_forward_bf16(s.walk, p, st) : walk_forward_f16(s.walk, p, st);
   if (w == ROWS) r = dtype == DT_F32 ? walk_rows_f32(s.walk, p, st) : dtype == DT_BF16 ? walk_rows_bf16(s.walk, p, st) : walk_rows_f16(s.walk, p, st);
   if (w == COLUMNS) r = dtype == DT_F32 ? walk_columns_f32(s.walk, p, st) : dtype == DT_BF16 ? walk_columns_bf16(s.walk, p, st) : walk_columns_f16(s.walk, p, st);
   if (r == 0) return 0;
   const int status = cuda_status();
   return status ? status : FUSEDMM_B200_ERR_CUDA;
}

int check_sizes(int32_t dtype, int64_t m, int64_t n, int64_t nnz, int32_t heads, int32_t kv_heads, int32_t d, int32_t dv)
{
   if (dtype != DT_F32 && dtype != DT_BF16 && dtype != DT_F16) return FUSEDMM_B200_ERR_ARG;
   if (m < 0 || n < 0 || nnz < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || d < 1 || dv < 1) return FUSEDMM_B200_ERR_ARG;
   if (d > FUSEDMM_B200_ATTN_MAX_WIDTH / 2 || dv > FUSEDMM_B200_ATTN_MAX_WIDTH || heads > FUSEDMM_B200_ATTN_MAX_HEADS)
      return FUSEDMM_B200_ERR_LIMIT;
   if (m > (1LL << 48) || nnz > (1LL << 48) || n >= INT_MAX) return FUSEDMM_B200_ERR_LIMIT;
   return 0;
}

// the kernels form the address of a row as base + id * stride with 32-bit factors
bool strides_fit(int32_t dtype, std::initializer_list<int64_t> strides)
{
   for (int64_t s : strides)
      if (s < 0 || s * (dtype == DT_F32 ? 4 : 2) >= INT_MAX) return false;
   return true;
}

// elements that one load of these rows may take at once; 16 bytes' worth: whole vectors
struct Step {
   int step;
   size_t elt;
   Step(int32_t dtype) : step(dtype == DT_F32 ? 4 : 8), elt(dtype == DT_F32 ? 4 : 2) {}
   void with(const void *p, long long a, long long b, long long c)
   {
      while (step > 1 && (reinterpret_cast<uintptr_t>(p) % (step * elt) || a % step || b % step || c % step)) step /= 2;
   }
   bool vector() const { return step * elt == 16; }
};

long long round256(long long b) { return (b + 255) / 256 * 256; }
long long max_ll(long long a, long long b) { return a > b ? a : b; }

long long walk_scratch(Walk w, int dtype, long long rows, long long edges, int heads, int kv_heads, int d, int dv, int sms)
{
   if (rows == 0) return 0;
   return max_ll(choose_shape(w, dtype, true, rows, edges, heads, kv_heads, d, dv, sms).scratch_bytes(),
                 choose_shape(w, dtype, false, rows, edges, heads, kv_heads, d, dv, sms).scratch_bytes());
}

// scratch of the backward pass in front of the walks': stats, dlam of every row, the sums of runs of rows,
// and the bias in the columns' order
long long backward_front(long long m, int heads, long long nnz)
{
   return round256(m * heads * 32) + round256(m * heads * 4) + round256(LAM_BLOCKS * heads * 4LL) + round256(nnz * 4);
}

}  // namespace
}  // namespace attn
}  // namespace fmm

using namespace fmm::attn;

extern "C" {

int64_t fusedmm_b200_diff_attention_workspace(int32_t backward, int32_t dtype, int64_t m, int64_t n, int64_t nnz,
                                              int32_t heads, int32_t kv_heads, int32_t d, int32_t dv)
{
   if (int s = check_sizes(dtype, m, n, nnz, heads, kv_heads, d, dv)) return s;
   int sms = 0;
   if (int s = sm_count(&sms)) return s;
   if (!backward) return walk_scratch(FORWARD, dtype, m, nnz, heads, kv_heads, d, dv, sms);
   return backward_front(m, heads, nnz) + max_ll(walk_scratch(ROWS, dtype, m, nnz, heads, kv_heads, d, dv, sms),
                                            walk_scratch(COLUMNS, dtype, n, nnz, heads, kv_heads, d, dv, sms));
}

int fusedmm_b200_diff_attention(int32_t dtype, int32_t ptr_bits, int32_t idx_bits, int64_t m, int64_t n, int64_t nnz,
                                const void *rowptr, const void *colidx, const float *bias, int32_t heads, int32_t kv_heads,
                                int32_t d, int32_t dv, const void *q, int64_t ldq, int64_t hsq, const void *k, int64_t ldk,
                                int64_t hsk, const void *v, int64_t ldv, int64_t hsv, const float *lam, int64_t ldlam,
                                double scale, void *out, float *lse, void *workspace, int64_t workspace_bytes, void *stream)
{
   if ((ptr_bits != 32 && ptr_bits != 64) || (idx_bits != 32 && idx_bits != 64)) return FUSEDMM_B200_ERR_ARG;
   if (int s = check_sizes(dtype, m, n, nnz, heads, kv_heads, d, dv)) return s;
   if (!strides_fit(dtype, {ldq, hsq, ldk, hsk, ldv, hsv, ldlam})) return FUSEDMM_B200_ERR_LIMIT;
   if (m == 0) return 0;
   const bool gathers = nnz > 0 && n > 0;
   if (!rowptr || !q || !lam || !out || (nnz > 0 && !colidx) || (gathers && (!k || !v))) return FUSEDMM_B200_ERR_ARG;
   int sms = 0;
   if (int s = sm_count(&sms)) return s;
   const long long need = walk_scratch(FORWARD, dtype, m, nnz, heads, kv_heads, d, dv, sms);
   if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256) return FUSEDMM_B200_ERR_ARG;
   if (!on_device({rowptr, q, lam, out, lse, workspace, nnz > 0 ? colidx : nullptr, nnz > 0 ? bias : nullptr,
                   gathers ? k : nullptr, gathers ? v : nullptr}))
      return FUSEDMM_B200_ERR_ARG;
   if (n == 0) k = v = workspace;  // nothing is gathered, but copies of nothing want an address too
   Step step(dtype);
   step.with(q, ldq, hsq, d);
   step.with(k, ldk, hsk, d);
   step.with(v, ldv, hsv, dv);
   step.with(out, 0, 0, dv);
   AttnParams p = {};
   p.rowptr = rowptr; p.colidx = colidx; p.ptr64 = ptr_bits == 64; p.idx64 = idx_bits == 64;
   p.m = m; p.n = n; p.nnz = nnz; p.bias = bias;
   p.q = q; p.k = k; p.v = v; p.lam = lam;
   p.ldq = ldq; p.hsq = hsq; p.ldk = ldk; p.hsk = hsk; p.ldv = ldv; p.hsv = hsv; p.ldlam = ldlam;
   p.out = out; p.lse = lse;
   p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads; p.d = d; p.dv = dv; p.step = step.step;
   p.scale = static_cast<float>(scale);
   const Shape s = choose_shape(FORWARD, dtype, step.vector(), m, nnz, heads, kv_heads, d, dv, sms);
   apply(p, s, static_cast<char *>(workspace));
   if (int r = launch(FORWARD, dtype, s, p, static_cast<cudaStream_t>(stream))) return r;
   return finish_call(stream);
}

int fusedmm_b200_diff_attention_backward(int32_t dtype, int32_t ptr_bits, int32_t idx_bits, int64_t m, int64_t n, int64_t nnz,
                                         const void *rowptr, const void *colidx, const float *bias, int32_t heads,
                                         int32_t kv_heads, int32_t d, int32_t dv, const void *q, int64_t ldq, int64_t hsq,
                                         const void *k, int64_t ldk, int64_t hsk, const void *v, int64_t ldv, int64_t hsv,
                                         const float *lam, int64_t ldlam, double scale, const float *lse, const void *dout,
                                         int64_t lddo, int64_t hsdo, const void *t_rowptr, const int32_t *t_row,
                                         const int32_t *t_edge, void *dq, void *dk, void *dv_out, float *dlam, void *workspace,
                                         int64_t workspace_bytes, void *stream)
{
   if ((ptr_bits != 32 && ptr_bits != 64) || (idx_bits != 32 && idx_bits != 64)) return FUSEDMM_B200_ERR_ARG;
   if (int s = check_sizes(dtype, m, n, nnz, heads, kv_heads, d, dv)) return s;
   if (m >= INT_MAX || nnz >= INT_MAX) return FUSEDMM_B200_ERR_LIMIT;
   if (!strides_fit(dtype, {ldq, hsq, ldk, hsk, ldv, hsv, lddo, hsdo, ldlam})) return FUSEDMM_B200_ERR_LIMIT;
   if (!dlam || (m > 0 && (!rowptr || !q || !lam || !lse || !dout || !dq)) || (n > 0 && (!k || !v || !dk || !dv_out || !t_rowptr)) ||
       (nnz > 0 && (!colidx || !t_row || (bias && !t_edge))))
      return FUSEDMM_B200_ERR_ARG;
   const int64_t need = fusedmm_b200_diff_attention_workspace(1, dtype, m, n, nnz, heads, kv_heads, d, dv);
   if (need < 0) return static_cast<int>(need);
   if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256) return FUSEDMM_B200_ERR_ARG;
   if (!on_device({m > 0 ? rowptr : nullptr, m > 0 ? q : nullptr, m > 0 ? lam : nullptr, m > 0 ? lse : nullptr, m > 0 ? dout : nullptr,
                   m > 0 ? dq : nullptr, n > 0 ? k : nullptr, n > 0 ? v : nullptr, n > 0 ? dk : nullptr, n > 0 ? dv_out : nullptr,
                   n > 0 ? t_rowptr : nullptr, nnz > 0 ? colidx : nullptr, nnz > 0 ? t_row : nullptr,
                   nnz > 0 ? bias : nullptr, nnz > 0 && bias ? t_edge : nullptr, m > 0 || ldlam == 0 ? dlam : nullptr, workspace}))
      return FUSEDMM_B200_ERR_ARG;
   int sms = 0;
   if (int s = sm_count(&sms)) return s;
   cudaStream_t st = static_cast<cudaStream_t>(stream);
   char *ws = static_cast<char *>(workspace);
   float *row_dlam = reinterpret_cast<float *>(ws + round256(m * heads * 32));
   float *lam_part = reinterpret_cast<float *>(ws + round256(m * heads * 32) + round256(m * heads * 4));
   char *scratch = ws + backward_front(m, heads, nnz);
   if (n == 0) k = v = workspace;  // nothing is gathered, but copies of nothing want an address too
   if (m == 0) q = dout = workspace;
   Step step(dtype);
   step.with(q, ldq, hsq, d);
   step.with(k, ldk, hsk, d);
   step.with(v, ldv, hsv, dv);
   step.with(dout, lddo, hsdo, dv);
   step.with(dq, 0, 0, d);
   step.with(dk, 0, 0, d);
   step.with(dv_out, 0, 0, dv);
   AttnParams p = {};
   p.bias = bias;
   p.q = q; p.k = k; p.v = v; p.lam = lam; p.dout = dout;
   p.ldq = ldq; p.hsq = hsq; p.ldk = ldk; p.hsk = hsk; p.ldv = ldv; p.hsv = hsv; p.ldo = lddo; p.hso = hsdo; p.ldlam = ldlam;
   p.lse = const_cast<float *>(lse);
   p.stats = reinterpret_cast<float4 *>(ws);
   p.dlam = ldlam ? dlam : row_dlam;
   p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads; p.d = d; p.dv = dv; p.step = step.step;
   p.scale = static_cast<float>(scale);
   p.nnz = nnz;
   p.ptr64 = ptr_bits == 64;
   if (m > 0) {
      p.rowptr = rowptr; p.colidx = colidx; p.idx64 = idx_bits == 64; p.m = m; p.n = n; p.out = dq;
      const Shape s = choose_shape(ROWS, dtype, step.vector(), m, p.nnz, heads, kv_heads, d, dv, sms);
      apply(p, s, scratch);
      if (int r = launch(ROWS, dtype, s, p, st)) return r;
   }
   if (!ldlam) {
      if (m > 0) {
         const long long each = (m + LAM_BLOCKS - 1) / LAM_BLOCKS;
         lam_sum_kernel<<<LAM_BLOCKS, 256, 0, st>>>(row_dlam, m, heads, lam_part, each);
         lam_sum_kernel<<<1, 256, 0, st>>>(lam_part, LAM_BLOCKS, heads, dlam, LAM_BLOCKS);
      } else if (cudaMemsetAsync(dlam, 0, heads * sizeof(float), st) != cudaSuccess) {
         return cuda_status();
      }
   }
   if (n > 0) {
      p.rowptr = t_rowptr; p.colidx = t_row; p.idx64 = 0; p.m = n; p.n = m; p.nnz = nnz; p.out = dk; p.out2 = dv_out;
      if (bias && nnz > 0) {
         float *moved = lam_part + round256(LAM_BLOCKS * heads * 4LL) / 4;
         permute_bias_kernel<<<static_cast<unsigned>((nnz + 255) / 256), 256, 0, st>>>(bias, t_edge, nnz, t_rowptr, p.ptr64, n, moved);
         p.bias = moved;
      }
      const Shape s = choose_shape(COLUMNS, dtype, step.vector(), n, p.nnz, heads, kv_heads, d, dv, sms);
      apply(p, s, scratch);
      if (int r = launch(COLUMNS, dtype, s, p, st)) return r;
   }
   return finish_call(stream);
}

}  // extern "C"
