// diff_attn_capi.cu -- the entry points of differential attention (include/fusedmm_b200.h): argument checks, the choice of
// the walk's shape, scratch layout.  The kernels are in diff_attn.cuh.
#include "attn_host.h"
#include "diff_attn.cuh"

#include <climits>

namespace fmm {
namespace attn {

constexpr int LAM_BLOCKS = 256;

bool set_shared(const void *kernel, int bytes, std::atomic<unsigned long long> &devices)
{
   int dev = 0;
   if (cudaGetDevice(&dev) != cudaSuccess) return false;
   const unsigned long long bit = dev < 64 ? 1ULL << dev : 0;
   if (devices.load(std::memory_order_relaxed) & bit) return true;
   if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
   devices.fetch_or(bit, std::memory_order_relaxed);
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

// Rows that are no vectors (their width, stride or address is no multiple of 16 bytes), packed: [rows][heads][maps][packed width],
// zeros behind the width.  Gathered as they are, such rows cost a load for each element at every edge (a cache of 220699 slots
// of 4 x (2 x 97 + 97) in bf16: 2149 us); packing costs two passes over them once.  With `ids` row e of the result is
// the row that edge e names, and `ids_out` names it: for few edges of a large cache.
template <typename T>
__global__ void __launch_bounds__(256) pack_rows_kernel(const T *src, long long ld, long long hs, int heads, int maps, int width, int step,
                                                        long long rows, const void *ids, int idx64, long long n, T *dst, int *ids_out)
{
   constexpr int W = Elt<T>::W;
   const int vectors = (width + W - 1) / W, per_row = heads * maps * vectors;
   const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x, row = i / per_row;
   if (row >= rows) return;
   const int rest = static_cast<int>(i - row * per_row), x = rest % vectors * W, map = rest / vectors % maps, head = rest / vectors / maps;
   long long from = row;
   bool live = true;
   if (ids) {
      from = load_index(ids, idx64, row);
      live = from >= 0 && from < n;
      if (ids_out && rest == 0) ids_out[row] = live ? static_cast<int>(row) : -1;
   }
   uint4 v = make_uint4(0u, 0u, 0u, 0u);
   if (live) v = ld_pieces(src + from * ld + head * hs + map * width + x, width - x, step < W ? step : W / 2);
   reinterpret_cast<uint4 *>(dst)[i] = v;
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

long long round256(long long b) { return (b + 255) / 256 * 256; }
long long max_ll(long long a, long long b) { return a > b ? a : b; }

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
   // 16-bit types go to the matrix units: a window of 128 over 4096 rows, 8 heads on 2, d 64: forward 78 us, 235 on the ordinary
   // units; 2^23 R-MAT edges, 4 heads of d 32: forward 1.13 and 1.49 ms, rows 1.58 and 2.02, columns 1.57 and 1.94.  Not half's
   // backward walks: their factors p dP and ds have no bound that half's 65504 covers, and they are operands there.
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
      lane_floats = w == FORWARD ? s.walk.width / 2 + 4 : w == ROWS ? s.walk.width / 2 + 8 : s.walk.width;
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
      lane_floats = w == COLUMNS ? 2 * s.walk.nv * width : s.walk.qb * (2 * s.walk.nv * width + (w == ROWS ? 4 : 2));
      s.part_bytes = static_cast<long long>(lane_floats) * s.walk.g * 4;
   }
   s.unit_blocks = s.units / s.slot_heads;
   // The warps of a block share every row where there are too few long rows to give each warp one: 48 tokens over 262144 slots, 4
   // kv heads of d 64: 103 us against 132, and 256 tokens 116 against 139; but 4096 rows of 512 edges, of which each warp can have
   // some, 1.71 ms shared and 1.61 not.  Blocks for an SM: the rings fill an SM with one or two, and each part costs the join (the
   // 48 tokens: 94 us with 6, 102 with 9, 104 with 12); the ordinary units' blocks are smaller (37 tokens over 84276 slots in
   // float: 275 us with 12, 362 with 6).
   // Otherwise a warp takes pieces of at most 128 items, or so many more that the table of parts stays short, and fewer where that
   // leaves warps without work (7600 edges over 400 rows, forward, rows and columns: 75 us with 128, 38 with 32).  Rows longer than a
   // piece (and a quarter, of short pieces) are cut: a hub row in one warp's hands is the walk's end (425984 R-MAT edges in float,
   // all walks: 457 us with rows of up to 512 items whole, 345 now).
   const long long items = edges + ROW_ITEMS * rows, mean = edges / rows;
   s.walk.together = rows * s.unit_blocks < 8LL * sms && mean >= 64;
   const long long share = items * s.unit_blocks / (16LL * sms);
   const long long lo = s.walk.together ? 256 : share < 32 ? 32 : share > 128 ? 128 : share, hi = s.walk.together ? 8192 : 1024;
   const long long jobs = static_cast<long long>(sms) * (!s.walk.together ? 128 : s.walk.width ? 6 : 12);
   s.piece = (items * s.unit_blocks + jobs - 1) / jobs;
   s.piece = s.piece < lo ? lo : s.piece > hi ? hi : s.piece;
   // One piece is the least there is, whatever its scratch (4097 units of 16 KB are above the limit); a warp counts the edges of a
   // piece and the row behind it in 32 bits.  (check_sizes keeps items * heads below 2^56, so that nothing here passes 63 bits.)
   for (;; s.piece *= 2) {
      s.pieces = (items + s.piece - 1) / s.piece;
      const bool fits = s.pieces * 2 * s.units * s.part_bytes <= SCRATCH_LIMIT;
      if ((fits || s.pieces == 1 || s.piece >= 1 << 29) && s.pieces * s.unit_blocks < INT_MAX / 2) break;
   }
   s.row_limit = s.walk.together || s.piece >= 256 ? s.piece : s.piece < 64 ? 80 : s.piece + s.piece / 4;
   return s;
}

void apply(AttnParams &p, const Shape &s, char *scratch)
{
   p.units = s.units; p.unit_blocks = s.unit_blocks; p.slot_heads = s.slot_heads;
   p.unit_kv = s.unit_kv; p.unit_heads = s.unit_heads; p.head_blocks = s.head_blocks;
   p.piece = s.piece; p.row_limit = s.row_limit; p.pieces = s.pieces;
   p.join_rows = s.walk.together && p.m <= s.pieces;
   p.join_pieces = s.pieces * s.unit_blocks <= 8192 ? 1 : 8;  // few pieces: their long rows side by side
   p.partial = reinterpret_cast<float *>(scratch);
   p.long_row = reinterpret_cast<long long *>(scratch + (s.pieces * 2 * s.units * s.part_bytes + 255) / 256 * 256);
}

// Two gathered arrays packed: bytes, and where they lie.
struct Packed {
   long long rows = 0;
   int heads = 0, a_width = 0, b_width = 0;
   size_t elt = 2;
   Packed(int dtype, long long rows_, int heads_, int d, int dv) : rows(rows_), heads(heads_), elt(dtype == DT_F32 ? 4 : 2)
   {
      const int w = dtype == DT_F32 ? 4 : 8;
      a_width = (d + w - 1) / w * w;
      b_width = (dv + w - 1) / w * w;
   }
   long long a_bytes() const { return round256(rows * heads * 2 * a_width * static_cast<long long>(elt)); }
   long long bytes() const { return a_bytes() + round256(rows * heads * b_width * static_cast<long long>(elt)); }
};

template <typename T>
void pack_array(const void *src, long long ld, long long hs, int heads, int maps, int width, int step, long long rows, const void *ids, int idx64,
                long long n, void *dst, int *ids_out, cudaStream_t st)
{
   const long long vectors = rows * heads * maps * ((width + Elt<T>::W - 1) / Elt<T>::W);
   if (vectors == 0) return;
   pack_rows_kernel<T><<<static_cast<unsigned>((vectors + 255) / 256), 256, 0, st>>>(static_cast<const T *>(src), ld, hs, heads, maps, width, step, rows,
                                                                                   ids, idx64, n, static_cast<T *>(dst), ids_out);
}

// The arrays a walk gathers: as they are, or (pack) packed into `room`; with by_edge the rows in the order of the edges, then
// p.colidx becomes `room`'s list behind them.
void set_gathered(AttnParams &p, int dtype, bool columns, bool pack, bool by_edge, char *room, cudaStream_t st)
{
   const long long elt = dtype == DT_F32 ? 4 : 2;
   const void *a = columns ? p.q : p.k, *b = columns ? p.dout : p.v;
   const long long lda = columns ? p.ldq : p.ldk, ha = columns ? p.hsq : p.hsk, ldb = columns ? p.ldo : p.ldv, hb = columns ? p.hso : p.hsv;
   const int heads = columns ? p.heads : p.kv_heads;
   p.a = static_cast<const char *>(a);
   p.b = static_cast<const char *>(b);
   p.a_stride = static_cast<unsigned>(lda * elt);
   p.b_stride = static_cast<unsigned>(ldb * elt);
   p.a_head = ha * elt;
   p.b_head = hb * elt;
   p.a_width = p.d;
   p.b_width = p.dv;
   if (!pack) return;
   const Packed k(dtype, by_edge ? p.nnz : p.n, heads, p.d, p.dv);
   char *pa = room, *pb = room + k.a_bytes();
   int *ids = by_edge ? reinterpret_cast<int *>(room + k.bytes()) : nullptr;
   const void *from = by_edge ? p.colidx : nullptr;
   auto both = [&](auto zero) {
      using T = decltype(zero);
      pack_array<T>(a, lda, ha, heads, 2, p.d, p.step, k.rows, from, p.idx64, p.n, pa, ids, st);
      pack_array<T>(b, ldb, hb, heads, 1, p.dv, p.step, k.rows, from, p.idx64, p.n, pb, nullptr, st);
   };
   if (dtype == DT_F32) both(0.0f);
   else if (dtype == DT_BF16) both(__nv_bfloat16());
   else both(__half());
   p.a = pa;
   p.b = pb;
   p.a_width = k.a_width;
   p.b_width = k.b_width;
   p.a_head = 2 * k.a_width * elt;
   p.b_head = k.b_width * elt;
   p.a_stride = static_cast<unsigned>(heads * p.a_head);
   p.b_stride = static_cast<unsigned>(heads * p.b_head);
   if (by_edge) {
      p.colidx = ids;
      p.idx64 = 0;
      p.n = p.nnz;
   }
}

int launch(Walk w, int dtype, const Shape &s, AttnParams &p, cudaStream_t st)
{
   p.subs = w == COLUMNS ? p.group / s.unit_heads : 1;
   p.kv_log2 = w == COLUMNS ? s.unit_heads >> 1 : 0;  // 1, 2, 4 -> 0, 1, 2
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
   if (nnz + ROW_ITEMS * (m > n ? m : n) > (1LL << 56) / heads) return FUSEDMM_B200_ERR_LIMIT;  // (far beyond any memory)
   return 0;
}

bool below(int64_t limit, std::initializer_list<int64_t> strides)
{
   for (int64_t s : strides)
      if (s < 0 || s >= limit) return false;
   return true;
}
// the walks form the address of a row that they gather as base + id * stride with 32-bit factors (packed rows are near)
bool gathered_strides_fit(int32_t dtype, std::initializer_list<int64_t> strides) { return below(INT_MAX / (dtype == DT_F32 ? 4 : 2), strides); }

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

long long walk_scratch(Walk w, int dtype, bool vector, long long rows, long long edges, int heads, int kv_heads, int d, int dv, int sms)
{
   return rows == 0 ? 0 : choose_shape(w, dtype, vector, rows, edges, heads, kv_heads, d, dv, sms).scratch_bytes();
}

// forward: packed rows of the cache or, where they are fewer, of the edges
bool pack_by_edge(long long n, long long nnz) { return nnz < n; }
long long forward_pack(int dtype, long long n, long long nnz, int kv_heads, int d, int dv)
{
   const bool by_edge = pack_by_edge(n, nnz);
   return Packed(dtype, by_edge ? nnz : n, kv_heads, d, dv).bytes() + (by_edge ? round256(nnz * 4) : 0);
}
// backward: first of k and v, then of q and do in the same place
long long backward_pack(int dtype, long long m, long long n, int heads, int kv_heads, int d, int dv)
{
   return max_ll(Packed(dtype, n, kv_heads, d, dv).bytes(), Packed(dtype, m, heads, d, dv).bytes());
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

int64_t fusedmm_b200_diff_attention_workspace(int32_t backward, int32_t aligned, int32_t dtype, int64_t m, int64_t n, int64_t nnz,
                                              int32_t heads, int32_t kv_heads, int32_t d, int32_t dv)
{
   if (int s = check_sizes(dtype, m, n, nnz, heads, kv_heads, d, dv)) return s;
   int sms = 0;
   if (int s = sm_count(&sms)) return s;
   const int width = dtype == DT_F32 ? 4 : 8;
   const bool vector = aligned && d % width == 0 && dv % width == 0;
   if (!backward) return walk_scratch(FORWARD, dtype, vector, m, nnz, heads, kv_heads, d, dv, sms) + (vector ? 0 : forward_pack(dtype, n, nnz, kv_heads, d, dv));
   return backward_front(m, heads, nnz) + max_ll(walk_scratch(ROWS, dtype, vector, m, nnz, heads, kv_heads, d, dv, sms),
                                                 walk_scratch(COLUMNS, dtype, vector, n, nnz, heads, kv_heads, d, dv, sms)) +
          (vector ? 0 : backward_pack(dtype, m, n, heads, kv_heads, d, dv));
}

int fusedmm_b200_diff_attention(int32_t dtype, int32_t ptr_bits, int32_t idx_bits, int64_t m, int64_t n, int64_t nnz,
                                const void *rowptr, const void *colidx, const float *bias, int32_t heads, int32_t kv_heads,
                                int32_t d, int32_t dv, const void *q, int64_t ldq, int64_t hsq, const void *k, int64_t ldk,
                                int64_t hsk, const void *v, int64_t ldv, int64_t hsv, const float *lam, int64_t ldlam,
                                double scale, void *out, float *lse, void *workspace, int64_t workspace_bytes, void *stream)
{
   if ((ptr_bits != 32 && ptr_bits != 64) || (idx_bits != 32 && idx_bits != 64)) return FUSEDMM_B200_ERR_ARG;
   if (int s = check_sizes(dtype, m, n, nnz, heads, kv_heads, d, dv)) return s;
   if (!below(INT64_MAX, {ldq, hsq, ldk, hsk, ldv, hsv, ldlam})) return FUSEDMM_B200_ERR_LIMIT;
   if (m == 0) return 0;
   const bool gathers = nnz > 0 && n > 0;
   if (!rowptr || !q || !lam || !out || (nnz > 0 && !colidx) || (gathers && (!k || !v))) return FUSEDMM_B200_ERR_ARG;
   if (n == 0) k = v = workspace;  // nothing is gathered, but copies of nothing want an address too
   Step step(dtype);
   step.with(q, ldq, hsq, d);
   step.with(k, ldk, hsk, d);
   step.with(v, ldv, hsv, dv);
   step.with(out, 0, 0, dv);
   if (step.vector() && !gathered_strides_fit(dtype, {ldk, ldv})) return FUSEDMM_B200_ERR_LIMIT;
   int sms = 0;
   if (int s = sm_count(&sms)) return s;
   const int64_t need = fusedmm_b200_diff_attention_workspace(0, step.vector(), dtype, m, n, nnz, heads, kv_heads, d, dv);
   if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256) return FUSEDMM_B200_ERR_ARG;
   if (!on_device({rowptr, q, lam, out, lse, workspace, nnz > 0 ? colidx : nullptr, nnz > 0 ? bias : nullptr,
                   gathers ? k : nullptr, gathers ? v : nullptr}))
      return FUSEDMM_B200_ERR_ARG;
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
   set_gathered(p, dtype, false, !step.vector() && gathers, pack_by_edge(n, nnz), static_cast<char *>(workspace) + s.scratch_bytes(),
                static_cast<cudaStream_t>(stream));
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
   if (!below(INT64_MAX, {ldq, hsq, ldk, hsk, ldv, hsv, lddo, hsdo, ldlam})) return FUSEDMM_B200_ERR_LIMIT;
   if (!dlam || (m > 0 && (!rowptr || !q || !lam || !lse || !dout || !dq)) || (n > 0 && (!k || !v || !dk || !dv_out || !t_rowptr)) ||
       (nnz > 0 && (!colidx || !t_row || (bias && !t_edge))))
      return FUSEDMM_B200_ERR_ARG;
   const void *k0 = n == 0 ? workspace : k, *v0 = n == 0 ? workspace : v;  // nothing is gathered, but copies of nothing want an address too
   const void *q0 = m == 0 ? workspace : q, *dout0 = m == 0 ? workspace : dout;
   Step step(dtype);
   step.with(q0, ldq, hsq, d);
   step.with(k0, ldk, hsk, d);
   step.with(v0, ldv, hsv, dv);
   step.with(dout0, lddo, hsdo, dv);
   step.with(dq, 0, 0, d);
   step.with(dk, 0, 0, d);
   step.with(dv_out, 0, 0, dv);
   if (step.vector() && !gathered_strides_fit(dtype, {ldk, ldv, ldq, lddo})) return FUSEDMM_B200_ERR_LIMIT;
   const int64_t need = fusedmm_b200_diff_attention_workspace(1, step.vector(), dtype, m, n, nnz, heads, kv_heads, d, dv);
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
   const long long walks = max_ll(walk_scratch(ROWS, dtype, step.vector(), m, nnz, heads, kv_heads, d, dv, sms),
                                  walk_scratch(COLUMNS, dtype, step.vector(), n, nnz, heads, kv_heads, d, dv, sms));
   AttnParams p = {};
   p.bias = bias;
   p.q = q0; p.k = k0; p.v = v0; p.lam = lam; p.dout = dout0;
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
      set_gathered(p, dtype, false, !step.vector(), false, scratch + walks, st);
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
      set_gathered(p, dtype, true, !step.vector(), false, scratch + walks, st);
      if (int r = launch(COLUMNS, dtype, s, p, st)) return r;
   }
   return finish_call(stream);
}

}  // extern "C"
