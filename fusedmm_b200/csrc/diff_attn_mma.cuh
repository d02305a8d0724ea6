// diff_attn_mma.cuh -- the walks of diff_attn.cuh for 16-bit types on the matrix units.
//
// The edges of a piece are one run, whatever rows they belong to.  A warp streams them through a ring of its own in shared
// memory: a block of the ring holds 16 gathered pairs (edge, head), `slots` neighbouring heads of 16/slots edges, and is
// filled by cp.async several blocks ahead of its use, so that the latency of the gathers, of the column ids before them and
// of the rows' ends is hidden however few edges a row has.  Blocks are swizzled so that ldmatrix meets no bank twice; the same
// block serves as operand with its elements as inner index (ldmatrix) and with the pairs as inner index (ldmatrix.trans).
//
// The products are mma m16n8k16 with 32-bit sums.  Forward:
//   scores  [16 pairs x 8 columns], column = (map, query head): A = gathered k, B = q.  A pair and a query head of
//           different kv heads give numbers nobody uses: at these sizes a wasted column costs less than the conversions and
//           lane sums of a product on the ordinary units.
//   output  [8 rows x dv] over the 16 pairs: A = weights, 0 where the heads differ or the edge is another row's,
//           B = gathered v.
// Weights are split into two 16-bit numbers, the second of which lies in the rows 8..15 of A that the first leaves free, so the
// split costs no product.  Their sum has 16 bits of the 32-bit value in bf16 (a result that is small against its values, where lam
// is near 1 and the maps nearly equal, is off by some 2^-17 of the values; more bits would take a second product).  Half's numbers
// are 2^-24 apart below 2^-14, so there weights are carried 2^8 times larger (the row's sum with them) and the second parts another
// 2^11 times (taken out where the two rows are added up): 22 bits of weights down to 2^-22 of the row's largest, and 2^-44 of that
// largest is what smaller ones lose at most.  Weights change from "pair by column" to "row by pair" with movmatrix.
// Why not tcgen05: a tile there has 64 or 128 rows that share one operand; here a gathered row meets at most 8 rows of q, and
// consecutive rows of a graph gather different rows.  (Those of a window share nearly all: 64 rows of a window of 128 have 191 between
// them and gather 8192.  A form for runs of ids is not built.)
#pragma once
#include <climits>

#include "diff_attn.cuh"

namespace fmm {
namespace attn {

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1)
{
   if constexpr (std::is_same<T, __half>::value)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
   else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// ... the first product of a sum
template <typename T>
__device__ __forceinline__ void mma16816_first(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1)
{
   const float z = 0.0f;
   if constexpr (std::is_same<T, __half>::value)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                   : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(z));
   else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                   : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(z));
}
template <typename T>
__device__ __forceinline__ void mma16816_at(bool start, float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1)
{
   if (start) mma16816_first<T>(c, a[0], a[1], a[2], a[3], b0, b1);
   else mma16816<T>(c, a[0], a[1], a[2], a[3], b0, b1);
}
__device__ __forceinline__ unsigned transpose8x8(unsigned v)
{
   unsigned r;
   asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
   return r;
}
__device__ __forceinline__ void ldmatrix4(unsigned (&r)[4], unsigned at)
{
   asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(unsigned (&r)[4], unsigned at)
{
   asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// `there` (0 or 16) bytes from global memory, zeros in the place of the others (0: nothing is read)
__device__ __forceinline__ void copy_async(unsigned to, const void *from, int there)
{
   asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there) : "memory");
}
// powers of two that half's weights, and the second parts of its split numbers, are carried larger by
template <typename T>
constexpr float WEIGHT_LOG2 = std::is_same<T, __half>::value ? 8.0f : 0.0f;
template <typename T>
constexpr float LOWER_SCALE = std::is_same<T, __half>::value ? 2048.0f : 1.0f;
// v as hi + lo / LOWER_SCALE, two numbers of T, for two neighbours
template <typename T>
__device__ __forceinline__ void split2(float a, float b, unsigned &hi, unsigned &lo)
{
   hi = Elt<T>::pack2(a, b);
   float x, y;
   Elt<T>::unpack2(hi, x, y);
   lo = Elt<T>::pack2((a - x) * LOWER_SCALE<T>, (b - y) * LOWER_SCALE<T>);
}

// two elements of a row, those of them that are there
template <typename T, int FORM>
__device__ __forceinline__ unsigned load_two(const T *p, int left, int step)
{
   if (FORM == EXACT || (left >= 2 && (FORM == RAGGED || step >= 2))) return __ldg(reinterpret_cast<const unsigned *>(p));
   const unsigned short *u = reinterpret_cast<const unsigned short *>(p);
   return (left > 0 ? __ldg(u) : 0u) | (left > 1 ? static_cast<unsigned>(__ldg(u + 1)) << 16 : 0u);
}
// a row as the B operand of this lane's column: elements 2c, 2c + 1 of every 8
template <typename T, int WIDTH, int FORM>
__device__ __forceinline__ void load_operand(const T *row, int c, int width, int step, unsigned (&r)[WIDTH / 8])
{
#pragma unroll
   for (int i = 0; i < WIDTH / 8; i++) r[i] = load_two<T, FORM>(row + 8 * i + 2 * c, width - 8 * i - 2 * c, step);
}
template <typename T, int FORM>
__device__ __forceinline__ void store_two(T *p, float a, float b, int left)
{
   if (FORM != PIECES) {
      if (left > 0) *reinterpret_cast<unsigned *>(p) = Elt<T>::pack2(a, b);
   } else {
      if (left > 0) p[0] = Elt<T>::down(a);
      if (left > 1) p[1] = Elt<T>::down(b);
   }
}

// Lane geometry that the three walks share.  Lane = 4 r + c.  As an operand's row (or column) r: column n = r of the scores,
// map r / 4, slot r % 4; as a result: the pairs r and r + 8, the columns 2c and 2c + 1.
struct Lanes {
   int r, c, slots, slots_log2, pair_slot;  // pair_slot: of the pairs r and r + 8
   __device__ __forceinline__ void set(const Place &at, int slots_)
   {
      r = at.lane >> 2;
      c = at.lane & 3;
      slots = slots_;
      slots_log2 = slots_ >> 1;  // 1, 2, 4 -> 0, 1, 2
      pair_slot = r & (slots - 1);
   }
};

// The ring of a warp: STAGES blocks of 16 pairs, each of two gathered rows of 2 DK elements (k of both maps and v, or q and
// do), 16 biases and, where the walk wants them, 16 records of 32 bytes.  What a block costs beside its products is mostly
// the addresses of its copies: everything that a lane's copies share is worked out once (Lane pointers, places).
template <typename T, int DK, int FORM, int STAGES_, bool RECORDS, bool SINGLE_>
struct Ring {
   static constexpr bool SINGLE = SINGLE_;  // one group of heads: every edge lies in one block
   static constexpr int STAGES = STAGES_, ROW = 4 * DK, CHUNKS = DK / 4, REGION = 16 * ROW;
   static constexpr int BIAS = 2 * REGION, RECORD = BIAS + 64, USED = RECORD + (RECORDS ? 16 * 32 : 0);
   static constexpr int STAGE = (USED + ROW - 1) / ROW * ROW;  // rows are aligned to their size, so that chunks can be named by exclusive or
   // one round of copies: 32 lanes take PER pairs of CHUNKS chunks of 8 elements
   static constexpr int PER = 32 / CHUNKS, ROUNDS = CHUNKS / 2;
   const char *a, *b;       // the two arrays at the lane's chunk of the unit's head 0 (of the lane's slot, if that is the same in all rounds)
   const char *a2, *b2;     // with two pairs a round: the slot of the odd rounds
   const char *records;     // [row][head][32 bytes], of the unit's first head
   EdgeStream edges;
   int batch_id;            // the present 32 edges
   float batch_bias;
   unsigned ring, place;    // shared address of block 0; the lane's chunk in a block
   unsigned fill, slot;     // block to fill next, block in use
   long long first;         // the run of edges
   int length;
   int issued, current;     // blocks
   unsigned on;             // bit i: the lane's pair of round i is gathered (all, but where the kv heads are taken one by one)

   // Byte offset of a chunk of 8 elements of a pair.  The chunk is exchanged by bits of the pair, so that the 8 pairs that
   // ldmatrix reads at one chunk lie in 8 different groups of banks; offset(pair, chunk ^ x) = offset(pair, chunk) ^ (x << 4).
   // (Rows 16 bytes longer do that too and save the exclusive ors, but the copies then end inside 32-byte sectors: columns 3 %
   // slower for a window of 128 over 4096 rows at d 64.)
   static __device__ __forceinline__ unsigned offset(int pair, int chunk)
   {
      const int key = CHUNKS >= 8 ? pair & 7 : (pair >> 1) & 3;
      return pair * ROW + ((chunk ^ key) << 4);
   }
   __device__ __forceinline__ void setup(const AttnParams &p, const Lanes &l, int lane, int head)
   {
      const int x = lane % CHUNKS, pair = lane / CHUNKS, s = PER >= 2 ? pair & (l.slots - 1) : 0;
      const int map = x / (CHUNKS / 2), xa = (x % (CHUNKS / 2)) * 8, xb = x * 8;
      a = p.a + (head + s) * p.a_head + static_cast<long long>(map * p.a_width + xa) * sizeof(T);
      b = p.b + (head + s) * p.b_head + static_cast<long long>(xb) * sizeof(T);
      place = offset(pair, x);
      if constexpr (PER == 2) {
         a2 = a + (l.slots == 4 ? 2 * p.a_head : 0);
         b2 = b + (l.slots == 4 ? 2 * p.b_head : 0);
      }
   }

   // gathers the next block, if there is one; always closes a group of copies
   __device__ __forceinline__ void issue(const AttnParams &p, const Lanes &l, int lane)
   {
      const int per_log2 = 4 - l.slots_log2;
      const int edge_block = SINGLE ? issued : issued / p.subs, sub = SINGLE ? 0 : issued - edge_block * p.subs;
      const int e = edge_block << per_log2;  // from the run's start
      if (e < length) {
         const int off = e & 31;
         if (off == 0 && sub == 0) {  // a new batch of ids; the one after it sets out
            batch_id = edges.take(p, first + e, first + length, lane);
            batch_bias = batch_id >= 0 ? edges.bias : -INFINITY;
            edges.fetch(p, first + e + 32, lane);
         }
         const float bias = __shfl_sync(FULL, batch_bias, off + (lane & ((1 << per_log2) - 1)));
         if ((lane >> per_log2) == 0) asm volatile("st.shared.f32 [%0], %1;" ::"r"(fill + BIAS + 4 * lane), "f"(bias) : "memory");
         const int pair0 = lane / CHUNKS;
         int left_a = 1, left_b = 1;  // EXACT: every lane's chunk is there
         if constexpr (FORM != EXACT) {
            const int x = lane % CHUNKS;
            left_a = p.a_width - (x % (CHUNKS / 2)) * 8;
            left_b = p.b_width - x * 8;
         }
         if (PER >= 4 && on == 0) left_a = left_b = 0;  // a lane whose pairs are all of one slot
         const char *la = a, *lb = b, *la2 = a2, *lb2 = b2;
         if (!SINGLE && sub > 0) {
            la += (sub << p.kv_log2) * p.a_head;
            lb += (sub << p.kv_log2) * p.b_head;
            la2 += (sub << p.kv_log2) * p.a_head;
            lb2 += (sub << p.kv_log2) * p.b_head;
         }
#pragma unroll
         for (int i = 0; i < ROUNDS; i++) {
            const int pair = i * PER + pair0;
            const int id = __shfl_sync(FULL, batch_id, off + (pair >> l.slots_log2));
            const bool live = id >= 0;
            const unsigned row = live ? id : 0;
            const bool here = PER >= 4 ? live : live && (on >> i & 1);
            const char *ra = (PER == 2 && (i & 1) ? la2 : la) + static_cast<unsigned long long>(row) * p.a_stride;
            const char *rb = (PER == 2 && (i & 1) ? lb2 : lb) + static_cast<unsigned long long>(row) * p.b_stride;
            if constexpr (PER == 1) {  // the slot is the round's
               ra += (i & (l.slots - 1)) * p.a_head;
               rb += (i & (l.slots - 1)) * p.b_head;
            }
            // the pair's bits that change from round to round, as in offset()
            const unsigned at = fill + (place ^ (CHUNKS >= 8 ? ((i * PER) & 7) << 4 : 0)) + i * PER * ROW;
            copy_async(at, ra, here && left_a > 0 ? 16 : 0);
            copy_async(at + REGION, rb, here && left_b > 0 ? 16 : 0);
         }
         if constexpr (RECORDS) {
            const int pair = lane >> 1, s = (pair & (l.slots - 1)) + (sub << p.kv_log2);
            const int id = __shfl_sync(FULL, batch_id, off + (pair >> l.slots_log2));
            const unsigned row = id >= 0 ? id : 0;
            copy_async(fill + RECORD + lane * 16, records + static_cast<unsigned long long>(row) * (p.heads * 32u) + (s * 32 + (lane & 1) * 16),
                           id >= 0 ? 16 : 0);
         }
      }
      issued++;
      fill = fill == ring + (STAGES - 1) * STAGE ? ring : fill + STAGE;
      asm volatile("cp.async.commit_group;" ::: "memory");
   }
   __device__ __forceinline__ void begin(const AttnParams &p, const Lanes &l, int lane, long long from, long long to, int only_kv)
   {
      drain();
      first = from;
      length = to > from ? static_cast<int>(to - from) : 0;
      on = ~0u;
      if (only_kv >= 0)
         for (int i = 0; i < 32; i++)  // (with PER >= 4 all rounds are alike)
            if ((((i * PER + lane / CHUNKS) & (l.slots - 1)) >> p.kv_log2) != only_kv) on &= ~(1u << i);
      issued = 0;
      current = -1;
      fill = ring;
      slot = ring + (STAGES - 1) * STAGE;
#pragma unroll 1
      for (int i = 0; i < STAGES - 1; i++) issue(p, l, lane);
   }
   // the next block; the one before it may be overwritten
   __device__ __forceinline__ void advance(const AttnParams &p, const Lanes &l, int lane)
   {
      __syncwarp();  // every lane is done with the block before
      issue(p, l, lane);
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      __syncwarp();  // every lane's copies are there
      current++;
      slot = slot == ring + (STAGES - 1) * STAGE ? ring : slot + STAGE;
   }
   __device__ __forceinline__ void drain()
   {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();
   }
};

__device__ __forceinline__ float shared_float(unsigned at)
{
   float f;
   asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(at) : "memory");
   return f;
}

// What a lane knows of the score columns.  A product has 8 columns, (map, slot); with four kv heads to a unit a pair has one
// column of each map that counts, so a lane has at most one (ONE); otherwise it has the columns 2c and 2c + 1.
template <bool ONE>
struct Columns {
   static constexpr int N = ONE ? 1 : 2;
   // value of column n = r from the lanes that hold it
   static __device__ __forceinline__ float of_row(const float (&x)[N], int r)
   {
      if constexpr (ONE) return __shfl_sync(FULL, x[0], 4 * (r & 3) + 2 * (r >> 2) + ((r >> 1) & 1));
      const float a = __shfl_sync(FULL, x[0], r >> 1), b = __shfl_sync(FULL, x[N - 1], r >> 1);
      return r & 1 ? b : a;
   }
   // over all pairs
   static __device__ __forceinline__ float sum(float v)
   {
      if constexpr (!ONE) {
         v += __shfl_xor_sync(FULL, v, 4);
         v += __shfl_xor_sync(FULL, v, 8);
      }
      return v + __shfl_xor_sync(FULL, v, 16);
   }
   static __device__ __forceinline__ float max(float v)
   {
      if constexpr (!ONE) {
         v = fmaxf(v, __shfl_xor_sync(FULL, v, 4));
         v = fmaxf(v, __shfl_xor_sync(FULL, v, 8));
      }
      return fmaxf(v, __shfl_xor_sync(FULL, v, 16));
   }
   // the scores of pair r + 8h that count, of the two maps' products
   static __device__ __forceinline__ float pick(const float (&s0)[4], const float (&s1)[4], int h, int x, const Lanes &l)
   {
      if constexpr (ONE) return l.pair_slot & 1 ? (l.c < 2 ? s0[2 * h + 1] : s1[2 * h + 1]) : (l.c < 2 ? s0[2 * h] : s1[2 * h]);
      return l.c < 2 ? s0[2 * h + x] : s1[2 * h + x];
   }
   static __device__ __forceinline__ float pick(const float (&s)[4], int h, int x, const Lanes &l)
   {
      if constexpr (ONE) return l.pair_slot & 1 ? s[2 * h + 1] : s[2 * h];
      return s[2 * h + x];
   }
   // the weights of pair r + 8h at the columns 2c, 2c + 1, split
   template <typename T>
   static __device__ __forceinline__ void split(const float (&w)[N], const Lanes &l, unsigned &hi, unsigned &lo)
   {
      if constexpr (ONE) split2<T>(l.pair_slot & 1 ? 0.0f : w[0], l.pair_slot & 1 ? w[0] : 0.0f, hi, lo);
      else split2<T>(w[0], w[N - 1], hi, lo);
   }
};

// The query heads of the row walks' columns: column n = 4 map + s, s = (kv head of the unit) * unit_heads + (query head of it).
template <bool ONE>
struct QueryHeads {
   static constexpr int N = ONE ? 1 : 2;
   int head;        // of column n = r, one that exists if that column is none
   bool live;       // column n = r is one
   int kv;          // which of the unit's kv heads column n = r is of
   bool valid[N];   // the pairs r and r + 8 belong to this lane's columns
   int col_head[N], col_kv[N];
   __device__ __forceinline__ void set(const AttnParams &p, const Place &at, const Lanes &l, int kv0)
   {
      const int first = (at.unit % p.head_blocks) * p.unit_heads, rest = p.group - first;
      const int heads = rest < p.unit_heads ? rest : p.unit_heads;
      const int s = l.r & 3, g = s % p.unit_heads;
      kv = s / p.unit_heads;
      live = kv < l.slots && g < heads;
      head = live ? (kv0 + kv) * p.group + first + g : kv0 * p.group + first;
#pragma unroll
      for (int x = 0; x < N; x++) {
         const int sx = (2 * l.c + (ONE ? l.pair_slot & 1 : x)) & 3, gx = sx % p.unit_heads;
         col_kv[x] = sx / p.unit_heads;
         valid[x] = col_kv[x] == l.pair_slot && gx < heads;
         col_head[x] = valid[x] ? (kv0 + col_kv[x]) * p.group + first + gx : head;
      }
   }
};

// the maximum may grow by this much (as a power of e) before sums are scaled anew: weights then stay below e^5 and a
// row's scaling is done once as a rule.  32-bit sums and 16-bit weights hold that (half: 2^8 e^5 = 37994 of 65504).
constexpr float SLACK = 5.0f;

// warps of a block and blocks of a multiprocessor: registers and rings decide (a warp's ring is STAGES x 128 DK bytes)
enum { WALK_FORWARD, WALK_ROWS, WALK_COLUMNS };
template <int DK, int WALK>
struct Budget {
   static constexpr int STAGES = DK == 16 ? 4 : DK == 32 ? 3 : 2;
   static constexpr int SOLO = DK == 128 ? 2 : 4, JOINT = DK >= 64 ? 4 : 8;
   // The backward walks run faster with fewer warps and their registers: 2^23 R-MAT edges at d 32 columns 1.75 ms with four
   // blocks, 1.57 with three, rows 1.75 and 1.58; a window of 128 over 4096 rows at d 64 columns 349 us with three blocks, 273 with
   // two, rows 102 and 96.  (Forward with one block less and a stage more: 1.21 ms for 1.13, 81 us for 76.)
   static constexpr int BLOCKS = DK == 16 ? 4 : DK == 32 ? (WALK == WALK_FORWARD ? 4 : 3) : DK == 64 ? (WALK == WALK_FORWARD ? 3 : 2) : 3;
   static constexpr bool AHEAD = DK <= 32;  // a row's own operands are fetched during the row before (wider: no registers left)
};

// ---------------------------------------------------------------------------------------------------------------------
// forward.  2^23 R-MAT edges, 4 heads of d 32, bf16: 1.13 ms, 7.6 TB/s of gathered rows (hubs from L2); 2^21 edges: 339 instructions
// a block of 16 pairs, issue slots 0.54 busy; 48 tokens over 262144 slots of 4 kv heads of d 64: 94 us, 5.7 TB/s from HBM.
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DK, int FORM, bool ONE>
struct ForwardMma {
   using Cols = Columns<ONE>;
   static constexpr int N = Cols::N;
   static constexpr int DV = 2 * DK, TILES = DV / 8, LANE_FLOATS = 2 * TILES + 4;
   using Gathered = Ring<T, DK, FORM, Budget<DK, WALK_FORWARD>::STAGES, false, true>;
   using Width = Budget<DK, WALK_FORWARD>;
   struct State {
      float acc[TILES][2];   // rows n = r: sums of weights times v, columns 8t + 2c, + 1
      float top[N], sum[N];  // of this lane's columns
   };
   State s;
   Lanes l;
   QueryHeads<ONE> heads;
   int kv0;
   unsigned next[DK / 8];
   bool lost;  // run() met a number that is none

   __device__ __forceinline__ void setup(const AttnParams &p, const Place &at, Gathered &ring)
   {
      l.set(at, p.unit_kv);
      kv0 = (at.unit / p.head_blocks) * p.unit_kv;
      heads.set(p, at, l, kv0);
      ring.setup(p, l, at.lane, kv0);
   }
   static __device__ __forceinline__ void clear(State &s)
   {
#pragma unroll
      for (int t = 0; t < TILES; t++) s.acc[t][0] = s.acc[t][1] = 0.0f;
#pragma unroll
      for (int x = 0; x < N; x++) {
         s.top[x] = -INFINITY;
         s.sum[x] = 0.0f;
      }
   }
   // the row's own operand, ahead of run()
   __device__ __forceinline__ void fetch(const AttnParams &p, long long row)
   {
      load_operand<T, DK, FORM>(static_cast<const T *>(p.q) + row * p.ldq + heads.head * p.hsq + (l.r >> 2) * p.d, l.c, p.d, p.step, next);
   }

   // edges [e0, e1) of the ring's run; `follow`: the row to fetch for, or -1
   __device__ __forceinline__ void run(const AttnParams &p, const Place &at, Gathered &ring, int e0, int e1, long long follow)
   {
      float acc[TILES][4];
#pragma unroll
      for (int t = 0; t < TILES; t++) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.0f;
#pragma unroll
      for (int x = 0; x < N; x++) {
         s.top[x] = -INFINITY;
         s.sum[x] = 0.0f;
      }
      unsigned q[DK / 8];
#pragma unroll
      for (int i = 0; i < DK / 8; i++) q[i] = next[i];
      if (Width::AHEAD && follow >= 0) fetch(p, follow);
      const int per_log2 = 4 - l.slots_log2;
      // the lane's row and chunk of ldmatrix: pairs 0..7 and 8..15 of one chunk, then of the next; chunks by exclusive or
      const unsigned mine = Gathered::offset(at.lane & 15, at.lane >> 4);
      for (int e = e0; e < e1;) {
         const int block = e >> per_log2;
         if (block != ring.current) ring.advance(p, l, at.lane);
         const int lo = e - (block << per_log2), left = e1 - (block << per_log2), hi = left < (1 << per_log2) ? left : 1 << per_log2;
         const unsigned slot = ring.slot;
         float s0[4], s1[4];
#pragma unroll
         for (int i = 0; i < DK / 16; i++) {
            unsigned k[4];
            ldmatrix4(k, (slot + mine) ^ ((2 * i) << 4));
            mma16816_at<T>(i == 0, s0, k, q[2 * i], q[2 * i + 1]);
            ldmatrix4(k, (slot + mine) ^ ((DK / 8 + 2 * i) << 4));
            mma16816_at<T>(i == 0, s1, k, q[2 * i], q[2 * i + 1]);
         }
         float score[2][N], high[N];
         bool grown = false;
#pragma unroll
         for (int h = 0; h < 2; h++) {
            const int edge = (l.r + 8 * h) >> l.slots_log2;
            const float bias = shared_float(slot + Gathered::BIAS + 4 * edge);
            const bool live = edge >= lo && edge < hi && bias != -INFINITY;
#pragma unroll
            for (int x = 0; x < N; x++) score[h][x] = heads.valid[x] && live ? fmaf(Cols::pick(s0, s1, h, x, l), p.scale, bias) : -INFINITY;
         }
#pragma unroll
         for (int x = 0; x < N; x++) {
            high[x] = fmaxf(score[0][x], score[1][x]);
            grown |= high[x] - s.top[x] > SLACK;  // (the difference: next to large scores a sum with 5 may be rounded to 8 more)
         }
         if (__any_sync(FULL, grown)) {
            float f[N];
#pragma unroll
            for (int x = 0; x < N; x++) {
               const float t = fmaxf(s.top[x], Cols::max(high[x]));
               f[x] = t == -INFINITY ? 1.0f : exp2_fast((s.top[x] - t) * LOG2E);
               s.top[x] = t;
               s.sum[x] *= f[x];
            }
            if (e != e0) {
               const float fr = Cols::of_row(f, l.r);
#pragma unroll
               for (int t = 0; t < TILES; t++)
#pragma unroll
                  for (int i = 0; i < 4; i++) acc[t][i] *= fr;
            }
         }
         unsigned a[4];
#pragma unroll
         for (int h = 0; h < 2; h++) {
            float w[N];
#pragma unroll
            for (int x = 0; x < N; x++) {
               // a row that has met no edge yet has the maximum -inf: its differences are taken from 0.
               // The difference is taken before the factor: scores near the type's largest numbers keep their order.
               w[x] = exp2_fast(fmaf(score[h][x] - (s.top[x] == -INFINITY ? 0.0f : s.top[x]), LOG2E, WEIGHT_LOG2<T>));
               s.sum[x] += w[x];
            }
            unsigned up, low;
            Cols::template split<T>(w, l, up, low);
            a[2 * h] = transpose8x8(up);
            a[2 * h + 1] = transpose8x8(low);
         }
#pragma unroll
         for (int t = 0; t < TILES; t += 2) {
            unsigned v[4];
            ldmatrix4_trans(v, (slot + mine + Gathered::REGION) ^ ((t) << 4));
            mma16816<T>(acc[t], a[0], a[1], a[2], a[3], v[0], v[1]);
            mma16816<T>(acc[t + 1], a[0], a[1], a[2], a[3], v[2], v[3]);
         }
         e = (block << per_log2) + hi;
      }
      float all = 0.0f;
#pragma unroll
      for (int t = 0; t < TILES; t++) {
         s.acc[t][0] = fmaf(acc[t][2], 1.0f / LOWER_SCALE<T>, acc[t][0]);
         s.acc[t][1] = fmaf(acc[t][3], 1.0f / LOWER_SCALE<T>, acc[t][1]);
         all += s.acc[t][0] * 0.0f + s.acc[t][1] * 0.0f;  // 0, or NaN once anything is infinite or NaN
      }
      lost = all != all;
#pragma unroll
      for (int x = 0; x < N; x++) s.sum[x] = Cols::sum(s.sum[x]);
   }

   __device__ __forceinline__ void join_from(const float *unit, const Place &at)
   {
      const float2 *from = reinterpret_cast<const float2 *>(unit) + at.lane;
      const float2 top = from[32 * TILES], sum = from[32 * (TILES + 1)];
      float2 o[TILES];
#pragma unroll
      for (int t = 0; t < TILES; t++) o[t] = from[32 * t];
      float f[N], g[N];
#pragma unroll
      for (int x = 0; x < N; x++) {
         const float ot = x ? top.y : top.x, os = x ? sum.y : sum.x;
         const float t = fmaxf(s.top[x], ot), ref = t == -INFINITY ? 0.0f : t;
         f[x] = exp2_fast((s.top[x] - ref) * LOG2E);
         g[x] = exp2_fast((ot - ref) * LOG2E);
         s.sum[x] = s.sum[x] * f[x] + os * g[x];
         s.top[x] = t;
      }
      const float fr = Cols::of_row(f, l.r), gr = Cols::of_row(g, l.r);
#pragma unroll
      for (int t = 0; t < TILES; t++) {
         s.acc[t][0] = s.acc[t][0] * fr + o[t].x * gr;
         s.acc[t][1] = s.acc[t][1] * fr + o[t].y * gr;
      }
   }
   __device__ __forceinline__ void put(float *unit, const Place &at, int only) const
   {
      float2 *to = reinterpret_cast<float2 *>(unit) + at.lane;
      if (only < 0 || heads.kv == only) {
#pragma unroll
         for (int t = 0; t < TILES; t++) to[32 * t] = make_float2(s.acc[t][0], s.acc[t][1]);
      }
      float *top = reinterpret_cast<float *>(to + 32 * TILES), *sum = reinterpret_cast<float *>(to + 32 * (TILES + 1));
#pragma unroll
      for (int x = 0; x < N; x++)
         if (only < 0 || heads.col_kv[x] == only) {
            top[x] = s.top[x];
            sum[x] = s.sum[x];
         }
   }

   __device__ __forceinline__ void finish(const AttnParams &p, const Place &at, long long row, int only)
   {
      const float sum = Cols::of_row(s.sum, l.r), top = Cols::of_row(s.top, l.r);
      const bool mine = heads.live && (only < 0 || heads.kv == only);
      const float lam = __ldg(p.lam + row * p.ldlam + heads.head), f = sum == 0.0f ? 0.0f : __frcp_rn(sum);
      const long long rh = row * p.heads + heads.head;
      // rows 0..3 hold map 0, rows 4..7 map 1: these take the even, those the odd tiles of the result
      const int odd = l.r >> 2;
      T *out = static_cast<T *>(p.out) + rh * p.dv + 8 * odd + 2 * l.c;
#pragma unroll
      for (int t = 0; t < TILES; t += 2) {
         float o[2];
#pragma unroll
         for (int x = 0; x < 2; x++) {
            const float keep = f * (odd ? s.acc[t + 1][x] : s.acc[t][x]), give = f * (odd ? s.acc[t][x] : s.acc[t + 1][x]);
            const float got = __shfl_xor_sync(FULL, give, 16);
            o[x] = odd ? got - lam * keep : keep - lam * got;
         }
         if (mine) store_two<T, FORM>(out + 8 * t, o[0], o[1], p.dv - 8 * (t + odd) - 2 * l.c);
      }
      if (mine && l.c == 0 && p.lse) p.lse[rh * 2 + odd] = top + LN2 * (log2f(sum) - WEIGHT_LOG2<T>);
   }
   __device__ __forceinline__ void finish_empty(const AttnParams &p, const Place &at, long long row)
   {
      if (!heads.live) return;
      const long long rh = row * p.heads + heads.head;
      T *out = static_cast<T *>(p.out) + rh * p.dv + 2 * l.c;
      if (l.r < 4) {
#pragma unroll
         for (int t = 0; t < TILES; t++) store_two<T, FORM>(out + 8 * t, 0.0f, 0.0f, p.dv - 8 * t - 2 * l.c);
      }
      if (l.c == 0 && p.lse) p.lse[rh * 2 + (l.r >> 2)] = -INFINITY;
   }
};

// ---------------------------------------------------------------------------------------------------------------------
// backward over the rows (the sums A = sum p (dP - c) k, B = sum p k, D' = sum p (dP - c), D = sum p dP, Z = sum p of BackwardRows;
// c is the D / Z of the edges so far, after the first block and after each with an edge that is heavy against all before it).  For
// map 0 the rows of A's operand are w = p (dP - c) of the columns 0..3 and p of the same, for map 1 the other way round.
// 2^23 R-MAT edges, 4 heads of d 32, bf16: 1.58 ms, 5.4 TB/s gathered (1.48 with c = 0 and without Z); 2^21 edges: 411 instructions a
// block.  Spilled: up to 76 bytes of a lane at d 64, 104 to 292 at d 128.
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DK, int FORM, bool ONE>
struct BackwardRowsMma {
   static_assert(LOWER_SCALE<T> == 1.0f, "the parts of split numbers are added up as they are");
   using Cols = Columns<ONE>;
   static constexpr int N = Cols::N;
   static constexpr int DV = 2 * DK, TILES = DK / 8, LANE_FLOATS = 4 * TILES + 8;
   using Gathered = Ring<T, DK, FORM, Budget<DK, WALK_ROWS>::STAGES, false, true>;
   using Width = Budget<DK, WALK_ROWS>;
   struct State {
      float acc[2][TILES][2];
      float delta[N], total[N], rest[N], ref[N];  // D, Z, D' and c of this lane's columns
   };
   State s;
   Lanes l;
   QueryHeads<ONE> heads;
   int kv0;
   unsigned next[DK / 8], next_out[DV / 8];
   float next_lse[N];
   bool lost;

   __device__ __forceinline__ void setup(const AttnParams &p, const Place &at, Gathered &ring)
   {
      l.set(at, p.unit_kv);
      kv0 = (at.unit / p.head_blocks) * p.unit_kv;
      heads.set(p, at, l, kv0);
      ring.setup(p, l, at.lane, kv0);
   }
   static __device__ __forceinline__ void clear(State &s)
   {
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
         for (int t = 0; t < TILES; t++) s.acc[m][t][0] = s.acc[m][t][1] = 0.0f;
#pragma unroll
      for (int x = 0; x < N; x++) s.delta[x] = s.total[x] = s.rest[x] = s.ref[x] = 0.0f;
   }
   __device__ __forceinline__ void fetch(const AttnParams &p, long long row)
   {
      load_operand<T, DK, FORM>(static_cast<const T *>(p.q) + row * p.ldq + heads.head * p.hsq + (l.r >> 2) * p.d, l.c, p.d, p.step, next);
      load_operand<T, DV, FORM>(static_cast<const T *>(p.dout) + row * p.ldo + heads.head * p.hso, l.c, p.dv, p.step, next_out);
#pragma unroll
      for (int x = 0; x < N; x++) next_lse[x] = __ldg(p.lse + (row * p.heads + heads.col_head[x]) * 2 + (l.c >> 1));
   }

   // A new reference for the columns, the mean of dP so far; `pr`, `dp`: weights and dP of the present block, which are in no sum yet.
   // `sums`: there are any.
   __device__ __forceinline__ void rebase(float (&acc)[2][TILES][4], float (&mark)[N], const float (&pr)[2][N], const float (&dp)[4], int map, bool sums)
   {
      float shift[N];
#pragma unroll
      for (int x = 0; x < N; x++) {
         float delta = s.delta[x], total = s.total[x];
#pragma unroll
         for (int h = 0; h < 2; h++)
            if (pr[h][x] != 0.0f) {
               delta = fmaf(pr[h][x], Cols::pick(dp, h, x, l), delta);
               total += pr[h][x];
            }
         total = Cols::sum(total);
         const float mean = __fdividef(Cols::sum(delta), total), ref = fabsf(mean) < INFINITY ? mean : s.ref[x];
         shift[x] = s.ref[x] - ref;
         s.rest[x] = fmaf(shift[x], s.total[x], s.rest[x]);
         s.ref[x] = ref;
         mark[x] = reference_mark(total);
      }
      if (!sums) return;
      const float row_shift = Cols::of_row(shift, l.r);
#pragma unroll
      for (int t = 0; t < TILES; t++)
#pragma unroll
         for (int i = 0; i < 2; i++) {
            // the B of this lane's A lies 16 lanes away, in the sums of the same map
            const float give = map ? acc[0][t][i] + acc[0][t][i + 2] : acc[1][t][i] + acc[1][t][i + 2];
            const float b = __shfl_xor_sync(FULL, give, 16);
            if (map) acc[1][t][i] = fmaf(row_shift, b, acc[1][t][i]);
            else acc[0][t][i] = fmaf(row_shift, b, acc[0][t][i]);
         }
   }

   __device__ __forceinline__ void run(const AttnParams &p, const Place &at, Gathered &ring, int e0, int e1, long long follow)
   {
      float acc[2][TILES][4];
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
         for (int t = 0; t < TILES; t++) acc[m][t][0] = acc[m][t][1] = acc[m][t][2] = acc[m][t][3] = 0.0f;
#pragma unroll
      for (int x = 0; x < N; x++) s.delta[x] = s.total[x] = s.rest[x] = s.ref[x] = 0.0f;
      unsigned q[DK / 8], dout[DV / 8];
      float lse[N];
#pragma unroll
      for (int x = 0; x < N; x++) lse[x] = next_lse[x];
#pragma unroll
      for (int i = 0; i < DK / 8; i++) q[i] = next[i];
#pragma unroll
      for (int i = 0; i < DV / 8; i++) dout[i] = next_out[i];
      if (Width::AHEAD && follow >= 0) fetch(p, follow);
      const int per_log2 = 4 - l.slots_log2;
      // the lane's row and chunk of ldmatrix: pairs 0..7 and 8..15 of one chunk, then of the next; chunks by exclusive or
      const unsigned mine = Gathered::offset(at.lane & 15, at.lane >> 4);
      const int map = l.r >> 2;
      float mark[N];
#pragma unroll
      for (int x = 0; x < N; x++) mark[x] = 0.0f;
      for (int e = e0; e < e1;) {
         const int block = e >> per_log2;
         if (block != ring.current) ring.advance(p, l, at.lane);
         const int lo = e - (block << per_log2), left = e1 - (block << per_log2), hi = left < (1 << per_log2) ? left : 1 << per_log2;
         const unsigned slot = ring.slot;
         float s0[4], s1[4], dp[4], dp2[4];
#pragma unroll
         for (int i = 0; i < DK / 16; i++) {
            unsigned k[4];
            ldmatrix4(k, (slot + mine) ^ ((2 * i) << 4));
            mma16816_at<T>(i == 0, s0, k, q[2 * i], q[2 * i + 1]);
            ldmatrix4(k, (slot + mine) ^ ((DK / 8 + 2 * i) << 4));
            mma16816_at<T>(i == 0, s1, k, q[2 * i], q[2 * i + 1]);
         }
#pragma unroll
         for (int i = 0; i < DV / 16; i++) {
            unsigned v[4];
            ldmatrix4(v, (slot + mine + Gathered::REGION) ^ ((2 * i) << 4));
            mma16816_at<T>(i < 2, i & 1 ? dp2 : dp, v, dout[2 * i], dout[2 * i + 1]);  // two sums side by side
         }
#pragma unroll
         for (int i = 0; i < 4; i++) dp[i] += dp2[i];
         float pr[2][N];
         bool grown = false;
#pragma unroll
         for (int h = 0; h < 2; h++) {
            const int edge = (l.r + 8 * h) >> l.slots_log2;
            const float bias = shared_float(slot + Gathered::BIAS + 4 * edge);
            const bool there = edge >= lo && edge < hi && bias != -INFINITY;
#pragma unroll
            for (int x = 0; x < N; x++) {
               // an edge that is masked has p = -0, and so has a row without edges (its lse is -inf)
               const bool live = heads.valid[x] && there && lse[x] != -INFINITY;
               pr[h][x] = live ? weight_of(fmaf(Cols::pick(s0, s1, h, x, l), p.scale, bias), lse[x]) : -0.0f;
               grown |= pr[h][x] > mark[x];
            }
         }
         if (__any_sync(FULL, grown)) rebase(acc, mark, pr, dp, map, e != e0);
         unsigned a0[4], a1[4];
#pragma unroll
         for (int h = 0; h < 2; h++) {
            float w[N];
#pragma unroll
            for (int x = 0; x < N; x++) {
               const float d = signbit(pr[h][x]) ? s.ref[x] : Cols::pick(dp, h, x, l);
               w[x] = pr[h][x] * (d - s.ref[x]);
               s.rest[x] += w[x];
               s.delta[x] = fmaf(pr[h][x], d, s.delta[x]);
               s.total[x] += pr[h][x];
            }
            unsigned wh, wl, ph, pl;
            Cols::template split<T>(w, l, wh, wl);
            Cols::template split<T>(pr[h], l, ph, pl);
            wh = transpose8x8(wh);
            wl = transpose8x8(wl);
            ph = __shfl_xor_sync(FULL, transpose8x8(ph), 16);
            pl = __shfl_xor_sync(FULL, transpose8x8(pl), 16);
            a0[2 * h] = l.r < 4 ? wh : ph;
            a0[2 * h + 1] = l.r < 4 ? wl : pl;
            a1[2 * h] = l.r < 4 ? ph : wh;
            a1[2 * h + 1] = l.r < 4 ? pl : wl;
         }
#pragma unroll
         for (int t = 0; t < TILES; t += 2) {
            unsigned k[4];
            ldmatrix4_trans(k, (slot + mine) ^ ((t) << 4));
            mma16816<T>(acc[0][t], a0[0], a0[1], a0[2], a0[3], k[0], k[1]);
            mma16816<T>(acc[0][t + 1], a0[0], a0[1], a0[2], a0[3], k[2], k[3]);
            ldmatrix4_trans(k, (slot + mine) ^ ((DK / 8 + t) << 4));
            mma16816<T>(acc[1][t], a1[0], a1[1], a1[2], a1[3], k[0], k[1]);
            mma16816<T>(acc[1][t + 1], a1[0], a1[1], a1[2], a1[3], k[2], k[3]);
         }
         e = (block << per_log2) + hi;
      }
      float all = 0.0f;
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
         for (int t = 0; t < TILES; t++) {
            s.acc[m][t][0] = acc[m][t][0] + acc[m][t][2];
            s.acc[m][t][1] = acc[m][t][1] + acc[m][t][3];
            all += s.acc[m][t][0] * 0.0f + s.acc[m][t][1] * 0.0f;
         }
      lost = all != all;
#pragma unroll
      for (int x = 0; x < N; x++) {
         s.delta[x] = Cols::sum(s.delta[x]);
         s.total[x] = Cols::sum(s.total[x]);
         s.rest[x] = Cols::sum(s.rest[x]);
      }
   }

   __device__ __forceinline__ void join_from(const float *unit, const Place &at)
   {
      const float2 *from = reinterpret_cast<const float2 *>(unit) + at.lane;
      float2 o[2][TILES];  // all loads before the first sum
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
         for (int t = 0; t < TILES; t++) o[m][t] = from[32 * (m * TILES + t)];
      // rows 0..3 hold A of map 0 and B of map 1, rows 4..7 B of map 0 and A of map 1: the B of this lane's A lies 16 lanes away
      const int map = l.r >> 2;
      const float2 *other = reinterpret_cast<const float2 *>(unit) + (at.lane ^ 16) + 32 * map * TILES;
      float2 c[TILES];
#pragma unroll
      for (int t = 0; t < TILES; t++) c[t] = other[32 * t];
      const float2 d = from[64 * TILES], z = from[64 * TILES + 32], rest = from[64 * TILES + 64], ref = from[64 * TILES + 96];
      float shift[N], shift_o[N];
      bool moved = false;
#pragma unroll
      for (int x = 0; x < N; x++) {
         const float total = x ? z.y : z.x;
         join_references(s.total[x], s.ref[x], total, x ? ref.y : ref.x, shift[x], shift_o[x]);
         moved |= shift[x] != 0.0f;
         s.delta[x] += x ? d.y : d.x;
         s.rest[x] = fmaf(shift[x], s.total[x], s.rest[x]) + fmaf(shift_o[x], total, x ? rest.y : rest.x);
         s.total[x] += total;
      }
      if (__any_sync(FULL, moved)) {
         const float f = Cols::of_row(shift, l.r);
#pragma unroll
         for (int t = 0; t < TILES; t++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
               const float b = __shfl_xor_sync(FULL, map ? s.acc[0][t][i] : s.acc[1][t][i], 16);
               if (map) s.acc[1][t][i] = fmaf(f, b, s.acc[1][t][i]);
               else s.acc[0][t][i] = fmaf(f, b, s.acc[0][t][i]);
            }
      }
      const float f = Cols::of_row(shift_o, l.r);
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
         for (int t = 0; t < TILES; t++) {
            s.acc[m][t][0] += m == map ? fmaf(f, c[t].x, o[m][t].x) : o[m][t].x;
            s.acc[m][t][1] += m == map ? fmaf(f, c[t].y, o[m][t].y) : o[m][t].y;
         }
   }
   __device__ __forceinline__ void put(float *unit, const Place &at, int only) const
   {
      float2 *to = reinterpret_cast<float2 *>(unit) + at.lane;
      if (only < 0 || heads.kv == only) {
#pragma unroll
         for (int m = 0; m < 2; m++)
#pragma unroll
            for (int t = 0; t < TILES; t++) to[32 * (m * TILES + t)] = make_float2(s.acc[m][t][0], s.acc[m][t][1]);
      }
      float *delta = reinterpret_cast<float *>(to + 64 * TILES), *total = delta + 64, *rest = delta + 128, *ref = delta + 192;
#pragma unroll
      for (int x = 0; x < N; x++)
         if (only < 0 || heads.col_kv[x] == only) {
            delta[x] = s.delta[x];
            total[x] = s.total[x];
            rest[x] = s.rest[x];
            ref[x] = s.ref[x];
         }
   }

   __device__ __forceinline__ void finish(const AttnParams &p, const Place &at, long long row, int only)
   {
      const float inverse = reciprocal_total(Cols::of_row(s.total, l.r));
      const float delta = Cols::of_row(s.delta, l.r) * inverse, rest = Cols::of_row(s.rest, l.r) * inverse;
      const bool mine = heads.live && (only < 0 || heads.kv == only);
      const int map = l.r >> 2;
      const long long rh = row * p.heads + heads.head;
      const float sign = (map ? -__ldg(p.lam + row * p.ldlam + heads.head) : 1.0f) * inverse, factor = sign * p.scale;
      T *out = static_cast<T *>(p.out) + (rh * 2 + map) * p.d + 2 * l.c;
#pragma unroll
      for (int t = 0; t < TILES; t++) {
         float o[2];
#pragma unroll
         for (int x = 0; x < 2; x++) {
            // rows 0..3 hold A of map 0 and B of map 1, rows 4..7 B of map 0 and A of map 1
            const float b = __shfl_xor_sync(FULL, map ? s.acc[0][t][x] : s.acc[1][t][x], 16);
            o[x] = factor * fmaf(-rest, b, map ? s.acc[1][t][x] : s.acc[0][t][x]);
         }
         if (mine) store_two<T, FORM>(out + 8 * t, o[0], o[1], p.d - 8 * t - 2 * l.c);
      }
      if (mine && l.c == 0) {
         p.stats[rh * 2 + map] = make_float4(__ldg(p.lse + rh * 2 + map), delta, sign, 0.0f);
         if (map) p.dlam[rh] = -delta;
      }
   }
   __device__ __forceinline__ void finish_empty(const AttnParams &p, const Place &at, long long row)
   {
      if (!heads.live) return;
      const int map = l.r >> 2;
      const long long rh = row * p.heads + heads.head;
      T *out = static_cast<T *>(p.out) + (rh * 2 + map) * p.d + 2 * l.c;
#pragma unroll
      for (int t = 0; t < TILES; t++) store_two<T, FORM>(out + 8 * t, 0.0f, 0.0f, p.d - 8 * t - 2 * l.c);
      if (l.c == 0 && map) p.dlam[rh] = 0.0f;  // nobody gathers the row: its record is not read
   }
};

// ---------------------------------------------------------------------------------------------------------------------
// backward over the columns: dk and dv.  A pair is an edge with a query head; the columns of the products are (map, kv head of
// the unit).  dk and dv are [16 elements x 8] products over the pairs: the columns 0..3 take the upper and 4..7 the lower part
// of the split ds (or weight) of the unit's kv heads.
// 2^23 R-MAT edges, 4 heads of d 32, bf16: 1.57 ms, 5.5 TB/s gathered, bound by the instructions' latency (2.14 ms without SINGLE,
// which leaves out the division of blocks among groups of heads, and with a longer exchange in write()); 2^21 edges: 423
// instructions a block.
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DK, int FORM, bool SINGLE>
struct BackwardColumnsMma {
   static_assert(LOWER_SCALE<T> == 1.0f, "the parts of split numbers are added up as they are");
   static constexpr int DV = 2 * DK, KT = DK / 16, VT = DV / 16, LANE_FLOATS = 4 * (2 * KT + VT);
   using Gathered = Ring<T, DK, FORM, Budget<DK, WALK_COLUMNS>::STAGES, true, SINGLE>;
   using Width = Budget<DK, WALK_COLUMNS>;
   struct State {
      float dk[2][KT][4], dv[VT][4];
   };
   State s;
   Lanes l;
   int kv0, per_kv;       // query heads of a kv head that a block holds
   int pair_kv;           // which of the unit's kv heads the pairs r and r + 8 are of
   unsigned next[DK / 8], next_v[DV / 8];
   bool lost;

   __device__ __forceinline__ void setup(const AttnParams &p, const Place &at, Gathered &ring)
   {
      l.set(at, p.unit_kv * p.unit_heads);
      kv0 = at.unit * p.unit_kv;
      per_kv = p.unit_heads;
      pair_kv = l.pair_slot / per_kv;
      const long long head = kv0 * p.group;
      ring.setup(p, l, at.lane, kv0 * p.group);
      ring.records = reinterpret_cast<const char *>(p.stats + head * 2);
   }
   static __device__ __forceinline__ void clear(State &s)
   {
#pragma unroll
      for (int t = 0; t < KT; t++)
#pragma unroll
         for (int i = 0; i < 4; i++) s.dk[0][t][i] = s.dk[1][t][i] = 0.0f;
#pragma unroll
      for (int t = 0; t < VT; t++)
#pragma unroll
         for (int i = 0; i < 4; i++) s.dv[t][i] = 0.0f;
   }
   __device__ __forceinline__ void fetch(const AttnParams &p, long long col)
   {
      // column n = r: map r / 4, kv head r % 4 of the unit (one that exists stands for those beyond)
      const int head = kv0 + ((l.r & 3) < p.unit_kv ? l.r & 3 : 0);
      load_operand<T, DK, FORM>(static_cast<const T *>(p.k) + col * p.ldk + head * p.hsk + (l.r >> 2) * p.d, l.c, p.d, p.step, next);
      load_operand<T, DV, FORM>(static_cast<const T *>(p.v) + col * p.ldv + head * p.hsv, l.c, p.dv, p.step, next_v);
   }

   __device__ __forceinline__ void run(const AttnParams &p, const Place &at, Gathered &ring, int e0, int e1, long long follow)
   {
      clear(s);
      unsigned k[DK / 8], v[DV / 8];
#pragma unroll
      for (int i = 0; i < DK / 8; i++) k[i] = next[i];
#pragma unroll
      for (int i = 0; i < DV / 8; i++) v[i] = next_v[i];
      if (Width::AHEAD && follow >= 0) fetch(p, follow);
      const int per_log2 = 4 - l.slots_log2;
      // the lane's row and chunk of ldmatrix: pairs 0..7 and 8..15 of one chunk, then of the next; chunks by exclusive or
      const unsigned mine = Gathered::offset(at.lane & 15, at.lane >> 4);
      // ... and as columns: pairs 0..7 of one chunk and the next, then pairs 8..15, the order of the A operand's registers
      const unsigned mine_t = Gathered::offset((at.lane & 7) + (at.lane >> 4) * 8, at.lane >> 3 & 1);
      // of the columns 2c, 2c + 1 at most one is of the pairs' kv head
      const bool valid = (l.c & 1) == pair_kv >> 1;
      const int x = pair_kv & 1, map = l.c >> 1;
      for (int e = e0; e < e1;) {
         const int edges = e >> per_log2;
         const int lo = e - (edges << per_log2), left = e1 - (edges << per_log2), hi = left < (1 << per_log2) ? left : 1 << per_log2;
         for (int sub = 0; sub < (SINGLE ? 1 : p.subs); sub++) {
            const int block = SINGLE ? edges : edges * p.subs + sub;
            if (block != ring.current) ring.advance(p, l, at.lane);
            const unsigned slot = ring.slot;
            float s0[4], s1[4], dp[4], dp2[4];
#pragma unroll
            for (int i = 0; i < DK / 16; i++) {
               unsigned q[4];
               ldmatrix4(q, (slot + mine) ^ ((2 * i) << 4));
               mma16816_at<T>(i == 0, s0, q, k[2 * i], k[2 * i + 1]);
               ldmatrix4(q, (slot + mine) ^ ((DK / 8 + 2 * i) << 4));
               mma16816_at<T>(i == 0, s1, q, k[2 * i], k[2 * i + 1]);
            }
#pragma unroll
            for (int i = 0; i < DV / 16; i++) {
               unsigned d[4];
               ldmatrix4(d, (slot + mine + Gathered::REGION) ^ ((2 * i) << 4));
               mma16816_at<T>(i < 2, i & 1 ? dp2 : dp, d, v[2 * i], v[2 * i + 1]);  // two sums side by side
            }
#pragma unroll
            for (int i = 0; i < 4; i++) dp[i] += dp2[i];
            unsigned b0[2], b1[2], bw[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
               const int edge = (l.r + 8 * h) >> l.slots_log2;
               const float bias = shared_float(slot + Gathered::BIAS + 4 * edge);
               float lse, delta, sign, none;
               asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(lse), "=f"(delta), "=f"(sign), "=f"(none)
                            : "r"(slot + Gathered::RECORD + (l.r + 8 * h) * 32 + map * 16) : "memory");
               // an edge of this column, of a row that has any, and this lane's column is the pair's
               const bool live = valid && edge >= lo && edge < hi && bias != -INFINITY && lse != -INFINITY;
               const float dot = map ? (x ? s1[2 * h + 1] : s1[2 * h]) : (x ? s0[2 * h + 1] : s0[2 * h]);
               const float pr = live ? weight_of(fmaf(dot, p.scale, bias), lse) : 0.0f;
               const float part = live ? sign * pr : 0.0f;  // this map's part of the weight
               const float w = part + __shfl_xor_sync(FULL, part, 2);
               const float ds = live ? part * ((x ? dp[2 * h + 1] : dp[2 * h]) - delta) : 0.0f;
               unsigned up, low, wh, wl;
               split2<T>(x ? 0.0f : ds, x ? ds : 0.0f, up, low);
               split2<T>(x ? 0.0f : w, x ? w : 0.0f, wh, wl);
               const unsigned got = __shfl_xor_sync(FULL, l.c < 2 ? low : up, 2);
               b0[h] = transpose8x8(l.c < 2 ? up : got);
               b1[h] = transpose8x8(l.c < 2 ? got : low);
               bw[h] = transpose8x8(l.c < 2 ? wh : wl);
            }
#pragma unroll
            for (int t = 0; t < KT; t++) {
               unsigned q[4];
               ldmatrix4_trans(q, (slot + mine_t) ^ ((2 * t) << 4));
               mma16816<T>(s.dk[0][t], q[0], q[1], q[2], q[3], b0[0], b0[1]);
               ldmatrix4_trans(q, (slot + mine_t) ^ ((DK / 8 + 2 * t) << 4));
               mma16816<T>(s.dk[1][t], q[0], q[1], q[2], q[3], b1[0], b1[1]);
            }
#pragma unroll
            for (int t = 0; t < VT; t++) {
               unsigned d[4];
               ldmatrix4_trans(d, (slot + mine_t + Gathered::REGION) ^ ((2 * t) << 4));
               mma16816<T>(s.dv[t], d[0], d[1], d[2], d[3], bw[0], bw[1]);
            }
         }
         e = (edges << per_log2) + hi;
      }
      float all = 0.0f;
#pragma unroll
      for (int t = 0; t < KT; t++)
#pragma unroll
         for (int i = 0; i < 4; i++) all += s.dk[0][t][i] * 0.0f + s.dk[1][t][i] * 0.0f;
#pragma unroll
      for (int t = 0; t < VT; t++)
#pragma unroll
         for (int i = 0; i < 4; i++) all += s.dv[t][i] * 0.0f;
      lost = all != all;
   }

   __device__ __forceinline__ void join_from(const float *unit, const Place &at)
   {
      const float4 *from = reinterpret_cast<const float4 *>(unit) + at.lane;
      float4 o[2 * KT + VT];  // all loads before the first sum
#pragma unroll
      for (int i = 0; i < 2 * KT + VT; i++) o[i] = from[32 * i];
#pragma unroll
      for (int i = 0; i < 2 * KT + VT; i++) {
         float (&f)[4] = i < KT ? s.dk[0][i] : i < 2 * KT ? s.dk[1][i - KT] : s.dv[i - 2 * KT];
         f[0] += o[i].x; f[1] += o[i].y; f[2] += o[i].z; f[3] += o[i].w;
      }
   }
   // a head's sums lie in the results' columns 2c, 2c + 1 (and 4 further): the lane's kv heads 2c % 4, 2c % 4 + 1
   __device__ __forceinline__ void put(float *unit, const Place &at, int only) const
   {
      float4 *to = reinterpret_cast<float4 *>(unit) + at.lane;
      const int kv = (2 * l.c) & 3;
#pragma unroll
      for (int i = 0; i < 2 * KT + VT; i++) {
         const float (&f)[4] = i < KT ? s.dk[0][i] : i < 2 * KT ? s.dk[1][i - KT] : s.dv[i - 2 * KT];
         if (only < 0) {
            to[32 * i] = make_float4(f[0], f[1], f[2], f[3]);
         } else {
            float *one = reinterpret_cast<float *>(to + 32 * i);
            if (kv == only) { one[0] = f[0]; one[2] = f[2]; }
            if (kv + 1 == only) { one[1] = f[1]; one[3] = f[3]; }
         }
      }
   }

   // Tile t of a head's sums lies in the lanes as rows r (elements 16t + r) and r + 8, upper parts of the kv heads 2c, 2c + 1 at
   // c < 2, lower parts at c + 2.  Those two lanes trade so that one has the elements 16t + r whole and the other 16t + 8 + r;
   // then neighbouring r trade so that one has two consecutive elements of the first head and the other of the second.
   template <int TILES>
   __device__ __forceinline__ void write(const float (&f)[TILES][4], T *row, long long head_step, int width, float factor, int only)
   {
      const bool low = l.c >= 2, odd = l.r & 1;
      const int kv = 2 * (l.c & 1) + odd, y = (low ? 8 : 0) + (l.r & ~1);
      const bool mine = only < 0 ? kv * per_kv < l.slots : kv == only;
      T *to = row + kv * head_step + y;
#pragma unroll
      for (int t = 0; t < TILES; t++) {
         const float g0 = __shfl_xor_sync(FULL, low ? f[t][0] : f[t][2], 2), g1 = __shfl_xor_sync(FULL, low ? f[t][1] : f[t][3], 2);
         const float v0 = factor * ((low ? f[t][2] : f[t][0]) + g0), v1 = factor * ((low ? f[t][3] : f[t][1]) + g1);
         const float got = __shfl_xor_sync(FULL, odd ? v0 : v1, 4);
         if (mine) store_two<T, FORM>(to + 16 * t, odd ? got : v0, odd ? v1 : got, width - y - 16 * t);
      }
   }
   __device__ __forceinline__ void finish(const AttnParams &p, const Place &at, long long col, int only)
   {
      const long long rh = col * p.kv_heads + kv0;
      write<KT>(s.dk[0], static_cast<T *>(p.out) + rh * 2 * p.d, 2 * p.d, p.d, p.scale, only);
      write<KT>(s.dk[1], static_cast<T *>(p.out) + rh * 2 * p.d + p.d, 2 * p.d, p.d, p.scale, only);
      write<VT>(s.dv, static_cast<T *>(p.out2) + rh * p.dv, p.dv, p.dv, 1.0f, only);
   }
   __device__ __forceinline__ void finish_empty(const AttnParams &p, const Place &at, long long col)
   {
      const long long rh = col * p.kv_heads + kv0;
      T *dk = static_cast<T *>(p.out) + rh * 2 * p.d, *dv = static_cast<T *>(p.out2) + rh * p.dv;
      for (int i = 2 * at.lane; i < p.unit_kv * 2 * p.d; i += 64) store_two<T, FORM>(dk + i, 0.0f, 0.0f, p.unit_kv * 2 * p.d - i);
      for (int i = 2 * at.lane; i < p.unit_kv * p.dv; i += 64) store_two<T, FORM>(dv + i, 0.0f, 0.0f, p.unit_kv * p.dv - i);
   }
};

// ---------------------------------------------------------------------------------------------------------------------
// the walk
// ---------------------------------------------------------------------------------------------------------------------
// the warps of a block that shared a row join their states by halves; the rings serve as the place
template <typename Op>
__device__ __forceinline__ void join_ring_warps(Op &op, const Place &at, float *shared, int warps)
{
   constexpr int STRIDE = Op::LANE_FLOATS * 32;
   for (int half = warps / 2; half > 0; half /= 2) {
      __syncthreads();
      if (at.warp >= half && at.warp < 2 * half) op.put(shared + (at.warp - half) * STRIDE, at, -1);
      __syncthreads();
      if (at.warp < half) op.join_from(shared + at.warp * STRIDE, at);
   }
}

// Where a sum came out infinite or as no number, a weight of 0 may have met an infinity or NaN of another row's edge in the same
// block, or of another head: the row's edges are then taken once more, in blocks of their own and each kv head by itself.
template <typename Op, bool TOGETHER>
__device__ __forceinline__ void ring_segment(Op &op, typename Op::Gathered &ring, const AttnParams &p, const Place &at, float *shared,
                                             long long row, long long e0, long long e1, long long part, long long follow, long long run_end)
{
   long long w0 = e0, w1 = e1;
   if (TOGETHER) {  // equal runs of whole blocks
      const int per_log2 = 4 - op.l.slots_log2;
      const long long blocks = (e1 - e0 + (1 << per_log2) - 1) >> per_log2, each = (blocks + Op::Width::JOINT - 1) / Op::Width::JOINT;
      w0 = e0 + ((at.warp * each) << per_log2);
      w1 = w0 + (each << per_log2);
      w0 = w0 < e1 ? w0 : e1;
      w1 = w1 < e1 ? w1 : e1;
      ring.begin(p, op.l, at.lane, w0, w1, -1);
   }
   op.run(p, at, ring, static_cast<int>(w0 - ring.first), static_cast<int>(w1 - ring.first), follow);
   const bool lost = TOGETHER ? p.unit_kv > 1 && __syncthreads_or(op.lost) : __any_sync(FULL, op.lost);
   for (int only = lost ? 0 : -1; only < (lost ? p.unit_kv : 0); only++) {
      if (lost) {
         op.fetch(p, row);
         ring.begin(p, op.l, at.lane, w0, w1, only);
         op.run(p, at, ring, 0, static_cast<int>(w1 - w0), only == p.unit_kv - 1 ? follow : -1);
      }
      if (TOGETHER) {
         ring.drain();
         join_ring_warps(op, at, shared, Op::Width::JOINT);
      }
      if (!TOGETHER || at.warp == 0) {
         if (part < 0) op.finish(p, at, row, only);
         else op.put(part_at<Op, 32>(p, at, part), at, only);
      }
      if (TOGETHER) __syncthreads();
   }
   if (lost && !TOGETHER && Op::Gathered::SINGLE) ring.begin(p, op.l, at.lane, e1, run_end, -1);
}

constexpr int RING_ALIGN = 512;  // the longest row of a ring

template <typename Op, bool TOGETHER>
__global__ void __launch_bounds__((TOGETHER ? Op::Width::JOINT : Op::Width::SOLO) * 32, TOGETHER ? 1 : Op::Width::BLOCKS)
ring_walk_kernel(const AttnParams p)
{
   extern __shared__ __align__(128) float shared[];
   constexpr int WARPS = TOGETHER ? Op::Width::JOINT : Op::Width::SOLO;
   const int warp = threadIdx.x >> 5;
   const long long job = TOGETHER ? blockIdx.x : static_cast<long long>(blockIdx.x) * WARPS + warp;
   const long long piece = job / p.unit_blocks;
   if (piece >= p.pieces) return;
   const Place at = Place::make<32>(p, static_cast<int>(job - piece * p.unit_blocks));
   const Rows rows(p);
   const long long lo = piece * p.piece, hi = lo + p.piece;
   Op op;
   typename Op::Gathered ring;
   ring.ring = ((static_cast<unsigned>(__cvta_generic_to_shared(shared)) + RING_ALIGN - 1) & ~(RING_ALIGN - 1u)) + warp * (Op::Gathered::STAGES * Op::Gathered::STAGE);
   op.setup(p, at, ring);
   long long u = rows.lower_bound(lo, 0, p.m, at.lane);
   // the rows that begin in this piece end before `last`: a row is ROW_ITEMS items at least
   const long long most = u + p.piece / ROW_ITEMS + 1;
   const long long last = rows.lower_bound(hi, u, most < p.m ? most : p.m, at.lane);
   long long begun = -1;
   if (u > 0) {  // the row before may reach into this piece: then it is this loop's first
      const long long fb = rows.items(u - 1), fe = rows.items(u);
      if (fe > lo && fe - fb > p.row_limit) u--;
   }
   // the run of edges: up to the last row's end, or where it is cut
   auto part_of = [&](long long row, long long b, long long e, long long &e0, long long &e1) {
      const long long fb = b - rows.first + ROW_ITEMS * row, fe = e - rows.first + ROW_ITEMS * (row + 1);
      e0 = b;
      e1 = e > b ? e : b;
      if (fe - fb <= p.row_limit) return -1LL;
      e0 = b + (lo - fb - ROW_ITEMS);
      e1 = b + (hi - fb - ROW_ITEMS);
      e0 = e0 < b ? b : e0;
      e1 = e1 > e ? e : e1 < e0 ? e0 : e1;
      return 2 * piece + (fb >= lo);
   };
   if (u < last) {
      long long run_begin, run_end, x;
      part_of(u, rows.begin(u), rows.begin(u + 1), run_begin, x);
      part_of(last - 1, rows.begin(last - 1), rows.begin(last), x, run_end);
      if (run_end - run_begin > INT_MAX - 64) run_end = run_begin + (INT_MAX - 64);  // (row pointers that decrease: the ring counts in 32 bits)
      // (where a row's edges are taken once for each of several groups of heads, every row is a run of its own)
      if (!TOGETHER && Op::Gathered::SINGLE) ring.begin(p, op.l, at.lane, run_begin, run_end, -1);
      // rows 31 at a time, their pointers one to a lane; rows with edges are found by their bits
      for (long long from = u; from < last; from += 31) {
         const int here = static_cast<int>(last - from < 31 ? last - from : 31);
         const long long mine = rows.begin(from + at.lane < p.m ? from + at.lane : p.m);
         const long long behind = __shfl_down_sync(FULL, mine, 1);
         long long m0 = 0, m1 = 0, part = -1;
         if (at.lane < here) part = part_of(from + at.lane, mine, behind, m0, m1);
         if (!TOGETHER && Op::Gathered::SINGLE) {  // likewise: no row leads out of the ring's run
            const long long end = ring.first + ring.length;
            m0 = m0 < ring.first ? ring.first : m0 > end ? end : m0;
            m1 = m1 < m0 ? m0 : m1 > end ? end : m1;
         }
         const unsigned busy = __ballot_sync(FULL, at.lane < here && (m1 > m0 || part >= 0));
         const unsigned starts = __ballot_sync(FULL, part >= 0 && (part & 1));
         if (starts) begun = from + __ffs(starts) - 1;
         for (unsigned none = ~busy & ((1u << here) - 1); none; none &= none - 1)
            if (!TOGETHER || warp == 0) op.finish_empty(p, at, from + __ffs(none) - 1);
         if (Op::Width::AHEAD && busy) op.fetch(p, from + __ffs(busy) - 1);
         for (unsigned todo = busy; todo;) {
            const int i = __ffs(todo) - 1;
            todo &= todo - 1;
            const long long e0 = __shfl_sync(FULL, m0, i), e1 = __shfl_sync(FULL, m1, i), pt = __shfl_sync(FULL, part, i);
            if (!TOGETHER && !Op::Gathered::SINGLE) ring.begin(p, op.l, at.lane, e0, e1, -1);
            if (!Op::Width::AHEAD) op.fetch(p, from + i);
            ring_segment<Op, TOGETHER>(op, ring, p, at, shared, from + i, e0, e1, pt, todo ? from + __ffs(todo) - 1 : -1, run_end);
         }
      }
   }
   ring.drain();
   if (at.lane == 0 && (!TOGETHER || warp == 0) && job == piece * p.unit_blocks) p.long_row[piece] = begun;
}

// the parts of the long rows, as join_kernel
template <typename Op>
__global__ void __launch_bounds__(512) ring_join_kernel(const AttnParams p)
{
   extern __shared__ __align__(16) float shared[];
   const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
   const Place at = Place::make<32>(p, static_cast<int>(blockIdx.x % p.unit_blocks));
   const Rows rows(p);
   Op op;
   typename Op::Gathered ring;
   ring.ring = 0;
   op.setup(p, at, ring);
   LongRows todo(p, blockIdx.x / p.unit_blocks);
   long long u, piece, parts;
   while (todo.next(p, rows, u, piece, parts)) {
      const long long each = (parts + warps - 1) / warps;
      Op::clear(op.s);
      for (long long i = warp * each; i < (warp + 1) * each && i < parts; i++)
         op.join_from(part_at<Op, 32>(p, at, 2 * (piece + i) + (i == 0 ? 1 : 0)), at);
      join_ring_warps(op, at, shared, warps);
      if (warp == 0) op.finish(p, at, u, -1);
   }
}

template <typename Op>
int launch_ring(const AttnParams &p, bool together, cudaStream_t st)
{
   constexpr int RING = Op::Gathered::STAGES * Op::Gathered::STAGE;
   constexpr int STATE = 32 * Op::LANE_FLOATS * static_cast<int>(sizeof(float));
   static_assert(Op::Width::JOINT / 2 * STATE <= Op::Width::JOINT * RING, "the rings serve as the place where warps meet");
   const long long jobs = p.pieces * p.unit_blocks;
   if (together) {
      constexpr int bytes = Op::Width::JOINT * RING + RING_ALIGN;
      if (!allow_shared<ring_walk_kernel<Op, true>>(bytes)) return -1;
      ring_walk_kernel<Op, true><<<static_cast<unsigned>(jobs), Op::Width::JOINT * 32, bytes, st>>>(p);
   } else {
      constexpr int bytes = Op::Width::SOLO * RING + RING_ALIGN;
      if (!allow_shared<ring_walk_kernel<Op, false>>(bytes)) return -1;
      ring_walk_kernel<Op, false><<<static_cast<unsigned>((jobs + Op::Width::SOLO - 1) / Op::Width::SOLO), Op::Width::SOLO * 32, bytes, st>>>(p);
   }
   // one row of a long list has hundreds of parts: many warps for it; few where many rows have a few
   const int join_warps = together ? 16 : 4;
   if (!allow_shared<ring_join_kernel<Op>>(8 * STATE)) return -1;
   ring_join_kernel<Op><<<join_blocks(p), join_warps * 32, join_warps / 2 * STATE, st>>>(p);
   return 0;
}

template <typename T, int DK, bool ONE, template <typename, int, int, bool> class Op>
int launch_mma_form(const WalkShape &s, const AttnParams &p, cudaStream_t st)
{
   if (s.form == EXACT) return launch_ring<Op<T, DK, EXACT, ONE>>(p, s.together, st);
   if (s.form == RAGGED) return launch_ring<Op<T, DK, RAGGED, ONE>>(p, s.together, st);
   return launch_ring<Op<T, DK, PIECES, ONE>>(p, s.together, st);
}

// The last parameter of a walk: over the rows, four kv heads to a unit; over the columns, one group of heads.
template <typename T, bool ROWS, template <typename, int, int, bool> class Op>
int launch_mma(const WalkShape &s, const AttnParams &p, cudaStream_t st)
{
   if (ROWS ? p.unit_kv == 4 : p.subs == 1) {
      if (s.width == 16) return launch_mma_form<T, 16, true, Op>(s, p, st);
      if (s.width == 32) return launch_mma_form<T, 32, true, Op>(s, p, st);
      if (s.width == 64) return launch_mma_form<T, 64, true, Op>(s, p, st);
      if (s.width == 128) return launch_mma_form<T, 128, true, Op>(s, p, st);
   }
   if (s.width == 16) return launch_mma_form<T, 16, false, Op>(s, p, st);
   if (s.width == 32) return launch_mma_form<T, 32, false, Op>(s, p, st);
   if (s.width == 64) return launch_mma_form<T, 64, false, Op>(s, p, st);
   if (s.width == 128) return launch_mma_form<T, 128, false, Op>(s, p, st);
   return -1;
}

}  // namespace attn
}  // namespace fmm
