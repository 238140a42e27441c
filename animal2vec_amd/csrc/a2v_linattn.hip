// Linear attention with a decay per head (no softmax; the recurrent counterpart of the ALiBi term): for one head
//     S_t = l S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t,   l = exp(-slope)            S: HD x HD, 32 bits
// Chunked form over C rows (i, j local to the chunk, Y = l S at its start, "the state as its first row sees it"):
//     o_i = scale (sum_{j <= i} l^(i-j) (q_i . k_j) v_j + l^i Y^T q_i)
//     Y'  = l^C Y + sum_j l^(C-j) k_j v_j^T
// Every power of l is <= 1, so nothing overflows however strong the decay.
//
// The backward pass is the same sum three times, with D_t = l D_{t+1} + scale q_t do_t^T running backwards in time:
//     dq_t = scale S_t do_t    forward in time,  (q, k, v) := (do, v, k),        state S^T
//     dv_t = D_t^T k_t         backwards,        (q, k, v) := (k, q, scale do),  state D
//     dk_t = D_t v_t           backwards,        (q, k, v) := (v, scale do, q),  state D^T
// so ONE kernel does all four: a "role" names its operands, its direction and where the scale goes.
//
// One workgroup owns a (sequence, head) or a segment of one -- or the same of two or four neighbouring heads, for longer pieces of rows -- and
// walks its chunks with the state in registers.  A wave owns 16 columns
// of v: the whole HD x 16 slice of the state lives in its MFMA accumulators, whose layout IS the A operand of Y^T q, so the state never
// passes through LDS.  The scores do: a wave forms one 16 x 16 tile of them for all waves (each wave forming all of them instead: 6 % more
// for the training pair of 140-row clips, 13 % with 128 channels).
// Products are issued swapped (P^T = K Q^T, O^T = V^T P^T + Y^T Q^T): see a2v_attn.hip for the layout argument.
//
// All products run on the bf16 matrix cores, fp32 values as sums of bf16 parts of 8 bits each (x = hi + mid + lo exactly; the products of
// parts are exact in the fp32 accumulators):
//   bf16 operands: q, k, v are one part; scores, the state that rows read and the scaled values that it sums are three, all of their 32 bits.
//     (Two parts, 2^-16 relative, turn over one rounding in 1000 of the results and are 6 % faster: 64 clips of 2000 rows 214 us against 218, the
//     training pair of 140-row clips 156 against 181.)
//   fp32 operands: three parts of everything, six products of parts (the three below 2^-24 are dropped): 96 matrix cycles for 32 channels
//     of a 16 x 16 tile where v_mfma_f32_16x16x4_f32 takes 256.
#include "a2v_common.h"
#include <type_traits>

typedef __attribute__((address_space(3))) s16x4 la_lds_s16x4;
// bfloat16 in both libraries: parts of scores and states need its range, not half's
typedef __attribute__((ext_vector_type(2))) __bf16 lb2;
typedef __attribute__((ext_vector_type(4))) __bf16 lb4;
typedef __attribute__((ext_vector_type(8))) __bf16 lb8;

typedef __attribute__((ext_vector_type(4))) unsigned lin_raw;     // 16 bytes in flight
typedef __attribute__((ext_vector_type(2))) unsigned lin_half;
typedef __attribute__((ext_vector_type(4))) int i32x4;

struct LinOperand { const char* p; long long n, s, h; };        // address; bytes between sequences, rows, heads
struct LinRole {
  LinOperand q, k, v, o;
  int shared;                                                    // operands of HK heads: bit 0 q, bit 1 k, bit 2 v
  int reverse;                                                   // rows are visited from the last to the first
  int first_t;                                                   // `first` is read transposed
  int ws_t;                                                      // so are the segment states: they are another role's
  int o32;                                                       // o is fp32 whatever the operands are
  float s_inter, s_state;                                        // factors of Y^T q and of k v^T (their product is the scale)
  const float* first;                                            // (B, H, HD, HD) state before the first row, or null
  float* last;                                                   // (B, H, HD, HD) state behind the last row, or null
  float* ws;                                                     // states of all segments but the last ones, each H x HD x HD
};
struct LinArgs {
  LinRole r[3];
  const float* slopes;
  const int* cu;                                                 // (B + 1) row offsets, or null: B sequences of S rows
  int B, S, H, T;                                                // T: rows in all (cu), S: rows of a sequence
  int seg, np;                                                   // rows of a segment, a multiple of the chunk; segments of a sequence (no cu)
  int slots;
  int fill;                                                      // rows outside every sequence become 0 (cu)
  int rep, HK;                                                   // heads that share one head of k and v; those heads
  int roles, roles_state, split;                                 // roles of the main and of the state kernel; the axis is cut into segments
};
#define LIN_GRID_Y 32768
// Sequences of up to so many segments: a segment sums the states in front of it itself.  More: the scan kernel does (one recording of 64
// segments: 16 heads x 64 x 16 KB for each of them).  One clip of 16 segments: 21.2 us with the scan kernel, 16.1 without.
#define LIN_INLINE 16

// Rows of a chunk: two tiles of 16.  64 rows pay the state's share half as often and meet half the barriers, but take 168 registers in place
// of 128: 3 workgroups on a CU, not 4 (64 clips of 2000 rows 11 % slower, the training pair of 140-row clips 24 %).
#define LIN_C 32
template <typename T> struct LinT;
template <> struct LinT<__bf16> { static constexpr int IN = 1, V = 8; };               // parts of the operands; elements of 16 bytes
template <> struct LinT<float> { static constexpr int IN = 3, V = 4; };
#define LIN_MID 3             /* parts of scores, scaled values and states: all of 32 bits */

// x[0 .. 2 N - 1] = the sum of PARTS bf16 parts: the nearest, the nearest to what is left, and so on; two elements at a time (v_cvt_pk,
// then a shift and a mask to get the pair back: 6 instructions a pair and part)
template <int PARTS, int N> __device__ __forceinline__ void lin_split(const float* x, unsigned (&w)[PARTS][N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int k = 0; k < PARTS; ++k) {
      w[k][i] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){a, b}, lb2));
      if (k + 1 < PARTS) { a -= __builtin_bit_cast(float, w[k][i] << 16); b -= __builtin_bit_cast(float, w[k][i] & 0xffff0000u); }
    }
  }
}
// The same for a pair of tiles of 16 x 16 in the accumulators' layout (row 4 g + i, column fr), which gives the operand of 32 rows and 16 columns:
// its inner index is row 4 g + i of tile h at element 4 h + i of lane group g.  What a part leaves is x - part, a product with minus one's
// matrix: exact, and one matrix instruction in place of eight vector ones, which are what these kernels run out of.  (A part that is not
// finite spoils its column of the tiles, whose sums it would enter as well.)
struct LinMinus { lb8 of[2]; };                                  // row fr of tile h: -1 at its own element
__device__ __forceinline__ LinMinus lin_minus(int fr, int g) {
  LinMinus m;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __bf16 v = fr == 4 * g + i ? (__bf16)-1.f : (__bf16)0.f;
    m.of[0][i] = m.of[1][4 + i] = v;
    m.of[0][4 + i] = m.of[1][i] = (__bf16)0.f;
  }
  return m;
}
template <int PARTS> __device__ __forceinline__ void lin_split_tiles(f32x4 a, f32x4 b, const LinMinus& minus, lb8 (&f)[PARTS]) {
#pragma unroll
  for (int k = 0; k < PARTS; ++k) {
    const lb4 lo = __builtin_convertvector(a, lb4), hi = __builtin_convertvector(b, lb4);
    f[k] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    if (k + 1 < PARTS) {
      a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(minus.of[0], f[k], a, 0, 0, 0);
      b = __builtin_amdgcn_mfma_f32_16x16x32_bf16(minus.of[1], f[k], b, 0, 0, 0);
    }
  }
}
// c += a b over 32 of the inner index, a and b in parts; products below the last part of the longer one are left out
template <int NA, int NB> __device__ __forceinline__ f32x4 lin_mma(const lb8 (&a)[NA], const lb8 (&b)[NB], f32x4 c) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < (NA > NB ? NA : NB)) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], c, 0, 0, 0);
  return c;
}

// A tile in LDS is its parts, each LIN_C rows of HD bf16.  Piece p (16 bytes) of row r lies at p ^ swz(r): 16 rows at one piece (row reads) and
// 256 bytes of neighbouring pieces (writes) each cover the 64 banks once, the transposed reads of half pieces twice, and rows 16 apart share
// it, so that a lane needs an address per piece and immediates for the rest.  (A padded pitch leaves 40 % of the LDS cycles to conflicts: no
// pitch serves the row reads and the transposed ones.)
//
// Channel 32 kd + 8 g + 4 h + i is row 4 g + i of the state's tile 2 kd + h, so that the eight channels which a lane group g holds of a pair of
// tiles -- the inner index of Y^T q -- are one piece of a row of q.
template <typename T, int HD> struct LinTile {
  static constexpr int IN = LinT<T>::IN, PITCH = 2 * HD, PART = LIN_C * PITCH, BYTES = IN * PART;
  static __device__ __forceinline__ int swz(int r) {             // the row bits that the pitch leaves on one bank, reversed
    if (HD == 32) return (r & 4) >> 1 | (r & 8) >> 3;            // 4 rows to 256 bytes, 4 pieces to a row
    if (HD == 64) return (r & 2) << 1 | (r & 4) >> 1 | (r & 8) >> 3;
    return (r & 1) << 3 | (r & 2) << 1 | (r & 4) >> 1 | (r & 8) >> 3;
  }
  static __device__ __forceinline__ int at(int r, int u) { return r * PITCH + (((u >> 1) ^ swz(r)) << 4) + ((u & 1) << 3); }     // u: half pieces
  static __device__ __forceinline__ void put(char* tile, int r, int c, lin_raw x) {            // 16 bytes, piece c of row r
    if constexpr (IN == 1) *(lin_raw*)(tile + at(r, 2 * c)) = x;
    else {
      const f32x4 f = __builtin_bit_cast(f32x4, x);
      const float e[4] = {f[0], f[1], f[2], f[3]};
      unsigned w[IN][2];
      lin_split<IN, 2>(e, w);
#pragma unroll
      for (int k = 0; k < IN; ++k) *(lin_half*)(tile + k * PART + at(r, c)) = (lin_half){w[k][0], w[k][1]};
    }
  }
  // 8 elements of row 16 rt + fr, from half piece u0 on
  static __device__ __forceinline__ void row(const char* tile, int rt, int fr, int u0, lb8 (&f)[IN]) {
#pragma unroll
    for (int k = 0; k < IN; ++k) f[k] = *(const lb8*)(tile + k * PART + rt * 16 * PITCH + at(fr, u0));
  }
  // transposed: rows {4 g ..+3} and {16 + 4 g ..+3} of the column that is lane % 16 of the four half pieces u, u + step ...
  static __device__ __forceinline__ void col(const char* tile, int u0, int step, int lane, lb8 (&f)[IN]) {
#pragma unroll
    for (int k = 0; k < IN; ++k) {
      const char* const p = tile + k * PART + at(4 * (lane >> 4) + ((lane & 15) >> 2), u0 + step * (lane & 3));
      union { struct { s16x4 a, b; } s; lb8 v; } u;
      u.s.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((la_lds_s16x4*)p);
      u.s.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((la_lds_s16x4*)(p + 16 * PITCH));
      f[k] = u.v;
    }
  }
};
__device__ __forceinline__ int lin_channel(int t, int g, int i) { return 32 * (t >> 1) + 8 * g + 4 * (t & 1) + i; }         // of row 4 g + i of tile t
// 16 bytes of each lane from base + off to lds + 16 lane, without a register in between.  In asm, so that the compiler does not wait for them in
// front of every read from LDS: what waits is lin_wait, with the number of memory operations that are surely younger.  (m0 cannot be named as
// clobbered, and nothing else here uses it: the tests hold the compiled kernels to that, and to the number of younger operations.)
__device__ __forceinline__ void lin_dma(const char* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(lds), "v"(off), "s"(base) : "memory");
}
// the lane, read again where it is needed: paths that are rarely taken keep nothing in registers for it
__device__ __forceinline__ int lin_lane() {
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
  return l;
}
template <int N> __device__ __forceinline__ void lin_wait() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }
template <int IN> __device__ __forceinline__ float lin_value(const lb8 (&f)[IN], int i) {       // the element that the parts stand for
  float x = (float)f[0][i];
#pragma unroll
  for (int k = 1; k < IN; ++k) x += (float)f[k][i];
  return x;
}
__device__ __forceinline__ void lin_store4(float* p, const f32x4& v) { *(f32x4*)p = v; }
__device__ __forceinline__ void lin_store4(__bf16* p, const f32x4& v) { *(lb4*)p = __builtin_convertvector(v, lb4); }

// slot -> (sequence, segment).  Sequences start wherever cu says, so sequence b gets the slots floor(start / seg) + b ...: that many are
// always enough (ceil(len / seg) <= floor((start + len) / seg) - floor(start / seg) + 1), none is shared, and their number is known to
// the host without reading cu.  Offsets are clamped to [0, T]: a wrong cu gives wrong rows, never an access outside the tensors.
// States are kept without the b: a sequence leaves one for each segment but its last, which are fewer than the multiples of seg that it
// reaches, so floor(start / seg) + p is not shared either, and S / seg of them are enough however many sequences there are.
struct LinSeq { int b, p, np, begin, len, kept; };               // begin: first row, len: rows, np: segments, kept: the first one's state
__device__ __forceinline__ int lin_cu(const LinArgs& a, int b) { const int c = a.cu[b]; return c < 0 ? 0 : (c > a.T ? a.T : c); }
// the last b in [0, n) for which `is` holds, 0 if it never does: one look of the wave's 64 lanes for up to 64 sequences, two for 4096, three for
// 262144.  (A look at 64 sequences after the other: 10000 packed clips of 140 rows took six times as long as the same clips side by side.)
template <typename F> __device__ __forceinline__ int lin_last(int n, F is) {
  int lo = 0;
  for (const int lane = threadIdx.x & 63; n > 1;) {
    const int step = (n + 63) >> 6, count = __popcll(__ballot(lane * step < n && is(lo + lane * step)));
    const int at = count > 0 ? (count - 1) * step : 0;
    lo += at;
    n = n - at < step ? n - at : step;
  }
  return lo;
}
__device__ __forceinline__ bool lin_find(const LinArgs& a, int slot, LinSeq& s) {
  if (!a.cu) {
    s.np = a.np;
    s.b = a.np == 1 ? slot : slot / a.np;
    s.p = slot - s.b * a.np;
    s.begin = 0;
    s.len = a.S;
    s.kept = s.b * (a.np - 1);
    return true;
  }
  const int lo = lin_last(a.B, [&](int b) { return lin_cu(a, b) / a.seg + b <= slot; });       // the slots ascend with b
  s.b = lo;
  s.begin = lin_cu(a, lo);
  const int end = lin_cu(a, lo + 1);
  s.len = end > s.begin ? end - s.begin : 0;
  s.np = s.len > a.seg ? (s.len + a.seg - 1) / a.seg : 1;
  s.kept = s.begin / a.seg;
  s.p = slot - (s.kept + lo);
  return s.p >= 0 && s.p < s.np;
}
__device__ __forceinline__ float lin_log2(const float* slopes, int h) {
  const float l2 = -slopes[h] * 1.44269504088896341f;
  return l2 < -4096.f ? -4096.f : l2;                            // (an infinite slope: l^0 = 1, l^n = 0; NaN stays NaN)
}
__device__ __forceinline__ float lin_uniform(float v) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); }
__device__ __forceinline__ float lin_pow(float l2, int n) { return __builtin_amdgcn_exp2f(l2 * (float)n); }

// What bounds it (16 heads of 64 channels, 16-bit).  64 clips of 2000 rows, 1049 MB: 215 us, 4.87 TB/s, where a large copy reaches 5.2 -- memory.
// The backward of 192 clips of 140 rows: 0.74 us for a chunk and CU, the vector pipe busy for 65 % of it and the matrix pipe for 49 %; a chunk is
// a chain of LDS reads, matrix and vector steps of 2 us and more, and four waves to a SIMD do not hide all of it.  A recording reads k and v twice,
// and a long backward's dq, which runs forward in time, shares nothing in the L2 with dk and dv, which run backwards: 7 operand reads from
// memory instead of 4.
// Registers: 128 with 16-bit operands, four waves to a SIMD; 32-bit ones take 166, three waves (two: 90 us against 84 for the training pair
// of 2 x 2000 rows in fp32), with 128 channels two.
//
// HEADS: neighbouring heads of a workgroup (lin_wide), each with waves, scores and state of its own, side by side in the tiles' rows.
// STATE: only the segment's own state (from zero) is formed, into ws: what the segments behind it start from.
template <typename T, int HD, int HEADS, bool STATE>
__global__ __launch_bounds__(HD * HEADS * 4, LinT<T>::IN == 1 ? 4 : HD == 128 ? 2 : 3) void lin_kernel(LinArgs a) {
  typedef LinT<T> L;
  constexpr int W = HD * HEADS;                                  // channels of a row of the tiles
  typedef LinTile<T, W> Tile;
  constexpr int C = LIN_C, ND = HD / 16, NK = HD / 32, THREADS = W * 4, OP = Tile::IN == 1 ? 2 * W : 4 * W + 16;            // OP: pitch of the result's tile, bytes
  constexpr int CPH = HD / L::V, CPR = W / L::V, NU = C * CPR / THREADS;         // 16-byte pieces of a row, and of a tile for each thread
  static_assert(C * CPR == NU * THREADS, "whole pieces per thread and tile");
  static_assert(L::IN > 1 || C * OP == Tile::BYTES, "the result takes the place of the queries");
  constexpr int WAVES = HD / 16, PP = 80, PPART = C * PP;        // scores: rows of 32 bf16 at a pitch of 20 words (16 rows, 16 lanes: all banks)
  // 16-bit operands go straight to LDS, into two stages of tiles in turn; 32-bit ones are split on the way, through registers.  (Two chunks
  // ahead instead of one: 0 to 3 % slower.)
  constexpr bool DMA = L::IN == 1;
  constexpr int LOADS = STATE ? 2 : 3, STAGE = LOADS * Tile::BYTES;
  // the result's tile: with two stages, over the chunk's queries, which are done with by then (four heads of 32 channels would not fit twice
  // on a CU with one of its own)
  constexpr int RES = STATE || DMA ? 0 : C * OP;
  __shared__ __attribute__((aligned(16))) char sm[(DMA ? 2 : 1) * STAGE + RES + (STATE ? 0 : HEADS * LIN_MID * PPART)];
  const int tid = threadIdx.x, lane = tid & 63, fr = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int me = HEADS == 1 ? 0 : wave / WAVES, wi = wave - me * WAVES, n0 = wi * 16, u0 = me * (HD / 4);       // head of the workgroup, wave of the head
  char* const sP = sm + (DMA ? 2 : 1) * STAGE + RES + (STATE ? 0 : me * LIN_MID * PPART);
  // Workgroups go to the eight XCDs in turn.  What reads the same rows at the same time -- the roles of a backward, the heads that share
  // k and v -- is put eight apart: one XCD, one L2.  (Side by side, the three roles of a backward read everything from memory three times.)
  const int nr = STATE ? a.roles_state : a.roles, in = blockIdx.x >> 3, turn = blockIdx.z * LIN_GRID_Y + blockIdx.y;
  // Neighbouring heads go to neighbouring XCDs, except where two of them share a cache line (32 channels of 16 bits: 320 us one by one, 293
  // in pairs for 64 x 2000 rows of 32 heads; pairs of 64 channels: 230 against 225).
  const int unit = W * (int)sizeof(T) < 128 ? (turn >> 1) * 16 + (blockIdx.x & 7) * 2 + (turn & 1) : turn * 8 + (blockIdx.x & 7);
  const int of = nr == 1 ? in : nr == 2 ? in >> 1 : in * 21846 >> 16;         // in / nr (in < 3 * 4096)
  const int per = a.HK / HEADS, slot0 = unit / per, hk0 = (unit - slot0 * per) * HEADS, hk = hk0 + me, h0 = hk0 * a.rep + of, h = hk * a.rep + of;
  if (slot0 >= a.slots) return;
  const LinRole r = a.r[in - of * nr];                           // by value: its fields in a few wide loads, not one by one where they are used
  // the main kernel of a split axis starts with the last segments: their k and v are what the state kernel has read last
  const int slot = !STATE && a.split ? a.slots - 1 - slot0 : slot0;
  // which score tiles this wave forms: the first of three waves changes from workgroup to workgroup (a wave stays on its SIMD)
  const int mine_p = (wi + blockIdx.y) % WAVES;
  LinSeq s;
  const bool mine = lin_find(a, slot, s);
  char* const out = (char*)r.o.p + h * r.o.h;
  if constexpr (!STATE) {
    if (a.fill) {                                                // rows in front of the first and behind the last sequence
      int z0 = 0, z1 = 0;
      const int c0 = lin_cu(a, 0), cB = lin_cu(a, a.B), behind = slot - (cB / a.seg + a.B);
      if (behind >= 0) { z0 = cB + behind * a.seg; z1 = z0 + a.seg < a.T ? z0 + a.seg : a.T; }
      else if (slot <= c0 / a.seg) { z0 = slot * a.seg; z1 = z0 + a.seg < c0 ? z0 + a.seg : c0; }
      for (long long i = tid - me * (HD * 4); i < (long long)(z1 - z0) * HD; i += HD * 4) {
        char* const at = out + (z0 + i / HD) * r.o.s;
        if (r.o32) ((float*)at)[i % HD] = 0.f; else ((T*)at)[i % HD] = (T)0.f;
      }
    }
  }
  if (!mine) return;
  if (STATE && s.p == s.np - 1) return;                          // nothing starts from the last segment's state
  const int b = s.b;
  const long long sh = ((long long)b * a.H + h) * HD * HD;
  const int from = s.p * a.seg, upto = STATE || s.len - from > a.seg ? from + a.seg : s.len;     // visited positions of this segment
  const bool ends = s.p == s.np - 1;                             // this workgroup meets the sequence's last position
  const float l2 = lin_log2(a.slopes, h);
  const int off = r.reverse ? 0 : 1;                             // `first` is S_0 forward (Y = l S_0) and Y itself backwards

  // A chunk's c rows lie in a row of memory, backwards in a reverse role: each operand is a uniform address that moves by a chunk, and an
  // offset per 16-byte piece that only the last chunk changes.  Its missing rows are copies of the last one (what they hold meets a zero
  // weight).  (Forming the addresses from the row number again in every chunk, with their 64-bit products and the reads of the strides,
  // took 10 % of a chunk's time.)
  const bool rev = r.reverse;
  const int row0 = rev ? s.begin + s.len - 1 : s.begin, dir = rev ? -1 : 1;        // row of position t: row0 + dir * t
  const int low = rev ? row0 - from - (C - 1) : row0 + from;
  const long long qs = r.q.s, ks = r.k.s, vs = r.v.s, os = r.o.s, n = a.cu ? 0 : b;
  const char* bq = r.q.p + n * r.q.n + (r.shared & 1 ? hk0 : h0) * r.q.h + low * qs;
  const char* bk = r.k.p + n * r.k.n + (r.shared & 2 ? hk0 : h0) * r.k.h + low * ks;
  const char* bv = r.v.p + n * r.v.n + (r.shared & 4 ? hk0 : h0) * r.v.h + low * vs;
  char* bo = (char*)r.o.p + h0 * r.o.h + n * r.o.n + low * os;
  const long long dq = qs * (dir * C), dk = ks * (dir * C), dv = vs * (dir * C), dO = os * (dir * C);
  const bool o32 = r.o32;
  lin_raw pq[NU], pk[NU], pv[NU];                                // the next chunk's tiles, in flight during this one's math
  unsigned aq[NU], ak[NU], av[NU], ao[NU];
  auto offsets = [&](unsigned (&off)[NU], long long stride, unsigned head, int c, bool in, int tid) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int at = tid + u * THREADS, i = at / CPR < c ? at / CPR : c - 1;
      const int piece = (at % CPR) ^ (in && DMA ? Tile::swz(at / CPR) : 0);
      off[u] = (unsigned)(rev ? c - 1 - i : i) * (unsigned)stride + (HEADS == 1 ? 0 : piece / CPH * head) + piece % CPH * 16;
    }
  };
  auto offsets_in = [&](int c, int tid) __attribute__((always_inline)) {
    if constexpr (!STATE) offsets(aq, qs, (unsigned)r.q.h, c, true, tid);
    offsets(ak, ks, (unsigned)r.k.h, c, true, tid);
    offsets(av, vs, (unsigned)r.v.h, c, true, tid);
  };
  const unsigned lds = (unsigned)(size_t)(__attribute__((address_space(3))) char*)sm + wave * 1024;
  auto fetch = [&](int c, int stage) __attribute__((always_inline)) {
    if (c < C) {
      offsets_in(c, wave * 64 + lin_lane());
      if (rev) { bq += (C - c) * qs; bk += (C - c) * ks; bv += (C - c) * vs; }
    }
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      if constexpr (DMA) {
        const unsigned to = lds + stage + u * THREADS * 16;
        lin_dma(bk, ak[u], to);
        lin_dma(bv, av[u], to + Tile::BYTES);
        if constexpr (!STATE) lin_dma(bq, aq[u], to + 2 * Tile::BYTES);
      } else {
        if constexpr (!STATE) pq[u] = *(const lin_raw*)(bq + aq[u]);
        pk[u] = *(const lin_raw*)(bk + ak[u]);
        pv[u] = *(const lin_raw*)(bv + av[u]);
      }
    }
    bq += dq; bk += dk; bv += dv;
  };
  auto place = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int at = tid + u * THREADS, i = at / CPR, e = at % CPR;
      Tile::put(sm, i, e, pk[u]);
      Tile::put(sm + Tile::BYTES, i, e, pv[u]);
      if constexpr (!STATE) Tile::put(sm + 2 * Tile::BYTES, i, e, pq[u]);
    }
  };

  if constexpr (!STATE) {                                        // the first queries' weights of the second tile of keys are zeros for good
#pragma unroll
    for (int k = 0; k < LIN_MID; ++k)
      if (wi == 0) *(lin_half*)(sP + k * PPART + fr * PP + 16 * g + 8) = (lin_half){0u, 0u};
  }
  offsets_in(C, tid);
  if constexpr (!STATE) offsets(ao, os, (unsigned)r.o.h, C, false, tid);
  auto rows_at = [&](int t) __attribute__((always_inline)) { return upto - t < C ? upto - t : C; };
  if (from < upto) fetch(rows_at(from), 0);

  f32x4 S[ND];                                                   // S[t][i]: row lin_channel(t, g, i) of the state, column n0 + fr
#pragma unroll
  for (int t = 0; t < ND; ++t) S[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  if constexpr (!STATE) {
    if (r.first) {
      const float f0 = s.len ? lin_pow(l2, from + off) : 1.f;    // an empty sequence hands its state on as it is
      const float* const p = r.first + sh;
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = lin_channel(t, g, i);
          S[t][i] = f0 * (r.first_t ? p[(n0 + fr) * HD + d] : p[d * HD + n0 + fr]);
        }
    }
    // what the segments in front have left: the scanned state, or (few segments) their own states summed here
    const float ls = lin_pow(l2, a.seg);
    float f = 1.f;
    constexpr int U = HD <= 64 ? 3 : 1;                          // segments whose loads are in flight together
    for (int p0 = s.p, stop = s.np > LIN_INLINE && s.p ? s.p - 1 : 0; p0 > stop; p0 -= U) {
      f32x4 x[U][ND];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (p0 - u <= stop) break;
        const float* const w = r.ws + ((long long)(s.kept + p0 - u - 1) * a.H + h) * HD * HD;
#pragma unroll
        for (int t = 0; t < ND; ++t) {
          if (!r.ws_t) x[u][t] = *(const f32x4*)(w + ((wi * ND + t) * 64 + lane) * 4);
          else {                                                 // element (row, column) = (c, d) of the role that left it
            const int c = n0 + fr, d = lin_channel(t, g, 0), tile = 2 * (c >> 5) + (c >> 2 & 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[u][t][i] = w[(((d >> 4) * ND + tile) * 64 + (c >> 3 & 3) * 16 + (d & 15) + i) * 4 + (c & 3)];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (p0 - u <= stop) break;
#pragma unroll
        for (int t = 0; t < ND; ++t) S[t] += f * x[u][t];
        f *= ls;
      }
    }
  }

  const LinMinus minus = lin_minus(fr, g);
  // l^(i - j) scale for a query column fr and key rows 4 g + i: inside a tile, and one tile apart
  const float scale = r.s_inter * r.s_state;
  float w0[4], w1[4], wv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = fr - 4 * g - i;
    w0[i] = d < 0 ? 0.f : scale * lin_pow(l2, d);
    w1[i] = scale * lin_pow(l2, 16 + d);
    wv[i] = r.s_state * lin_pow(l2, 16 - 4 * g - i);
  }
  const float l16 = lin_uniform(lin_pow(l2, 16)), lC = lin_uniform(lin_pow(l2, C)), lrow = r.s_inter * lin_pow(l2, fr);

  // one chunk of c rows; END: the segment's last one, which may be short and may end the sequence
  auto chunk = [&](auto end, int t0, int c, int stage) __attribute__((always_inline)) {
    constexpr bool END = decltype(end)::value;
    const char* const sK = sm + stage;
    const char* const sV = sK + Tile::BYTES;
    const char* const sQ = sK + (STATE ? 0 : 2) * Tile::BYTES;
    char* const sO = sm + (DMA ? stage + 2 * Tile::BYTES : STAGE);
    if constexpr (DMA) {
      // Younger than this chunk's loads are the rows that the last chunk has stored; nothing waits for them.  (Waiting is 1 % faster where memory
      // binds and the card is full, and up to 13 % slower elsewhere: 16 x 2000 rows of 32 heads of 32 channels 85 us against 74.)
      if (END || STATE || o32 || t0 == from) lin_wait<0>();
      else lin_wait<NU>();
    } else place();
    __syncthreads();
    if constexpr (!END) fetch(rows_at(t0 + C), DMA ? STAGE - stage : 0);
    f32x4 acc[2];                                                // results of the two query tiles
    acc[0] = acc[1] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if constexpr (!STATE) {
      constexpr bool HOLD = L::IN == 1 && W <= 64;              // else read again where they are used: too many registers
      lb8 qf[2][NK][L::IN];
      auto query = [&](int ti, int kd) __attribute__((always_inline)) { Tile::row(sQ, ti, fr, u0 + 8 * kd + 2 * g, qf[ti][kd]); };
      if constexpr (HOLD)
#pragma unroll
        for (int kd = 0; kd < 2 * NK; ++kd) query(kd & 1, kd >> 1);
      // the scores of the tiles (queries, keys) = (0, 0), (1, 0), (1, 1), one wave to a tile, for all waves: in LDS, in parts
#pragma unroll
      for (int n = 0; n < 3; ++n)
        if (n % (WAVES < 3 ? WAVES : 3) == mine_p) {
          const int ti = n > 0, e = n > 1;
          f32x4 p = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kd = 0; kd < NK; ++kd) {
            lb8 kf[L::IN];
            Tile::row(sK, e, fr, u0 + 8 * kd + 2 * g, kf);
            if constexpr (!HOLD) query(ti, kd);
            p = lin_mma(kf, qf[ti][kd], p);
          }
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)                            // on the diagonal a select, not a product: a non-finite key stays behind
            x[i] = n == 1 ? p[i] * w1[i] : fr < 4 * g + i ? 0.f : p[i] * w0[i];
          unsigned w[LIN_MID][2];
          lin_split<LIN_MID, 2>(x, w);
#pragma unroll
          for (int k = 0; k < LIN_MID; ++k) *(lin_half*)(sP + k * PPART + (16 * ti + fr) * PP + 16 * g + 8 * e) = (lin_half){w[k][0], w[k][1]};
        }
#pragma unroll
      for (int kd = 0; kd < NK; ++kd) {
        lb8 y[LIN_MID];
        lin_split_tiles<LIN_MID>(S[2 * kd], S[2 * kd + 1], minus, y);
        if constexpr (!HOLD) { query(0, kd); query(1, kd); }
        acc[0] = lin_mma(y, qf[0][kd], acc[0]);
        acc[1] = lin_mma(y, qf[1][kd], acc[1]);
      }
      acc[0] *= lrow;
      acc[1] *= lrow * l16;
    }
    lb8 vf[L::IN];
    Tile::col(sV, u0 + n0 / 4, 1, lane, vf);                     // column n0 + fr
    if (!END || !ends || r.last) {
      const int e = END && ends ? c - off : C;                   // the state behind the last row itself, or as the next row sees it
      const float le = END ? lin_pow(l2, e) : lC;
#pragma unroll
      for (int t = 0; t < ND; ++t) S[t] *= le;
      f32x4 x[2];
      if (!END || e == C) {                                      // l^(C - j), j = 16 tile + 4 g + i
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[0][i] = lin_value(vf, i) * (l16 * wv[i]);
          x[1][i] = lin_value(vf, 4 + i) * wv[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = 4 * g + 16 * (i >> 2) + (i & 3);
          x[i >> 2][i & 3] = j < c ? lin_value(vf, i) * (r.s_state * lin_pow(l2, e - j)) : 0.f;     // (rows behind the end are copies of the last)
        }
      }
      lb8 p[LIN_MID];
      lin_split_tiles<LIN_MID>(x[0], x[1], minus, p);
#pragma unroll
      for (int t = 0; t < ND; ++t) {
        lb8 kf[L::IN];
        Tile::col(sK, u0 + 8 * (t >> 1) + (t & 1), 2, lane, kf); // the columns lin_channel(t, ., .)
        S[t] = lin_mma(kf, p, S[t]);
      }
    }
    if constexpr (!STATE || !DMA) __syncthreads();
    if constexpr (!STATE) {
      // A value that is not finite would meet the zero weights of the rows in front of it, and 0 * inf is NaN: such values leave the product, and
      // the rows that they reach are NaN.  (minus one's matrix, mostly zeros, shows them: a channel with one is not finite in any column.)
      const f32x4 probe = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[0], minus.of[0], (f32x4){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) bad |= !__builtin_isfinite(probe[i]);
      if (__builtin_expect(__any(bad), 0)) {
        const int lane = lin_lane(), fr = lane & 15, g = lane >> 4;
        int row = C;                                             // first row of channel n0 + fr that is not finite
#pragma unroll
        for (int i = 7; i >= 0; --i) {
          const bool ok = __builtin_isfinite((float)vf[0][i]);
          row = ok ? row : 16 * (i >> 2) + 4 * g + (i & 3);
#pragma unroll
          for (int k = 0; k < L::IN; ++k) vf[k][i] = ok ? vf[k][i] : (__bf16)0.f;
        }
        row = min(row, __builtin_amdgcn_ds_bpermute((lane ^ 16) << 2, row));
        row = min(row, __builtin_amdgcn_ds_bpermute((lane ^ 32) << 2, row));
#pragma unroll
        for (int i = 0; i < 4; ++i) {                            // (of the channel and the two rows that an accumulator holds)
          const int r0 = __builtin_amdgcn_ds_bpermute((4 * g + i) << 2, row);
          if (fr >= r0) acc[0][i] = __builtin_nanf("");
          if (16 + fr >= r0) acc[1][i] = __builtin_nanf("");
        }
      }
#pragma unroll
      for (int ti = 0; ti < 2; ++ti) {
        lb8 p[LIN_MID];
#pragma unroll
        for (int k = 0; k < LIN_MID; ++k) p[k] = *(const lb8*)(sP + k * PPART + (16 * ti + fr) * PP + 16 * g);
        acc[ti] = lin_mma(vf, p, acc[ti]);
      }
    }
    if constexpr (!STATE) {
#pragma unroll
      for (int ti = 0; ti < 2; ++ti) {
        if (!o32) lin_store4((T*)(sO + (Tile::IN == 1 ? 16 * ti * OP + Tile::at(fr, u0 + n0 / 4 + g) : (16 * ti + fr) * OP + (n0 + 4 * g) * 4)), acc[ti]);
        else {
          const int t = t0 + 16 * ti + fr;
          if (t < upto) *(f32x4*)(out + n * r.o.n + (long long)(row0 + dir * t) * os + (n0 + 4 * g) * 4) = acc[ti];
        }
      }
    }
    if constexpr (!STATE) {
      __syncthreads();
      // whole rows, 16 bytes a lane: 8-byte pieces straight from the accumulators cost 10 % of the launch.  Past the L2, which the
      // operands need: 2 to 5 % on every long case.
      if (!o32) {
        if (END && c < C) {
          offsets(ao, os, (unsigned)r.o.h, c, false, wave * 64 + lin_lane());
          if (rev) bo += (C - c) * os;
        }
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const int at = tid + u * THREADS;
          if (!END || at / CPR < c) __builtin_nontemporal_store(*(const lin_raw*)(sO + (Tile::IN == 1 ? Tile::at(at / CPR, 2 * (at % CPR)) : (at / CPR) * OP + (at % CPR) * 16)), (lin_raw*)(bo + ao[u]));
        }
        bo += dO;
      }
    }
  };
  int t0 = from, stage = 0;
  for (; t0 + C < upto; t0 += C) {
    chunk(std::false_type{}, t0, C, stage);
    if constexpr (DMA) stage = STAGE - stage;
  }
  if (t0 < upto) chunk(std::true_type{}, t0, upto - t0, stage);
  if constexpr (STATE) {
    f32x4* const w = (f32x4*)(r.ws + ((long long)(s.kept + s.p) * a.H + h) * HD * HD) + wi * ND * 64 + lane;
#pragma unroll
    for (int t = 0; t < ND; ++t) w[t * 64] = S[t];
  } else if (ends && r.last) {
    float* const p = r.last + sh;
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) p[lin_channel(t, g, i) * HD + n0 + fr] = S[t][i];
  }
}

// The state of segment p := the state in front of segment p + 1: carried through the sequence's segments in order, one thread to an
// element (any order of them: the waves' register image), eight loads in flight.  The part of `first` is added by the kernel that starts
// from it.  A group of workgroups takes a sequence; of packed ones each that has something to scan, which reaches a multiple of LIN_INLINE
// segments of rows: the group of the first such row looks for the sequence around it, so there are few groups however many sequences there
// are.  (Short ones alone pay the launch, 4.8 us: their lengths are on the device.)
__global__ __launch_bounds__(256) void lin_scan_kernel(LinArgs a, int HH) {
  const int per = a.H * HH / 256, group = blockIdx.x / per;
  const int i = (blockIdx.x - group * per) * 256 + threadIdx.x, h = i / HH;    // element of (H, HD, HD); HD * HD % 256 == 0
  int b = group, begin = 0, len = a.S;
  if (a.cu) {
    const int row = group * LIN_INLINE * a.seg;
    b = lin_last(a.B, [&](int b) { return lin_cu(a, b) <= row; });
    begin = lin_cu(a, b);
    const int end = lin_cu(a, b + 1);
    if (row < begin || row >= end || row - begin >= LIN_INLINE * a.seg) return;
    len = end - begin;
  }
  const int np = len > a.seg ? (len + a.seg - 1) / a.seg : 1;
  if (np <= LIN_INLINE) return;
  const float f = lin_pow(lin_log2(a.slopes, h), a.seg);
  const long long step = (long long)a.H * HH;
  float* const w = a.r[blockIdx.y].ws + (long long)(a.cu ? begin / a.seg : b * (np - 1)) * step + i;
  float carry = 0.f;
  int p = 0;
  for (; p + 8 < np; p += 8) {                                   // (the last segment has no state of its own)
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = w[(p + u) * step];
#pragma unroll
    for (int u = 0; u < 8; ++u) w[(p + u) * step] = carry = carry * f + x[u];
  }
  for (; p < np - 1; ++p) w[p * step] = carry = carry * f + w[p * step];
}

// the gradients of a shared k / v head: the sum over its heads, of fp32 rows (T, H, HD) -> rows of HK heads
template <typename T>
__global__ __launch_bounds__(256) void lin_join_kernel(const float* dk32, const float* dv32, T* dk, T* dv, long long kn, long long ks, long long kh,
                                                       long long vn, long long vs, long long vh, const int* cu, int B, int S, int T_, int H, int rep, int HD, int fill) {
  const int HK = H / rep, per = HK * HD / 4;
  const long long rows = cu ? T_ : (long long)B * S, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * per) return;
  const long long row = i / per;
  const int e = (int)(i - row * per) * 4, hk = e / HD, d = e - hk * HD;
  const long long n = cu ? 0 : row / S, t = cu ? row : row - n * S;
  f32x4 a = {0.f, 0.f, 0.f, 0.f}, c = a;
  const bool in = !cu || (t >= cu[0] && t < cu[B]);
  if (!in && !fill) return;
  if (in) {
    const float* p = dk32 + (row * H + hk * rep) * HD + d;
    const float* q = dv32 + (row * H + hk * rep) * HD + d;
    for (int u = 0; u < rep; ++u) { a += *(const f32x4*)(p + u * HD); c += *(const f32x4*)(q + u * HD); }
  }
  lin_store4(dk + n * kn + t * ks + hk * kh + d, a);
  lin_store4(dv + n * vn + t * vs + hk * vh + d, c);
}

// One token of each of N streams, the state updated in place: state once in, once out, everything else is negligible (HBM, or latency
// where N H is small: 256 streams of 16 heads of 64 channels 22.5 us, 6.1 TB/s of state, part of it out of the Infinity Cache; one stream
// 3.2 us).  A thread holds four neighbouring columns of HD * HD / 1024 rows of the state.
// slots[n] names the state of row n.  Rows that name the same slot are successive tokens of one stream, in row order: the workgroup of
// the first of them takes them all (the others find an earlier row and leave), so there is no race and no order left open.  A slot
// outside [0, n_slots) leaves every state alone and gives a row of zeros (padding rows of a captured graph).
// So a workgroup reads all slots, which grows with the square of N.  It therefore takes N / LIN_STEP_SLOTS heads of its row one after the other: fewer
// workgroups for each row, and never so few that the card is not full (16 heads of 64 channels: 40000 rows 4.3 ms against 12.3 with one head to
// a workgroup, 10000 1.08 against 1.45, 3.9 and 0.97 without slots; 700 rows 56 us, 66 with a limit of 128).
#define LIN_STEP_SLOTS 512
struct LinStep {
  const void* q; const void* k; const void* v; void* o;
  long long qn, qh, kn, kh, vn, vh, on, oh;
  const float* slopes; float* state; const int* slots;
  int n_slots, N, H, rep, heads;                                 // heads: of a workgroup
  float scale;
};
template <typename T, int HD>
__global__ __launch_bounds__(256) void lin_step_kernel(LinStep a) {
  constexpr int LPR = HD / 4, RPP = 256 / LPR, NP = HD / RPP;    // lanes of a row, rows of a pass, passes
  __shared__ f32x4 part[4 * LPR];
  const int groups = (a.H + a.heads - 1) / a.heads, n = blockIdx.x / groups, tid = threadIdx.x;
  const int h0 = (blockIdx.x - n * groups) * a.heads, h1 = h0 + a.heads < a.H ? h0 + a.heads : a.H;
  const int c = (tid % LPR) * 4, r0 = tid / LPR;
  const int slot = a.slots ? a.slots[n] : n;
  T* const out = (T*)a.o;
  if (slot < 0 || slot >= a.n_slots) {
    for (int h = h0; h < h1; ++h)
      if (tid < LPR) Vec4<T>::store(out + n * a.on + h * a.oh + c, (f32x4){0.f, 0.f, 0.f, 0.f});
    return;
  }
  float* const st = a.state + (long long)slot * a.H * HD * HD + r0 * HD + c;
  f32x4 S[NP];
#pragma unroll
  for (int p = 0; p < NP; ++p) S[p] = *(const f32x4*)(st + ((long long)h0 * HD + p * RPP) * HD);
  bool more = false;
  if (a.slots) {
    bool before = false;
    auto look = [&](int m, int other) __attribute__((always_inline)) { before |= m < n && other == slot; more |= m > n && other == slot; };
    const int lead = (int)(-(uintptr_t)a.slots >> 2 & 3), quads = a.N > lead ? (a.N - lead) >> 2 : 0;        // 16 bytes a lane between the ends
    for (int i = tid; i < quads; i += 256) {
      const int m = lead + 4 * i;
      const i32x4 x = *(const i32x4*)(a.slots + m);
#pragma unroll
      for (int u = 0; u < 4; ++u) look(m + u, x[u]);
    }
    if (tid < 8) {
      const int m = tid < 4 ? tid : lead + 4 * quads + tid - 4;
      if (tid < 4 ? m < lead && m < a.N : m < a.N) look(m, a.slots[m]);
    }
    if (__syncthreads_or(before)) return;
    more = __syncthreads_or(more);
  }
  for (int h = h0; h < h1; ++h) {
    const int hk = h / a.rep;
    const float l = lin_pow(lin_log2(a.slopes, h), 1);
    for (int m = n; m < a.N; ++m) {
      if (m > n && a.slots[m] != slot) continue;
      const T* const q = (const T*)a.q + m * a.qn + h * a.qh;
      const T* const k = (const T*)a.k + m * a.kn + hk * a.kh;
      const f32x4 v = Vec4<T>::load((const T*)a.v + m * a.vn + hk * a.vh + c);
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int d = r0 + p * RPP;
        S[p] = S[p] * l + v * ldf(k + d);
        o += S[p] * ldf(q + d);
      }
#pragma unroll
      for (int x = LPR; x < 64; x <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], x, 64);
      if ((tid & 63) < LPR) part[(tid >> 6) * LPR + (tid & 63)] = o;
      __syncthreads();
      if (tid < LPR) Vec4<T>::store(out + m * a.on + h * a.oh + c, (part[tid] + part[LPR + tid] + part[2 * LPR + tid] + part[3 * LPR + tid]) * a.scale);
      if (!more && h + 1 == h1) break;
      __syncthreads();
      if (!more) break;
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      *(f32x4*)(st + ((long long)h * HD + p * RPP) * HD) = S[p];
      if (h + 1 < h1) S[p] = *(const f32x4*)(st + ((long long)(h + 1) * HD + p * RPP) * HD);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------ host side
#define LIN_WGS 1024          /* workgroups that fill the card: four on each of 256 CUs */

// Rows of a segment.  Enough (sequence, head) pairs: one segment each, k and v read once.  Fewer: the axis is cut until LIN_WGS
// workgroups run, which costs a second pass over k and v; not below 4 HD rows, where writing and reading the states (HD * HD * 4 bytes)
// costs as much as it gives (4 clips of 2000 rows, 16 heads: 26 us at 256 rows, 33 at 128), except that fewer than a workgroup for
// each compute unit are worse still: then 2 HD (one such clip: 19.0 us at 256 rows, 16.1 at 128, 23.4 at 64).
static int lin_seg(int B, long long rows, int S, int H, int HD, bool packed, int C) {
  const long long all = packed ? rows : S;
  if (!packed && (long long)B * H >= LIN_WGS / 2) return all > 0 ? cdiv(all, C) * C : C;
  long long seg = (rows * H + LIN_WGS - 1) / LIN_WGS;
  const int least = rows * H < 256LL * 4 * HD ? 2 * HD : 4 * HD;
  if (seg < least) seg = least;
  if (seg > all) seg = all;
  return seg < C ? C : cdiv(seg, C) * C;
}
struct LinPlan { int C, seg, slots; bool split; size_t states; };
static bool lin_plan(int dtype, int B, int S, int H, int HD, bool packed, LinPlan& p) {
  p.C = LIN_C;
  const long long rows = packed ? S : (long long)B * S;
  if (rows >= (1LL << 30)) return false;
  p.seg = lin_seg(B, rows, S, H, HD, packed, p.C);
  const long long slots = packed ? (long long)S / p.seg + B + 1 : (long long)B * (S > p.seg ? (S + p.seg - 1) / p.seg : 1);
  if ((slots + 16) * H * 3 >= (1LL << 31) || (long long)H * HD * HD >= (1LL << 28)) return false;      // (a launch has at most 2^32 threads in x)
  p.slots = (int)slots;
  p.split = S > p.seg;
  const long long kept = packed ? S / p.seg : slots - B;         // every segment's but the last one's of a sequence
  p.states = p.split ? (size_t)kept * H * HD * HD * sizeof(float) : 0;
  return true;
}
static bool lin_shape_ok(int B, int S, int H, int HK, int HD) {
  return B >= 0 && S >= 0 && H > 0 && HK > 0 && H % HK == 0 && H / HK <= 1024 && (HD == 32 || HD == 64 || HD == 128);
}
// The state that a call leaves may not lie in the one that it reads: every segment of a sequence starts from the latter.
static bool lin_states_apart(const float* in, const float* out, int B, int H, int HD) {
  const uintptr_t a = (uintptr_t)in, b = (uintptr_t)out, n = (uintptr_t)B * H * HD * HD * sizeof(float);
  return !in || !out || a + n <= b || b + n <= a;
}
static bool lin_tensor_ok(const void* p, const long long* st, int es) {
  return p && !((uintptr_t)p & 15) && !((st[0] * es) & 15) && !((st[1] * es) & 15) && !((st[2] * es) & 15) && st[1] >= 0 &&
         st[1] * es < (1 << 26);                                 // (offsets inside a chunk are 32 bits)
}

static dim3 lin_grid(const LinArgs& a, int roles, int heads) {
  const unsigned groups = (unsigned)(((long long)a.slots * (a.HK / heads) + 15) / 16 * 2);       // (of eight, in pairs)
  return dim3(8 * roles * a.rep, groups < LIN_GRID_Y ? groups : LIN_GRID_Y, (groups + LIN_GRID_Y - 1) / LIN_GRID_Y);
}
template <typename T, int HD, int HEADS>
static void lin_launch_heads(const LinArgs& a, const LinPlan& p, hipStream_t stream) {
  const dim3 block(HD * HEADS * 4);
  if (p.split) {
    hipLaunchKernelGGL((lin_kernel<T, HD, HEADS, true>), lin_grid(a, a.roles_state, HEADS), block, 0, stream, a);
    if ((a.S + a.seg - 1) / a.seg > LIN_INLINE) {
      const unsigned groups = a.cu ? a.S / (LIN_INLINE * a.seg) + 1 : a.B, per = a.H * (HD * HD / 256);          // (B H < LIN_WGS / 2 where sequences are cut)
      hipLaunchKernelGGL(lin_scan_kernel, dim3(per * groups, a.roles_state), dim3(256), 0, stream, a, HD * HD);
    }
  }
  hipLaunchKernelGGL((lin_kernel<T, HD, HEADS, false>), lin_grid(a, a.roles, HEADS), block, 0, stream, a);
}
// A head's 16-bit row is 64 or 128 bytes.  Four or two neighbouring heads to a workgroup read and write 256 at a time, which is worth more to
// the memory than the larger workgroup costs, except where the card is not full of them or the kernel waits for its own steps:
//   64 channels   64 x 2000 rows 221 us against 245, one recording 305 against 341; but 48 x 2000 rows (384 workgroups) 182 against 170, one clip
//                 19.5 against 16.9, the training pair of 140-row clips 194 against 181 (its forward alone 58 against 57)
//   32 channels   64 x 2000 rows 216 us against 296, the training pairs of 140-row clips 169 against 193 and of 4 x 11025 rows 352 against 463;
//                 of 2 x 2000 rows 53 against 48
static bool lin_wide(const LinArgs& a, int HD, int heads) {
  if (heads == 1 || a.HK % heads || a.rep > 1 || (HD > 32 && a.roles > 1)) return false;
  if ((long long)a.slots * a.HK / heads < (HD > 32 ? LIN_WGS / 2 : LIN_WGS / 4)) return false;
  for (int i = 0; i < a.roles; ++i)
    for (const LinOperand* o : {&a.r[i].q, &a.r[i].k, &a.r[i].v, &a.r[i].o})
      if (o->h < 0 || o->h >= (1 << 26)) return false;           // (offsets inside a chunk are 32 bits)
  return true;
}
template <typename T, int HD>
static void lin_launch_hd(const LinArgs& a, const LinPlan& p, hipStream_t stream) {
  constexpr int HEADS = LinT<T>::IN == 1 ? 128 / HD : 1;
  if (lin_wide(a, HD, HEADS)) lin_launch_heads<T, HD, HEADS>(a, p, stream);
  else lin_launch_heads<T, HD, 1>(a, p, stream);
}
template <typename T>
static void lin_launch_t(const LinArgs& a, const LinPlan& p, int HD, hipStream_t stream) {
  if (HD == 32) lin_launch_hd<T, 32>(a, p, stream);
  else if (HD == 64) lin_launch_hd<T, 64>(a, p, stream);
  else lin_launch_hd<T, 128>(a, p, stream);
}
static void lin_launch(int dtype, const LinArgs& a, const LinPlan& p, int HD, hipStream_t stream) {
  if (dtype == A2V_F32) lin_launch_t<float>(a, p, HD, stream);
  else lin_launch_t<__bf16>(a, p, HD, stream);
}
static int lin_dtype(int dtype) {
  if (dtype != A2V_F32 && dtype != A2V_BF16) return A2V_ERR_DTYPE;
#ifdef A2V_ELT_F16
  if (dtype == A2V_BF16) return A2V_ERR_UNSUPPORTED;             // (a half operand would be two bfloat16 parts: not built)
#endif
  return A2V_OK;
}

static LinOperand lin_op(const void* p, const long long* st, int es) { return LinOperand{(const char*)p, st[0] * es, st[1] * es, st[2] * es}; }
static void lin_args(LinArgs& a, const LinPlan& p, const float* slopes, const int* cu, int B, int S, int H, int HK, int zero_outside) {
  a.slopes = slopes; a.cu = cu; a.B = B; a.S = S; a.H = H; a.T = S; a.seg = p.seg; a.slots = p.slots; a.fill = cu && zero_outside;
  a.np = S > p.seg ? (S + p.seg - 1) / p.seg : 1;
  a.HK = HK; a.rep = H / HK; a.split = p.split;
}

extern "C" size_t a2v_linear_attention_workspace(int dtype, int backward, int packed, int B, int S, int H, int HK, int HD) {
  LinPlan p;
  if (!lin_shape_ok(B, S, H, HK, HD) || !lin_plan(dtype, B, S, H, HD, packed != 0, p)) return 0;
  const size_t rows = packed ? (size_t)S : (size_t)B * S;
  return (backward ? 2 : 1) * p.states + (backward && H != HK ? 2 * rows * H * HD * sizeof(float) : 0);
}

extern "C" int a2v_linear_attention_fwd(int dtype, const void* q, const void* k, const void* v, void* out, const long long* strides,
                                        const float* slopes, const float* state, float* state_out, const int* cu_seqlens, int B, int S, int H,
                                        int HK, int HD, float scale, int zero_outside, void* ws, size_t ws_bytes, hipStream_t stream) {
  if (int e = lin_dtype(dtype)) return e;
  LinPlan p;
  if (!strides || !slopes || !lin_shape_ok(B, S, H, HK, HD) || !lin_plan(dtype, B, S, H, HD, cu_seqlens != nullptr, p)) return A2V_ERR_ARG;
  if (B == 0) return A2V_OK;                                     // no sequence: nothing is read or written
  const int es = dtype == A2V_F32 ? 4 : 2;
  if (S > 0 && !(lin_tensor_ok(q, strides, es) && lin_tensor_ok(k, strides + 3, es) && lin_tensor_ok(v, strides + 6, es) && lin_tensor_ok(out, strides + 9, es)))
    return A2V_ERR_ARG;
  if (!lin_states_apart(state, state_out, B, H, HD)) return A2V_ERR_ARG;
  if (p.states > ws_bytes || (p.states && (!ws || ((uintptr_t)ws & 15)))) return A2V_ERR_ARG;
  LinArgs a;
  lin_args(a, p, slopes, cu_seqlens, B, S, H, HK, zero_outside);
  const int kv = H != HK ? 6 : 0;
  a.r[0] = LinRole{lin_op(q, strides, es), lin_op(k, strides + 3, es), lin_op(v, strides + 6, es), lin_op(out, strides + 9, es),
                   kv, 0, 0, 0, 0, scale, 1.f, state, state_out, (float*)ws};
  a.r[1] = a.r[2] = a.r[0];
  a.roles = a.roles_state = 1;
  lin_launch(dtype, a, p, HD, stream);
  A2V_CHECK_LAUNCH();
  return A2V_OK;
}

extern "C" int a2v_linear_attention_bwd(int dtype, const void* q, const void* k, const void* v, const void* d_out, void* dq, void* dk, void* dv,
                                        const long long* strides, const float* slopes, const float* state, const float* d_state_out, float* d_state,
                                        const int* cu_seqlens, int B, int S, int H, int HK, int HD, float scale, int zero_outside, void* ws,
                                        size_t ws_bytes, hipStream_t stream) {
  if (int e = lin_dtype(dtype)) return e;
  LinPlan p;
  if (!strides || !slopes || !lin_shape_ok(B, S, H, HK, HD) || !lin_plan(dtype, B, S, H, HD, cu_seqlens != nullptr, p)) return A2V_ERR_ARG;
  if (B == 0) return A2V_OK;                                     // no sequence: nothing is read or written
  const int es = dtype == A2V_F32 ? 4 : 2, rep = H / HK;
  const void* const t[7] = {q, k, v, d_out, dq, dk, dv};
  if (S > 0)
    for (int i = 0; i < 7; ++i)
      if (!lin_tensor_ok(t[i], strides + 3 * i, es)) return A2V_ERR_ARG;
  if (!lin_states_apart(state, d_state, B, H, HD) || !lin_states_apart(d_state_out, d_state, B, H, HD)) return A2V_ERR_ARG;
  if (rep > 1 && (cu_seqlens ? 1LL : (long long)B) * S * HK * HD / 4 >= (1LL << 32)) return A2V_ERR_ARG;    // (threads of the join)
  const size_t need = a2v_linear_attention_workspace(dtype, 1, cu_seqlens != nullptr, B, S, H, HK, HD);
  if (need > ws_bytes || (need && (!ws || ((uintptr_t)ws & 15)))) return A2V_ERR_ARG;
  char* w = (char*)ws;
  const size_t rows = cu_seqlens ? (size_t)S : (size_t)B * S;
  float* const dk32 = (float*)(w + 2 * p.states);
  float* const dv32 = dk32 + rows * H * HD;
  LinArgs a;
  lin_args(a, p, slopes, cu_seqlens, B, S, H, HK, zero_outside);
  LinOperand o[7];
  for (int i = 0; i < 7; ++i) o[i] = lin_op(t[i], strides + 3 * i, es);
  LinOperand &Q = o[0], &K = o[1], &V = o[2], &D = o[3], gk = o[5], gv = o[6];
  if (rep > 1) {                                                 // fp32 rows of every head, summed behind the kernel
    const long long one[3] = {(long long)S * H * HD, (long long)H * HD, HD};
    gk = lin_op(dk32, one, 4);
    gv = lin_op(dv32, one, 4);
  }
  const int o32 = rep > 1, kv = rep > 1;
  a.r[0] = LinRole{D, V, K, o[4], 6 * kv, 0, 1, 0, 0, scale, 1.f, state, nullptr, (float*)w};
  a.r[1] = LinRole{K, Q, D, gv, kv, 1, 0, 0, o32, 1.f, scale, d_state_out, d_state, (float*)(w + p.states)};
  a.r[2] = LinRole{V, D, Q, gk, kv, 1, 1, 1, o32, 1.f, scale, d_state_out, nullptr, (float*)(w + p.states)};
  a.roles = 3; a.roles_state = 2;                                // dk's segment states are the transposes of dv's
  lin_launch(dtype, a, p, HD, stream);
  if (rep > 1 && rows) {
    const dim3 grid((unsigned)cdiv((long)(rows * HK * HD / 4), 256));
    if (dtype == A2V_F32)
      hipLaunchKernelGGL(lin_join_kernel<float>, grid, dim3(256), 0, stream, dk32, dv32, (float*)dk, (float*)dv, strides[15], strides[16], strides[17], strides[18], strides[19], strides[20],
                         cu_seqlens, B, S, S, H, rep, HD, a.fill);
    else
      hipLaunchKernelGGL(lin_join_kernel<__bf16>, grid, dim3(256), 0, stream, dk32, dv32, (__bf16*)dk, (__bf16*)dv, strides[15], strides[16], strides[17], strides[18], strides[19], strides[20],
                         cu_seqlens, B, S, S, H, rep, HD, a.fill);
  }
  A2V_CHECK_LAUNCH();
  return A2V_OK;
}

extern "C" int a2v_linear_attention_step(int dtype, const void* q, const void* k, const void* v, void* out, const long long* strides,
                                         const float* slopes, float* state, const int* slots, int n_slots, int N, int H, int HK, int HD, float scale,
                                         hipStream_t stream) {
  if (dtype != A2V_F32 && dtype != A2V_BF16) return A2V_ERR_DTYPE;
  if (!strides || !slopes || !state || ((uintptr_t)state & 15) || ((uintptr_t)slots & 3) || N < 0 || H <= 0 || HK <= 0 || H % HK || (HD != 32 && HD != 64 && HD != 128) ||
      n_slots < (slots ? 0 : N) || (long long)N * H >= (1LL << 24))              // (2^32 threads)
    return A2V_ERR_ARG;
  if (N == 0) return A2V_OK;
  const int es = dtype == A2V_F32 ? 4 : 2;
  const void* const t[4] = {q, k, v, out};
  for (int i = 0; i < 4; ++i)
    if (!t[i] || ((uintptr_t)t[i] & (4 * es - 1)) || strides[2 * i] % 4 || strides[2 * i + 1] % 4) return A2V_ERR_ARG;
  const int heads = !slots || N < LIN_STEP_SLOTS ? 1 : N / LIN_STEP_SLOTS < H ? N / LIN_STEP_SLOTS : H;
  const LinStep a{q, k, v, out, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], strides[6], strides[7],
                  slopes, state, slots, n_slots, N, H, H / HK, heads, scale};
  const dim3 grid((unsigned)(N * ((H + heads - 1) / heads))), block(256);
#define LIN_STEP(T_, HD_) hipLaunchKernelGGL((lin_step_kernel<T_, HD_>), grid, block, 0, stream, a)
  if (dtype == A2V_F32) { if (HD == 32) LIN_STEP(float, 32); else if (HD == 64) LIN_STEP(float, 64); else LIN_STEP(float, 128); }
  else { if (HD == 32) LIN_STEP(bf16, 32); else if (HD == 64) LIN_STEP(bf16, 64); else LIN_STEP(bf16, 128); }
#undef LIN_STEP
  A2V_CHECK_LAUNCH();
  return A2V_OK;
}
