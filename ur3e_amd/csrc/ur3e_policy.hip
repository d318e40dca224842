/* Operators of a policy with memory (include/ur3e_policy.h): attention with a decaying state and keyed
 * dropout.
 *
 * Attention over a sequence (k_attn_walk).  One wave owns one (sequence, head, slab of value channels) and walks
 * its tokens in chunks with the state S [dk][slab] in registers.  With chunk-local positions i, j, n tokens in the
 * chunk and the state S that enters it:
 *     o_i  = scale gamma^(i+1) S^T q_i + sum_{j <= i} scale gamma^(i-j) (q_i . k_j) v_j
 *     S'   = gamma^n S + sum_j gamma^(n-1-j) k_j v_j^T
 * All four products are matrix instructions on tiles of 16 x 16, and the register layouts chain without a trip
 * through LDS: the scores are formed transposed (P^T = K Q^T), which leaves them as the right operand of O^T = V^T P^T,
 * and the accumulators of S are the left operand of S^T Q^T as they stand.  That leaves two forms of a token tile,
 * "rows" (a lane holds one token's channels) and "columns" (a lane holds a few channels of four tokens), both read
 * straight from memory.  Products do not care in which order the contracted index runs, so the channels are dealt
 * to the tiles by what reads well (Place), the same way in either form.
 *
 * A chunk is a tile of 16 tokens, for 16-bit types of up to 64 key channels two of them.  Sequences that are too few to fill
 * the card are split along time (splits_of): the sums of the splits first (STATE), joined into the state that enters
 * each (k_attn_join), then all outputs at once.
 *
 * float is multiplied as float.  16-bit elements are multiplied as bfloat16 (a half is the exact sum of two), with
 * the float operands, scores and state, in leading parts (split4).
 *
 * Gradients are the same walk with other operands.  G_t = scale q_t do_t^T + a_{t+1} G_{t+1} is the state
 * of the reversed sequence, so
 *     dq = walk(do, v, k) on S^T,  dk = reversed walk(v, do, q) on G^T,  dv = reversed walk(k, q, do) on G.
 *
 * What bounds it (MI355X, a copy of 4 GiB runs at 4.75 TB/s): 2,048 sequences x 512 tokens x 4 heads of 64 channels take,
 * forward, 482 us in bfloat16 (4.5 TB/s) and 931 us in float (4.6), bound by memory, and 487 us in half (4.4).  Their
 * gradients take 1.14 ms in bfloat16 (3.3 TB/s of the tensors; the walks run against each other in time and read some of
 * them twice), 2.47 ms in float, whose matrix instructions alone take 1.64, and 1.28 ms in half.  With 128 channels the
 * vector instructions around the products bound it: 1.54 ms in bfloat16 (2.8 TB/s).  Short calls are chains of latencies: a
 * chunk of 16 float tokens takes a lone wave 3.3 us, 2.1 us in a slab of 16 value channels. */
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "../../include/ur3e_batch.h"
#include "../../include/ur3e_policy.h"

int ur3e_internal_fail(int code, const char* msg);

#define PL_CHK(x)                                                                       \
  do {                                                                                  \
    hipError_t _e = (x);                                                                \
    if (_e != hipSuccess) return ur3e_internal_fail(UR3E_EHIP, hipGetErrorString(_e));  \
  } while (0)

typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u6 __attribute__((ext_vector_type(6)));

struct Bf16 { unsigned short x; };
typedef _Float16 F16;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(Bf16 x) { return __builtin_bit_cast(float, (unsigned)x.x << 16); }
__device__ __forceinline__ float to_f(F16 x) { return (float)x; }
/* round to nearest even, once, where a result leaves the kernel */
template <class T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ F16 from_f<F16>(float x) { return (F16)x; }
template <> __device__ __forceinline__ Bf16 from_f<Bf16>(float x) {
  return __builtin_bit_cast(Bf16, (__bf16)x);
}

/* two bfloat16 in a dword */
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, b2{(__bf16)lo, (__bf16)hi});
}

/* eight consecutive elements, on a boundary of 16 bytes (WHOLE) or of an element */
template <class T, bool WHOLE> struct Eight {
  struct alignas(WHOLE ? 16 : sizeof(T)) Pack { T e[8]; };
  static __device__ __forceinline__ void load(const T* p, float* x) {
    const Pack v = *reinterpret_cast<const Pack*>(p);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = to_f(v.e[i]);
  }
  static __device__ __forceinline__ void store(T* p, const float* x) {
    Pack v;
#pragma unroll
    for (int i = 0; i < 8; i++) v.e[i] = from_f<T>(x[i]);
    *reinterpret_cast<Pack*>(p) = v;
  }
};

/* One walk: which tensors play q, k and v, and which way time runs.  `kdim` channels are contracted in the
   scores (and are the state's rows), `vdim` are read out. */
struct Tok {
  const void* p;
  long long sb, st, sh;
  int hdiv = 1; /* head = query head / hdiv */
};
struct Walk {
  Tok q, k, v, o;           /* o.p is written */
  const float* s_in;        /* [b][h][dk * dv] or null */
  float* s_out;             /* or null (always where state_t) */
  float* ws;                /* nsplit > 1: [b][h][split][room(kdim * vdim)], split s holds the state that enters it, */
  float* wf;                /* and [b][h][split], what split s - 1 multiplies the state by, or DROPS */
  int state_t;              /* a [dk][dv] state is this walk's transposed: kdim = dv */
  int reversed;
  int out_f32;              /* out is float whatever the token type (gradients that are summed over heads) */
  float in_scale, p_scale, w_scale; /* on the read-out of the entering state, on the scores, on k in the state */
};
/* In the place of a factor: an episode starts, and what was in front is dropped whatever it holds.  (A factor of 0 is a product
   that left float's range.  0 times a NaN or an infinity stays a NaN.) */
#define DROPS -1.0f
/* floats between the states of two splits: on boundaries of 16 bytes */
__host__ __device__ __forceinline__ int room(int elems) { return (elems + 3) / 4 * 4; }
struct WalkArgs {
  Walk w[3];
  int nw; /* walks of this launch, all of the same tile shape */
  int b, t, h, kdim, vdim, slabs, nsplit, split_len;
  /* Channels that the last slab takes from the one in front of it: one load of a lane where fewer are left for it, so that no
     channel is read and written by two slabs (they may round it differently: a chunk with a value that is not finite
     is taken token by token). */
  int lent;
  int near; /* consecutive workgroups that share a sequence's tensors */
  int chunk; /* 16, or 1 where tokens lie too far apart for 30-bit offsets inside a chunk */
  const float* log_decay;
  const unsigned char* starts;
  long long starts_sb, starts_st;
  const int* lengths;
};

/* a value that all lanes share, in a scalar register */
__device__ __forceinline__ float uniform(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}
/* gamma^n with gamma^0 = 1 whatever gamma (log_decay = -inf is a head without memory) */
__device__ __forceinline__ float pw(float l, int n) { return n == 0 ? 1.0f : expf((float)n * l); }

__device__ __forceinline__ f4 mfma4(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

/* Every tile is read and written through buffer instructions, whose bounds check stands in for a branch: a lane
   without an element carries an offset past the 2^30 bytes of the resource, reads 0 and writes nothing, so
   the loads of a chunk issue back to back.  FAR_T (no such token) and FAR_D (no such channel) stay past the
   limit when both are added. */
#define FAR_T 0x80000000u
#define FAR_D 0x40000000u
typedef __amdgpu_buffer_rsrc_t Rsrc;
/* The value, opaque from here on: what a rare branch derives from it is computed there, not kept in registers
   through the loop around the branch. */
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
__device__ __forceinline__ unsigned at(unsigned off, bool there, unsigned far) { return there ? off : far; }
__device__ __forceinline__ Rsrc rsrc_of(const void* p, bool there = true) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, there ? (int)FAR_D : 0, 0x00027000);
}

/* N consecutive elements as dwords, on any boundary of an element */
template <class T, int N> struct Raw {
  static constexpr int B = N * (int)sizeof(T), D = (B + 3) / 4;
  unsigned d[D];
  __device__ __forceinline__ void load(Rsrc r, unsigned off) {
    if constexpr (B == 2) d[0] = __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
    else if constexpr (B == 4) d[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
    else if constexpr (B == 8) {
      const u2 x = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0);
      d[0] = x.x; d[1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < B / 16; i++) {
        const u4 x = __builtin_amdgcn_raw_buffer_load_b128(r, off + 16 * i, 0, 0);
        d[4 * i] = x.x; d[4 * i + 1] = x.y; d[4 * i + 2] = x.z; d[4 * i + 3] = x.w;
      }
    }
  }
  /* zeros for the first n elements (n <= 0: none) */
  __device__ __forceinline__ void clear(int n) {
#pragma unroll
    for (int i = 0; i < D; i++) {
      if constexpr (sizeof(T) == 4) d[i] = i < n ? 0 : d[i];
      else d[i] &= 2 * i + 1 < n ? 0u : 2 * i < n ? 0xffff0000u : 0xffffffffu;
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, d[i]);
    else return to_f(__builtin_bit_cast(T, (unsigned short)(d[i / 2] >> (16 * (i & 1)))));
  }
};
template <class T, int N> __device__ __forceinline__ void store_n(Rsrc r, unsigned off, const float* x) {
  constexpr int B = N * (int)sizeof(T);
  unsigned d[(B + 3) / 4] = {};
#pragma unroll
  for (int i = 0; i < N; i += sizeof(T) == 4 ? 1 : 2) {
    if constexpr (sizeof(T) == 4) d[i] = __builtin_bit_cast(unsigned, x[i]);
    else if constexpr (N == 1) d[0] = __builtin_bit_cast(unsigned short, from_f<T>(x[0]));
    else if constexpr (__is_same(T, Bf16)) d[i / 2] = pack_bf16(x[i], x[i + 1]); /* one conversion for both */
    else {
      struct Two { T a, b; };
      d[i / 2] = __builtin_bit_cast(unsigned, Two{from_f<T>(x[i]), from_f<T>(x[i + 1])});
    }
  }
  if constexpr (B == 2) __builtin_amdgcn_raw_buffer_store_b16((unsigned short)d[0], r, off, 0, 0);
  else if constexpr (B == 4) __builtin_amdgcn_raw_buffer_store_b32(d[0], r, off, 0, 0);
  else if constexpr (B == 8) __builtin_amdgcn_raw_buffer_store_b64(u2{d[0], d[1]}, r, off, 0, 0);
  else {
#pragma unroll
    for (int i = 0; i < B / 16; i++)
      __builtin_amdgcn_raw_buffer_store_b128(u4{d[4 * i], d[4 * i + 1], d[4 * i + 2], d[4 * i + 3]}, r, off + 16 * i, 0, 0);
  }
}

/* The largest magnitude met so far, as the bits of an unsigned integer (two 16-bit ones), and whether it is an
   infinity or a NaN. */
template <class T> struct Peak {
  typedef unsigned short us2 __attribute__((ext_vector_type(2)));
  unsigned m = 0;
  __device__ __forceinline__ void add(unsigned d) {
    if constexpr (sizeof(T) == 4) {
      const unsigned x = d & 0x7fffffffu;
      m = x > m ? x : m;
    } else {
      const unsigned x = d & 0x7fff7fffu;
      m = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(us2, x), __builtin_bit_cast(us2, m)));
    }
  }
  __device__ __forceinline__ bool not_finite() const {
    if constexpr (sizeof(T) == 4) return m >= 0x7f800000u;
    constexpr unsigned inf = __is_same(T, Bf16) ? 0x7f80u : 0x7c00u;
    return (m >= inf << 16) | ((m & 0xffffu) >= inf);
  }
};

/* bfloat16 fragments of 16-bit tensors, two elements to a dword.  A 32-bit operand enters the matrix instructions
   as the sum of its leading parts of 8 bits each: two (error 2^-17) for scores and state, whose results are rounded
   to 2^-9 or 2^-11 on the way out, three (2^-25) for what is added to a state that leaves.  (Outputs of the plain form and of
   these kernels are the same 0.0017 from the definition in bfloat16, one rounding, and 1.1e-4 from each other, where sums that
   differ by 2^-17 round to either side.) */
/* the K = 32 shape throughout, half empty where four elements are all there is: a K = 16 instruction right behind
   a K = 32 one on the same accumulators read them before the first had written (the compiler had put one wait
   state between the two; measured at one tile, where nothing else stands between them) */
__device__ __forceinline__ f4 mfma32(u4 a, u4 b, f4 c) {
  typedef __bf16 b8 __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}
/* the same of half elements, as they are in memory */
template <class T> __device__ __forceinline__ f4 mfma_raw(u4 a, u4 b, f4 c) {
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  if constexpr (__is_same(T, F16)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else return mfma32(a, b, c);
}
/* The packed leading parts of four elements that lie as an accumulator does (rows 4 g + e of column idx); x
   becomes the rest, x - hi, a product with the negative unit matrix: one instruction of the matrix pipe
   in place of eight of the vector pipe, which is the busier one.  Exact: every sum has one product.  An infinity
   or a NaN spreads to the rest of its column, whose elements all feed the same result. */
__device__ __forceinline__ u2 split4(f4& x, u6 minus_one) {
  const u2 hi = {pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
  x = mfma32(__builtin_shufflevector(minus_one, minus_one, 0, 1, 2, 3), u4{hi.x, hi.y, 0, 0}, x);
  return hi;
}
/* Two at once, packed next to each other: the unit matrix stands in the half of the contraction that is the tile's, so
   nothing is padded with zeros (which would be moves: the operands are whole quads of registers). */
__device__ __forceinline__ u4 split4x2(f4& x, f4& y, u6 minus_one) {
  const u4 hi = {pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
  x = mfma32(__builtin_shufflevector(minus_one, minus_one, 0, 1, 2, 3), hi, x);
  y = mfma32(__builtin_shufflevector(minus_one, minus_one, 2, 3, 4, 5), hi, y);
  return hi;
}
__device__ __forceinline__ u4 pack4x2(f4 x, f4 y) {
  return u4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
}
__device__ __forceinline__ u4 both(u2 x, u2 y) { return u4{x.x, x.y, y.x, y.y}; }
__device__ __forceinline__ u2 pack4(f4 x) { return u2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])}; }

/* Which channels position 4 g + e of N tiles stands for: N consecutive ones from `of` on.  Groups e lie so that the
   four lanes of a token read 64 consecutive bytes of its row with each load (C groups of a lane at once, NC channels,
   up to 16 bytes): half the cache lines a load of 32 bytes a lane would touch.
   The lanes' NC channels number NC (4 (e / C) + g) on; where dim ends inside them they are taken from dim - NC on
   instead, so that no load leaves its row.  The channels that come twice then are harmless as values (the
   same results are stored twice); as keys they are zeros (`own` tells which), and so are their rows of the state. */
template <class T, int N> struct Place {
  static constexpr int U = N * (int)sizeof(T), C = U >= 16 ? 1 : U >= 4 ? 16 / U : 4, R = 4 / C, NC = N * C;
  static __device__ __forceinline__ int first(int g, int e) { return NC * (e / C * 4 + g); }
  static __device__ __forceinline__ bool there(int g, int e, int dim) { return first(g, e) < dim; }
  /* (rows of less than NC are copied into wider ones) */
  static __device__ __forceinline__ int of(int g, int e, int dim, int low = 0) {
    const int f = first(g, e), last = dim - NC < f ? dim - NC : f;
    return (last > low ? last : low) + e % C * N;
  }
};
/* the row form of a token: channels of(g, 0 .. 3) + 0 .. N - 1 */
template <class T, int N> struct Row {
  typedef Place<T, N> P;
  Raw<T, N * P::C> x[P::R];
  __device__ __forceinline__ void load(Rsrc r, const unsigned (&off)[P::R]) {
#pragma unroll
    for (int i = 0; i < P::R; i++) x[i].load(r, off[i]);
  }
  __device__ __forceinline__ float get(int e, int mt) const { return x[e / P::C].get(e % P::C * N + mt); }
};
/* (From the packed registers.  Taken from the chunk element by element, at one tile of keys, the compiler widened loads
   past the rows and kept the chunk in memory: 17.5 us a call, with this 4.7.) */
__device__ __forceinline__ f4 four_halves(u2 x) {
  typedef _Float16 h4 __attribute__((ext_vector_type(4)));
  return __builtin_convertvector(__builtin_bit_cast(h4, x), f4);
}
/* elements i of x and j of y as two halves */
template <class X> __device__ __forceinline__ unsigned halves(const X& x, int i, const X& y, int j) {
  if (&x == &y && i + 1 == j && i % 2 == 0) return x.d[i / 2];
  const unsigned sel = (i & 1 ? 0x0302u : 0x0100u) | (j & 1 ? 0x07060000u : 0x05040000u);
  return __builtin_amdgcn_perm(y.d[j / 2], x.d[i / 2], sel);
}
/* the four tokens of tile nt in the column form */
template <class T, int VT> __device__ __forceinline__ u2 pack_col(const Raw<T, VT> (&x)[4], int nt) {
  return u2{halves(x[0], nt, x[1], nt), halves(x[2], nt, x[3], nt)};
}
/* the row form by tiles: e = 0 .. 3 of tile mt, as the rows of an accumulator lie */
template <class T, int KT> __device__ __forceinline__ void pack_row(const Row<T, KT>& r, u2 (&y)[KT]) {
  constexpr int C = Place<T, KT>::C;
#pragma unroll
  for (int mt = 0; mt < KT; mt++)
    y[mt] = u2{halves(r.x[0], mt, r.x[1 / C], 1 % C * KT + mt), halves(r.x[2 / C], 2 % C * KT + mt, r.x[3 / C], 3 % C * KT + mt)};
}

/* KT, VT: tiles of 16 key channels and of 16 value channels per wave; H: tiles of 16 tokens per chunk.  STATE: only the
   state at the end of each split (from zero), for sequences that several waves share.  FINE (16-bit types): a state
   leaves as floats and is summed to their precision, from keys in three parts; where it only feeds 16-bit outputs,
   from keys in two (of the products of two parts of a half, that of the two rests, 2^-18, is left out then where it
   is not free). */
template <class T, int KT, int VT, bool STATE, int H, bool FINE>
__global__ __launch_bounds__(256, 2) void k_attn_walk(WalkArgs a) {
  constexpr int ES = (int)sizeof(T), C = 16 * H;
  constexpr bool TWO = __is_same(T, F16); /* an element is two bfloat16 parts */
  static_assert(H == 1 || ES == 2, "two tiles of tokens: 16-bit types only");
  const int lane = threadIdx.x & 63, idx = lane & 15, g = lane >> 4;
  /* Workgroups go round the 8 XCDs in turn; the `near` of them that share a sequence's tensors and states stay on
     one, behind its L2.  The wave's task is in scalar registers, and with it every address base and loop bound. */
  const unsigned slot = blockIdx.x >> 3, group = (slot / a.near * 8 + (blockIdx.x & 7)) * a.near + slot % a.near;
  const unsigned task = group * (blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nsp = STATE ? a.nsplit - 1 : a.nsplit;
  unsigned r = task;
  const int slab = (int)(r % a.slabs); r /= a.slabs;
  const int wi = (int)(r % a.nw); r /= a.nw;
  const int split = (int)(r % nsp); r /= nsp;
  const int h = (int)(r % a.h); r /= a.h;
  if (r >= (unsigned)a.b) return;
  const int b = (int)r;
  const Walk w = a.w[wi];
  const int kdim = a.kdim, vdim = a.vdim, chunk = a.chunk, nsplit = a.nsplit;
  const long long starts_st = a.starts_st;
  typedef Place<T, KT> PK;
  typedef Place<T, VT> PV;
  /* first channel of this slab, channels from there on */
  const int v0 = slab * 16 * VT - (slab == a.slabs - 1 ? a.lent : 0);
  const int vleft = slab == a.slabs - 2 ? 16 * VT - a.lent : vdim - v0;
  const float l = a.log_decay[h];
  int len = a.t;
  if (a.lengths) {
    len = a.lengths[b];
    len = len < 0 ? 0 : len > a.t ? a.t : len;
  }
  const int lo = split * a.split_len, end = lo + a.split_len < a.t ? lo + a.split_len : a.t;
  const int hi = end < len ? end : len;
  const bool rev = w.reversed;
  const char* q = (const char*)w.q.p + ES * (b * w.q.sb + (h / w.q.hdiv) * w.q.sh);
  const char* k = (const char*)w.k.p + ES * (b * w.k.sb + (h / w.k.hdiv) * w.k.sh);
  const char* v = (const char*)w.v.p + ES * (b * w.v.sb + (h / w.v.hdiv) * w.v.sh);
  const int os = w.out_f32 ? 4 : ES;
  char* out = (char*)const_cast<void*>(w.o.p) + os * (b * w.o.sb + (h / w.o.hdiv) * w.o.sh);
  const long long qst = ES * w.q.st, kst = ES * w.k.st, vst = ES * w.v.st, ost = os * w.o.st;
  const unsigned char* starts = a.starts ? a.starts + b * a.starts_sb : nullptr;

  /* byte offsets of a lane's channels and tokens, in the row form and in the column form, for tiles of n: the lowest
     token of the tile is the base */
  unsigned qrow[PK::R], krow[PK::R], kcol[4], vcol[4];
  auto place = [&](int n) {
    const int idx = fresh(lane & 15), g = fresh(lane >> 4), gi = idx >> 2, ei = idx & 3;
    const unsigned back = n - 1 - idx, rel = rev ? back : idx;
    const unsigned kidx = at(PK::of(gi, ei, kdim) * ES, PK::there(gi, ei, kdim), FAR_D);
    const unsigned vidx = at((v0 + PV::of(gi, ei, vleft, -v0)) * ES, PV::there(gi, ei, vleft), FAR_D);
#pragma unroll
    for (int i = 0; i < PK::R; i++) {
      const unsigned kd = at(PK::of(g, i * PK::C, kdim) * ES, PK::there(g, i * PK::C, kdim), FAR_D);
      qrow[i] = at(rel * (unsigned)qst, idx < n, FAR_T) + kd;
      krow[i] = at(rel * (unsigned)kst, idx < n, FAR_T) + kd;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int j = 4 * g + e;
      const unsigned backj = n - 1 - j, rc = rev ? backj : j;
      kcol[e] = at(rc * (unsigned)kst, j < n, FAR_T) + kidx;
      vcol[e] = at(rc * (unsigned)vst, j < n, FAR_T) + vidx;
    }
  };
  /* o[e][nt]: channel of(g, e) + nt of this lane's token */
  auto put = [&](Rsrc ro, unsigned rel, bool there, const float (&o)[4][VT]) {
    const unsigned orow = at(rel * (unsigned)ost, there, FAR_T);
    int wide = w.out_f32;
    asm volatile("" : "+s"(wide)); /* (tested here: as a condition kept through the loop it was spilled) */
    if (wide) {
#pragma unroll
      for (int e = 0; e < 4; e++)
        store_n<float, VT>(ro, orow + at(4 * (v0 + PV::of(g, e, vleft, -v0)), PV::there(g, e, vleft), FAR_D), o[e]);
    } else {
#pragma unroll
      for (int i = 0; i < PV::R; i++) {
        float x[PV::NC];
#pragma unroll
        for (int j = 0; j < PV::NC; j++) x[j] = o[i * PV::C + j / VT][j % VT];
        store_n<T, PV::NC>(ro, orow + at((v0 + PV::of(g, i * PV::C, vleft, -v0)) * ES, PV::there(g, i * PV::C, vleft), FAR_D), x);
      }
    }
  };

  /* padding: zeros, in forward order whatever the walk */
  if (!STATE) {
    const float zero[4][VT] = {};
    const int tile = chunk < 16 ? chunk : 16;
    for (int t = len > lo ? len : lo; t < end; t += tile) {
      const int n = end - t < tile ? end - t : tile;
      put(rsrc_of(out + t * ost), idx, idx < n, zero);
    }
  }

  const long long bh = (long long)b * a.h + h;
  const long long elems = (long long)kdim * vdim;
  f4 S[KT][VT];
  const float* s_in = STATE ? nullptr : nsplit > 1 ? w.ws + (bh * nsplit + split) * room((int)elems)
                                                     : w.s_in ? w.s_in + bh * elems : nullptr;
  /* S[mt][nt][e]: key channel of(g, e) + mt, value channel of this lane's column + nt */
  const int vcolumn = v0 + PV::of(idx >> 2, idx & 3, vleft);
  const bool vthere = PV::there(idx >> 2, idx & 3, vleft) & (vcolumn < vdim);
  const unsigned srow = 4 * (w.state_t ? 1 : vdim), scol = 4 * (w.state_t ? kdim : 1);
  auto own = [&](int e, int mt) {
    const int d = PK::of(g, e, kdim) + mt;
    return (d >= PK::first(g, e)) & (d < kdim);
  };
  if (s_in) {
    const Rsrc rs = rsrc_of(s_in);
    if (!w.state_t) {
#pragma unroll
      for (int mt = 0; mt < KT; mt++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          Raw<float, VT> x;
          x.load(rs, at((PK::of(g, e, kdim) + mt) * srow, own(e, mt), FAR_T) + at(vcolumn * scol, vthere, FAR_D));
#pragma unroll
          for (int nt = 0; nt < VT; nt++) S[mt][nt][e] = x.get(nt);
        }
    } else {
#pragma unroll
      for (int nt = 0; nt < VT; nt++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          Raw<float, KT> x;
          x.load(rs, at(PK::of(g, e, kdim) * srow, PK::there(g, e, kdim) & (PK::of(g, e, kdim) < kdim), FAR_T) + at((vcolumn + nt) * scol, vthere, FAR_D));
#pragma unroll
          for (int mt = 0; mt < KT; mt++) S[mt][nt][e] = x.get(mt);
        }
      if (kdim % PK::NC) {
#pragma unroll
        for (int mt = 0; mt < KT; mt++)
#pragma unroll
          for (int e = 0; e < 4; e++)
#pragma unroll
            for (int nt = 0; nt < VT; nt++) S[mt][nt][e] = own(e, mt) ? S[mt][nt][e] : 0.0f;
      }
    }
  } else {
#pragma unroll
    for (int mt = 0; mt < KT; mt++)
#pragma unroll
      for (int nt = 0; nt < VT; nt++) S[mt][nt] = f4{0, 0, 0, 0};
  }

  const int e0 = rev ? 0 : 1; /* the entering state has decayed by one step at position 0, or by none yet */
  float dm[H][4], wk[4]; /* dm[x]: from a key to a query x tiles behind it; wk: from a key of the last tile to the end */
#pragma unroll
  for (int f = 0; f < H; f++) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int d = 16 * f + idx - (4 * g + e);
      dm[f][e] = d >= 0 ? w.p_scale * pw(l, d) : 0.0f;
    }
  }
  const float fi = w.in_scale * pw(l, idx + e0), g16 = uniform(pw(l, 16));
  const unsigned unit = idx >> 2 != g ? 0u : idx & 1 ? 0xbf800000u : 0xbf80u;
  /* this lane's part of the negative unit matrix, zeros, and the same again: its registers serve either half */
  u6 minus_one = {idx & 2 ? 0u : unit, idx & 2 ? unit : 0u, 0, 0, idx & 2 ? 0u : unit, idx & 2 ? unit : 0u};
  asm volatile("" : "+v"(minus_one));
  float gn = 1.0f;

  float through = 1.0f; /* STATE: what the split multiplies an entering state by, or DROPS */
  int single = 0;       /* tokens left to take one by one */
  int placed = 0, scaled = 0; /* the chunk sizes that the offsets and the factors stand for */
  int p = lo, n = 0;
  /* whether anything reads the state behind the chunk */
  const bool kept = STATE || (split == nsplit - 1 && w.s_out);
  auto carried = [&](int n) { return kept || p + n < hi; };
  /* the lowest token of tile f of the chunk */
  auto low_of = [&](int n, int f) -> long long {
    const int n0 = n < 16 ? n : 16;
    return rev ? len - p - n0 - 16 * f : p + 16 * f;
  };
  struct Chunk {
    Row<T, KT> kr[H], qr[H];
    Raw<T, KT> kc[H][4];
    Raw<T, VT> vc[H][4];
    unsigned start;
  };
  /* The keys' column form is the state's, which is done last: where registers are short it is read behind the
     scores, from the cache lines that the row form brought. */
  constexpr bool LATE = H == 2;
  auto load_columns = [&](Chunk& c, Rsrc rk, int f) {
    if (STATE || carried(n)) {
#pragma unroll
      for (int e = 0; e < 4; e++) c.kc[f][e].load(rk, kcol[e]);
    }
  };
  const int twice = kdim > PK::NC && kdim % PK::NC ? PK::NC - kdim % PK::NC : 0;
  auto clear_columns = [&](Chunk& c) {
    const int gi = fresh(idx >> 2), ei = idx & 3;
    const int n = ei / PK::C * 4 + gi == kdim / PK::NC ? twice - ei % PK::C * KT : 0;
#pragma unroll
    for (int f = 0; f < H; f++)
#pragma unroll
      for (int e = 0; e < 4; e++) c.kc[f][e].clear(n);
  };
  auto load = [&](Chunk& c, int p, int n) {
    const int n0 = n < 16 ? n : 16;
    if (n0 != placed) {
      placed = n0;
      place(n0);
    }
    {
      /* position x of a reversed walk is token len - 1 - x, behind the start that token len - x may carry */
      const Rsrc rs = rsrc_of(starts + (rev ? len - p - n + 1 : p) * starts_st, starts != nullptr);
      const int i = lane & (C - 1);
      const bool there = (i < n) & ((p + i != 0) | !rev);
      const unsigned back = n - 1 - i, rel = rev ? back : i;
      c.start = __builtin_amdgcn_raw_buffer_load_b8(rs, at(rel * (unsigned)starts_st, there, FAR_T), 0, 0);
    }
#pragma unroll
    for (int f = 0; f < H; f++) {
      const bool there = 16 * f < n; /* the tile behind is whole or missing */
      const long long low = low_of(n, f);
      const Rsrc rk = rsrc_of(k + low * kst, there), rv = rsrc_of(v + low * vst, there), rq = rsrc_of(q + low * qst, there);
#pragma unroll
      for (int e = 0; e < 4; e++) c.vc[f][e].load(rv, vcol[e]);
      if (!STATE) {
        c.kr[f].load(rk, krow);
        c.qr[f].load(rq, qrow);
      }
      if (STATE || !LATE) load_columns(c, rk, f);
    }
  };
  /* one chunk; false: it holds a value that is not finite and has to be taken token by token */
  auto work = [&](Chunk& c) {
    if (n != scaled) {
      scaled = n;
      gn = uniform(pw(l, n));
      const int n0 = n > 16 ? 16 : n, j0 = fresh(4 * g);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int j = j0 + e;
        wk[e] = j < n0 ? w.w_scale * pw(l, n0 - 1 - j + (1 - e0)) : 0.0f;
      }
    }
    /* a value that is not finite must not meet the zeros of the mask (0 * inf): its chunk is taken token by
       token, where every product belongs to the token */
    Peak<T> peak;
#pragma unroll
    for (int f = 0; f < H; f++)
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int i = 0; i < Raw<T, VT>::D; i++) peak.add(c.vc[f][e].d[i]);
    if (n > 1 && __any(peak.not_finite())) return false;

    /* key channels that come twice */
    if (twice) {
      const int g = fresh(lane >> 4);
      if constexpr (!STATE) {
#pragma unroll
        for (int i = 0; i < PK::R; i++)
          if (i == kdim / PK::NC / 4)
#pragma unroll
            for (int f = 0; f < H; f++) c.kr[f].x[i].clear(g == kdim / PK::NC % 4 ? twice : 0);
      }
      if (!LATE || STATE) clear_columns(c);
    }

    /* bit i: an episode starts between positions i - 1 and i.  Most chunks have none, and skip what a start cuts. */
    const unsigned brk = (unsigned)__ballot(c.start != 0) & (unsigned)((1ull << C) - 1);
    const bool cut = brk != 0;
    auto upto = [&](int f) { return (2u << (16 * f + fresh(idx))) - 1u; }; /* breaks at or in front of a query */
    /* the scores of query tile fq with key tile fk: decayed, later keys masked (pt[e]: query idx, key 4 g + e) */
    auto scores = [&](f4& pt, int fq, int fk) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float x = pt[e] * dm[fq - fk][e];
        /* the sign of the distance as a mask of bits, not a select: a select by VCC takes six times an AND here */
        const int later = (idx - 4 * g - e) >> 31;
        pt[e] = fq != fk ? x : __builtin_bit_cast(float, __builtin_bit_cast(int, x) & ~later);
      }
    };
    /* a start between key and query, or in front of the query: no score, nothing from the entering state */
    auto cut_scores = [&](f4& pt, int fq, int fk) {
#pragma unroll
      for (int e = 0; e < 4; e++) pt[e] = (brk & upto(fq) & ~((2u << (16 * fk + fresh(4 * g) + e)) - 1u)) == 0 ? pt[e] : 0.0f;
    };
    auto cut_entering = [&](f4& x, int f) {
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = (brk & upto(f)) == 0 ? x[e] : 0.0f;
    };
    auto decay = [&] {
      if (cut) {
#pragma unroll
        for (int mt = 0; mt < KT; mt++)
#pragma unroll
          for (int nt = 0; nt < VT; nt++) S[mt][nt] = f4{0, 0, 0, 0};
        /* keys in front of the last start do not enter the state */
#pragma unroll
        for (int f = 0; f < H; f++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int j = 16 * f + fresh(4 * g) + e;
            const bool ok = (brk & ~((2u << j) - 1u)) == 0;
#pragma unroll
            for (int i = 0; i < Raw<T, KT>::D; i++) c.kc[f][e].d[i] = ok ? c.kc[f][e].d[i] : 0;
          }
      }
#pragma unroll
      for (int mt = 0; mt < KT; mt++)
#pragma unroll
        for (int nt = 0; nt < VT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) S[mt][nt][e] *= gn;
    };
    const float ahead = H == 2 && n > 16 ? g16 : 1.0f; /* tile 0, where another one follows */
    auto key = [&](int f, int mt, int e) { /* as it enters the state */
      return c.kc[f][e].get(mt) * (f == H - 1 ? wk[e] : wk[e] * ahead);
    };
    auto put_tile = [&](int f, const float (&o)[4][VT]) {
      const int n0 = n < 16 ? n : 16;
      put(rsrc_of(out + low_of(n, f) * ost, 16 * f < n), rev ? n0 - 1 - idx : idx, idx < n0, o);
    };
    if constexpr (ES == 2) {
      u2 vq[H][VT], vr[H][VT]; /* leading part (the element itself where it is bfloat16) and rest */
      auto values = [&] {
#pragma unroll
        for (int f = 0; f < H; f++)
#pragma unroll
          for (int nt = 0; nt < VT; nt++) {
            if constexpr (TWO) {
              f4 x;
#pragma unroll
              for (int e = 0; e < 4; e++) x[e] = c.vc[f][e].get(nt);
              vq[f][nt] = split4(x, minus_one);
              vr[f][nt] = pack4(x);
            } else vq[f][nt] = pack_col<T, VT>(c.vc[f], nt);
          }
      };
      if (STATE || !TWO) values();
      if (!STATE) {
        u2 kq[H][KT], qq[H][KT];
#pragma unroll
        for (int f = 0; f < H; f++) {
          pack_row<T, KT>(c.kr[f], kq[f]);
          pack_row<T, KT>(c.qr[f], qq[f]);
        }
        /* Instructions that add to the same accumulators stand apart by those of the other tiles. */
        f4 pt[H][H]; /* [query tile][key tile] */
#pragma unroll
        for (int i = 0; i < (KT + 1) / 2; i++)
#pragma unroll
          for (int fq = 0; fq < H; fq++)
#pragma unroll
            for (int fk = 0; fk <= fq; fk++) {
              const auto &x = kq[fk], &y = qq[fq];
              const f4 z = i ? pt[fq][fk] : f4{0, 0, 0, 0};
              if constexpr (KT == 1) pt[fq][fk] = mfma_raw<T>(u4{x[0].x, x[0].y, 0, 0}, u4{y[0].x, y[0].y, 0, 0}, z);
              else
                pt[fq][fk] = mfma_raw<T>(u4{x[2 * i].x, x[2 * i].y, x[2 * i + 1].x, x[2 * i + 1].y},
                                    u4{y[2 * i].x, y[2 * i].y, y[2 * i + 1].x, y[2 * i + 1].y}, z);
            }
        f4 x[H][VT];
#pragma unroll
        for (int i = 0; i < (KT + 1) / 2; i++) {
          constexpr int STEP = KT > 1;
          const int m0 = 2 * i, m1 = 2 * i + STEP;
          u4 qh[H], ql[H]; /* queries: leading part and rest */
#pragma unroll
          for (int f = 0; f < H; f++) {
            if constexpr (TWO) {
              f4 y = four_halves(qq[f][m0]), z = four_halves(qq[f][m1]);
              qh[f] = split4x2(y, z, minus_one);
              ql[f] = pack4x2(y, z);
            } else qh[f] = both(qq[f][m0], qq[f][m1]);
          }
          u4 lo; /* of the tile in front, whose products wait for this one's: they add to the same accumulators */
#pragma unroll
          for (int nt = 0; nt <= VT; nt++) {
            u4 next;
            if (nt < VT) {
              f4 r0 = S[m0][nt], r1 = S[m1][nt];
              if constexpr (KT == 1) r1 = f4{0, 0, 0, 0};
              const u4 hi = split4x2(r0, r1, minus_one);
#pragma unroll
              for (int f = 0; f < H; f++) {
                x[f][nt] = mfma32(hi, qh[f], i ? x[f][nt] : f4{0, 0, 0, 0});
                if constexpr (TWO) x[f][nt] = mfma32(hi, ql[f], x[f][nt]);
              }
              next = pack4x2(r0, r1);
            }
            if (nt > 0) {
#pragma unroll
              for (int f = 0; f < H; f++) x[f][nt - 1] = mfma32(lo, qh[f], x[f][nt - 1]);
            }
            lo = next;
          }
        }
#pragma unroll
        for (int f = 0; f < H; f++) {
#pragma unroll
          for (int nt = 0; nt < VT; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[f][nt][e] *= f ? fi * g16 : fi;
#pragma unroll
          for (int fk = 0; fk <= f; fk++) scores(pt[f][fk], f, fk);
        }
        if constexpr (LATE) {
#pragma unroll
          for (int f = 0; f < H; f++) load_columns(c, rsrc_of(k + low_of(n, f) * kst, 16 * f < n), f);
          if (twice) clear_columns(c);
        }
        if (cut) {
#pragma unroll
          for (int f = 0; f < H; f++) {
#pragma unroll
            for (int nt = 0; nt < VT; nt++) cut_entering(x[f][nt], f);
#pragma unroll
            for (int fk = 0; fk <= f; fk++) cut_scores(pt[f][fk], f, fk);
          }
        }
        if (TWO) values(); /* (where registers are not needed for queries and scores any more) */
        /* leading parts and rests of the scores */
        u2 ph, pl;
        u4 ph1 = {}, pl1 = {};
        ph = split4(pt[0][0], minus_one);
        pl = pack4(pt[0][0]);
        if constexpr (H == 2) {
          ph1 = split4x2(pt[1][0], pt[1][1], minus_one);
          pl1 = pack4x2(pt[1][0], pt[1][1]);
        }
#pragma unroll
        for (int nt = 0; nt < VT; nt++) {
          x[0][nt] = mfma32(both(vq[0][nt], vq[0][nt]), both(ph, pl), x[0][nt]);
          if constexpr (H == 2) x[1][nt] = mfma32(both(vq[0][nt], vq[1][nt]), ph1, x[1][nt]);
        }
        if constexpr (H == 2) {
#pragma unroll
          for (int nt = 0; nt < VT; nt++) x[1][nt] = mfma32(both(vq[0][nt], vq[1][nt]), pl1, x[1][nt]);
        }
        if constexpr (TWO) {
#pragma unroll
          for (int nt = 0; nt < VT; nt++) {
            x[0][nt] = mfma32(both(vr[0][nt], vr[0][nt]), both(ph, pl), x[0][nt]);
            if constexpr (H == 2) x[1][nt] = mfma32(both(vr[0][nt], vr[1][nt]), ph1, x[1][nt]);
          }
        }
#pragma unroll
        for (int f = 0; f < H; f++) {
          float o[4][VT];
#pragma unroll
          for (int nt = 0; nt < VT; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[e][nt] = x[f][nt][e];
          put_tile(f, o);
        }
      }
      if (!carried(n)) return true;
      decay();
#pragma unroll
      for (int mt = 0; mt < KT; mt++) {
        f4 kx[H];
#pragma unroll
        for (int f = 0; f < H; f++)
#pragma unroll
          for (int e = 0; e < 4; e++) kx[f][e] = key(f, mt, e);
        if constexpr (H == 2) {
          const u4 kh = split4x2(kx[0], kx[1], minus_one);
          u4 km;
          if constexpr (FINE) km = split4x2(kx[0], kx[1], minus_one);
          else km = pack4x2(kx[0], kx[1]);
#pragma unroll
          for (int nt = 0; nt < VT; nt++) S[mt][nt] = mfma32(kh, both(vq[0][nt], vq[1][nt]), S[mt][nt]);
#pragma unroll
          for (int nt = 0; nt < VT; nt++) S[mt][nt] = mfma32(km, both(vq[0][nt], vq[1][nt]), S[mt][nt]);
          if constexpr (FINE) {
            const u4 kl = pack4x2(kx[0], kx[1]);
#pragma unroll
            for (int nt = 0; nt < VT; nt++) S[mt][nt] = mfma32(kl, both(vq[0][nt], vq[1][nt]), S[mt][nt]);
          }
          if constexpr (TWO) {
#pragma unroll
            for (int nt = 0; nt < VT; nt++) S[mt][nt] = mfma32(kh, both(vr[0][nt], vr[1][nt]), S[mt][nt]);
            if constexpr (FINE) {
#pragma unroll
              for (int nt = 0; nt < VT; nt++) S[mt][nt] = mfma32(km, both(vr[0][nt], vr[1][nt]), S[mt][nt]);
            }
          }
        } else {
          const u2 kh = split4(kx[0], minus_one);
          u2 km;
          if constexpr (FINE) km = split4(kx[0], minus_one);
          else km = pack4(kx[0]);
#pragma unroll
          for (int nt = 0; nt < VT; nt++) S[mt][nt] = mfma32(both(kh, km), both(vq[0][nt], vq[0][nt]), S[mt][nt]);
          if constexpr (TWO) {
#pragma unroll
            for (int nt = 0; nt < VT; nt++) S[mt][nt] = mfma32(both(kh, km), both(vr[0][nt], vr[0][nt]), S[mt][nt]);
          }
          if constexpr (FINE) {
            const u2 kl = pack4(kx[0]);
#pragma unroll
            for (int nt = 0; nt < VT; nt++) S[mt][nt] = mfma32(both(kl, u2{0, 0}), both(vq[0][nt], vq[0][nt]), S[mt][nt]);
          }
        }
      }
    } else {
      if (!STATE) {
        f4 part[4] = {};
#pragma unroll
        for (int mt = 0; mt < KT; mt++)
#pragma unroll
          for (int e = 0; e < 4; e++) part[e] = mfma4(c.kr[0].get(e, mt), c.qr[0].get(e, mt), part[e]);
        f4 x[VT];
#pragma unroll
        for (int nt = 0; nt < VT; nt++) x[nt] = f4{0, 0, 0, 0};
#pragma unroll
        for (int mt = 0; mt < KT; mt++)
#pragma unroll
          for (int e = 0; e < 4; e++)
#pragma unroll
            for (int nt = 0; nt < VT; nt++) x[nt] = mfma4(S[mt][nt][e], c.qr[0].get(e, mt), x[nt]);
        f4 pt;
#pragma unroll
        for (int e = 0; e < 4; e++) pt[e] = (part[0][e] + part[1][e]) + (part[2][e] + part[3][e]);
        scores(pt, 0, 0);
#pragma unroll
        for (int nt = 0; nt < VT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) x[nt][e] *= fi;
        if (cut) {
          cut_scores(pt, 0, 0);
#pragma unroll
          for (int nt = 0; nt < VT; nt++) cut_entering(x[nt], 0);
        }
        float o[4][VT];
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
          for (int nt = 0; nt < VT; nt++) x[nt] = mfma4(c.vc[0][e].get(nt), pt[e], x[nt]);
#pragma unroll
        for (int nt = 0; nt < VT; nt++)
#pragma unroll
          for (int e = 0; e < 4; e++) o[e][nt] = x[nt][e];
        put_tile(0, o);
      }
      if (!carried(n)) return true;
      decay();
#pragma unroll
      for (int mt = 0; mt < KT; mt++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float kw = key(0, mt, e);
#pragma unroll
          for (int nt = 0; nt < VT; nt++) S[mt][nt] = mfma4(kw, c.vc[0][e].get(nt), S[mt][nt]);
        }
    }
    if (STATE) through = cut || through < 0.0f ? DROPS : through * gn;
    return true;
  };
  while (p < hi) {
    Chunk c;
    /* whole chunks, then tiles */
    const int left = hi - p;
    n = single || chunk == 1 ? 1 : left >= C ? C : left < 16 ? left : 16;
    load(c, p, n);
    if (!work(c)) {
      single = n;
      continue;
    }
    p += n;
    if (single) single--;
  }

  float* s_out = nullptr;
  if (STATE) {
    s_out = w.ws + (bh * nsplit + split + 1) * room((int)elems);
    if (slab == 0 && lane == 0) w.wf[bh * nsplit + split + 1] = through;
  }
  else if (split == nsplit - 1 && w.s_out) s_out = w.s_out + bh * elems;
  if (s_out) {
    /* the state in front of a start that the first token carries gets no gradient */
    if (!STATE && rev && starts && len > 0 && starts[0]) {
#pragma unroll
      for (int mt = 0; mt < KT; mt++)
#pragma unroll
        for (int nt = 0; nt < VT; nt++) S[mt][nt] = f4{0, 0, 0, 0};
    }
    const Rsrc rs = rsrc_of(s_out);
    /* (the walks on transposed states only read them) */
#pragma unroll
    for (int mt = 0; mt < KT; mt++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float x[VT];
#pragma unroll
        for (int nt = 0; nt < VT; nt++) x[nt] = S[mt][nt][e];
        store_n<float, VT>(rs, at((PK::of(g, e, kdim) + mt) * srow, own(e, mt), FAR_T) + at(vcolumn * scol, vthere, FAR_D), x);
      }
  }
}

/* Rows of less than four channels, which no lane's load fits, are copied into rows of eight, padded with zeros;
   padding tokens are left out.  A thread moves a row. */
struct PackArgs {
  struct One {
    Tok src;
    void* dst;
    int heads, d;
  } x[4];
  int b, t;
  const int* lengths;
};
template <class T> __global__ __launch_bounds__(256) void k_attn_pack(PackArgs a) {
  const PackArgs::One x = a.x[blockIdx.y];
  const unsigned long long n = (unsigned long long)a.b * a.t * x.heads;
  struct alignas(16) Whole { T e[8]; };
  for (unsigned long long i = (unsigned long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (unsigned long long)gridDim.x * 256) {
    unsigned long long r = i;
    const int h = (int)(r % x.heads);
    r /= x.heads;
    const int t = (int)(r % a.t), b = (int)(r / a.t);
    if (a.lengths && t >= a.lengths[b]) continue;
    const T* src = (const T*)x.src.p + b * x.src.sb + t * x.src.st + h * x.src.sh;
    Whole y;
#pragma unroll
    for (int e = 0; e < 8; e++) y.e[e] = e < x.d ? src[e] : from_f<T>(0.0f);
    reinterpret_cast<Whole*>(x.dst)[i] = y;
  }
}

/* States that enter each split: ws[s] holds split s - 1's own sum (k_attn_walk, STATE) and becomes
   X_s = wf[s] X_{s-1} + ws[s], X_0 = s_in.  Nothing but the chain of multiply-adds depends on the split in front.

   Many elements: a thread owns VW of them and runs along the splits, whose sums it loads LOT at a time, the next
   lot while one is chained; the bytes bound it (both directions of eight demonstrations of 10,500 tokens: 15.6 us). */
__device__ __forceinline__ float carry_on(float f, float x, float u) { return (f < 0.0f ? 0.0f : f * x) + u; }
__global__ __launch_bounds__(64) void k_attn_join(WalkArgs a) {
  constexpr int VW = 4, LOT = 8;
  const Walk w = a.w[blockIdx.z];
  const long long bh = blockIdx.y;
  const int elems = a.kdim * a.vdim, next_state = room(elems), nsplit = a.nsplit;
  const int e = (blockIdx.x * 64 + threadIdx.x) * VW;
  if (e >= elems) return;
  struct alignas(4 * VW) Pack { float x[VW]; };
  float* ws = w.ws + bh * nsplit * next_state + e;
  const float* wf = w.wf + bh * nsplit;
  struct Lot { Pack u[LOT]; float f[LOT]; };
  auto load = [&](Lot& l, int s0) {
#pragma unroll
    for (int i = 0; i < LOT; i++) {
      const int s = s0 + 1 + i < nsplit ? s0 + 1 + i : nsplit - 1;
      l.u[i] = *reinterpret_cast<const Pack*>(ws + (long long)s * next_state);
      l.f[i] = wf[s];
    }
  };
  Lot l;
  load(l, 0);
  Pack x = {};
  if (w.s_in)
#pragma unroll
    for (int c = 0; c < VW; c++) x.x[c] = e + c < elems ? w.s_in[bh * elems + e + c] : 0.0f;
  for (int s0 = 0; s0 < nsplit; s0 += LOT) {
    Lot next;
    if (s0 + LOT < nsplit) load(next, s0 + LOT);
#pragma unroll
    for (int i = 0; i < LOT; i++) {
      if (s0 + i < nsplit) *reinterpret_cast<Pack*>(ws + (long long)(s0 + i) * next_state) = x;
#pragma unroll
      for (int c = 0; c < VW; c++) x.x[c] = carry_on(l.f[i], x.x[c], l.u[i].x[c]);
    }
    l = next;
  }
}
/* Few elements wait for the chain: the waves of a workgroup take 32 splits each of the same 64 elements, all loads at
   once, chain their own from zero and pass on the result and the product of their factors; each then starts from
   what the waves in front make of the state.  The 165 splits of one demonstration of 10,500 tokens take 7.6 us, by the
   kernel above 22.0. */
#define JOIN_WAVES 16
__global__ __launch_bounds__(64 * JOIN_WAVES) void k_attn_join_wide(WalkArgs a) {
  constexpr int LOT = 32;
  __shared__ float sum[JOIN_WAVES][64], factor[JOIN_WAVES], last[64];
  const Walk w = a.w[blockIdx.z];
  const long long bh = blockIdx.y;
  const int elems = a.kdim * a.vdim, next_state = room(elems), nsplit = a.nsplit;
  const int lane = threadIdx.x & 63, me = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int e = blockIdx.x * 64 + lane;
  const bool ok = e < elems;
  float* ws = w.ws + bh * nsplit * next_state + (ok ? e : 0);
  const float* wf = w.wf + bh * nsplit;
  float start = ok && w.s_in ? w.s_in[bh * elems + e] : 0.0f;
  for (int s0 = 0; s0 < nsplit; s0 += waves * LOT) {
    const int mine = s0 + me * LOT; /* this wave turns ws[mine + 1 ..] into the states behind the state of split `mine` */
    float u[LOT], f[LOT], x = 0.0f, g = 1.0f;
#pragma unroll
    for (int i = 0; i < LOT; i++) {
      const int s = mine + 1 + i < nsplit ? mine + 1 + i : nsplit - 1;
      u[i] = ws[(long long)s * next_state];
      f[i] = wf[s];
    }
#pragma unroll
    for (int i = 0; i < LOT; i++)
      if (mine + 1 + i < nsplit) {
        x = carry_on(f[i], x, u[i]);
        g = g < 0.0f || f[i] < 0.0f ? DROPS : g * f[i];
      }
    sum[me][lane] = x;
    if (lane == 0) factor[me] = g;
    __syncthreads();
    x = start;
    for (int i = 0; i < me; i++) x = carry_on(factor[i], x, sum[i][lane]);
#pragma unroll
    for (int i = 0; i < LOT; i++)
      if (mine + i < nsplit) {
        if (ok) ws[(long long)(mine + i) * next_state] = x;
        x = carry_on(f[i], x, u[i]);
      }
    if (me == waves - 1) last[lane] = x;
    __syncthreads();
    start = last[lane];
  }
}

/* Sums of the per-query-head gradients over the `grp` heads that share a key / value head: rows of `width` floats,
   [b][t][hk][grp][width], to d channels of [b][t][hk] rows.  With grp = 1 it narrows the rows of less than four
   channels that the walks write eight wide.  A thread sums four channels; every tensor of a call in one launch.  Memory
   bounds it: 33 x 777 tokens, 6 heads over 2, 48 + 96 channels take 16.4 us (6.2 TB/s: they come from the Infinity
   Cache). */
struct SumArgs {
  struct One {
    const float* src;
    void* dst;
    long long sb, st, sh;
    unsigned hk, grp, d, width, n; /* n: threads */
  } x[3];
  unsigned t;
};
template <class T> __global__ __launch_bounds__(256) void k_attn_group_sum(SumArgs a) {
  const SumArgs::One x = a.x[blockIdx.y];
  struct alignas(4) Four { float e[4]; };
  const unsigned groups = (x.d + 3) / 4;
  for (unsigned long long i0 = (unsigned long long)blockIdx.x * 256; i0 < x.n; i0 += (unsigned long long)gridDim.x * 256) {
    const unsigned i = (unsigned)i0 + threadIdx.x;
    if (i >= x.n) return;
    unsigned r = i / groups;
    const unsigned c = (i - r * groups) * 4, left = x.d - c;
    const float* s = x.src + (long long)r * x.grp * x.width + c;
    const unsigned kh = r % x.hk;
    r /= x.hk;
    T* o = (T*)x.dst + r / a.t * x.sb + r % a.t * x.st + kh * x.sh + c;
    if (left >= 4) {
      Four y = {};
      for (unsigned k = 0; k < x.grp; k++) {
        const Four z = *reinterpret_cast<const Four*>(s + (long long)k * x.width);
#pragma unroll
        for (int e = 0; e < 4; e++) y.e[e] += z.e[e];
      }
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] = from_f<T>(y.e[e]);
    } else {
      for (unsigned e = 0; e < left; e++) {
        float y = 0.0f;
        for (unsigned k = 0; k < x.grp; k++) y += s[(long long)k * x.width + e];
        o[e] = from_f<T>(y);
      }
    }
  }
}

/* ---- one token -----------------------------------------------------------------------------------
   The state is read and written once and bounds the call: 4,096 envs x 4 heads of 64 x 64 take 102 us,
   5.4 TB/s (one env: 4.8 us, a launch and two trips to memory).
   A wave owns one (sequence, head) and a slab of CL groups of VW value channels: its lanes are the groups by 64 / CL
   rows, which they stream ROWS at a time: S' = a S + k v^T stored, o += q S' kept per lane and summed over the rows
   at the end.  Few sequences are cut into narrower slabs, so that more waves share their rows. */
struct StepArgs {
  Tok q, k, v, o;
  int b, h, kdim, vdim;
  float scale;
  const float* log_decay;
  const unsigned char* starts;
  long long starts_sb;
  const float* s_in;
  float* s_out;
};
template <class T, int VW> __global__ __launch_bounds__(256) void k_attn_step(StepArgs a, int cl_log, int slabs) {
  constexpr int ES = (int)sizeof(T), ROWS = 8;
  const int lane = threadIdx.x & 63;
  const unsigned task = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned bh = task / slabs;
  if (bh >= (unsigned)a.b * a.h) return;
  const int slab = task % slabs, b = (int)(bh / a.h), h = (int)(bh % a.h);
  const int CL = 1 << cl_log, RG = 64 >> cl_log;
  const int r0 = lane >> cl_log, d = (slab * CL + (lane & (CL - 1))) * VW;
  const bool ok = d < a.vdim; /* VW divides vdim */
  const bool cut = a.starts && a.starts[b * a.starts_sb];
  const float decay = expf(a.log_decay[h]);
  const Rsrc rq = rsrc_of((const char*)a.q.p + ES * (b * a.q.sb + h / a.q.hdiv * a.q.sh));
  const Rsrc rk = rsrc_of((const char*)a.k.p + ES * (b * a.k.sb + h / a.k.hdiv * a.k.sh));
  const T* v = (const T*)a.v.p + b * a.v.sb + h / a.v.hdiv * a.v.sh;
  T* o = (T*)a.o.p + b * a.o.sb + h / a.o.hdiv * a.o.sh;
  const long long base = (long long)bh * a.kdim * a.vdim;
  const Rsrc rs = rsrc_of(a.s_in + base, !cut); /* a state in front of a start is not read: zeros */
  const Rsrc rw = rsrc_of(a.s_out + base, a.s_out != nullptr);
  float vv[VW], acc[VW];
#pragma unroll
  for (int i = 0; i < VW; i++) { vv[i] = ok ? to_f(v[d + i]) : 0.0f; acc[i] = 0.0f; }
  for (int rr = r0; rr < a.kdim + r0; rr += RG * ROWS) {
    Raw<float, VW> s[ROWS];
    Raw<T, 1> kk[ROWS], qq[ROWS];
    unsigned off[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; u++) {
      const int row = rr + u * RG;
      const bool in = row < a.kdim;
      off[u] = at(4 * (row * a.vdim + d), in & ok, FAR_T);
      s[u].load(rs, off[u]);
      kk[u].load(rk, at(row * ES, in, FAR_T));
      qq[u].load(rq, at(row * ES, in, FAR_T));
    }
#pragma unroll
    for (int u = 0; u < ROWS; u++) {
      float x[VW];
#pragma unroll
      for (int i = 0; i < VW; i++) {
        x[i] = fmaf(kk[u].get(0), vv[i], decay * s[u].get(i));
        acc[i] = fmaf(qq[u].get(0), x[i], acc[i]);
      }
      store_n<float, VW>(rw, off[u], x);
    }
  }
#pragma unroll
  for (int i = 0; i < VW; i++) {
    for (int m = CL; m < 64; m <<= 1) acc[i] += __shfl_xor(acc[i], m);
    if (ok && r0 == 0) o[d + i] = from_f<T>(acc[i] * a.scale);
  }
}

/* ---- keyed dropout ------------------------------------------------------------------------------- */

/* Philox4x32-10 (Salmon et al., 2011), as the env's reset noise uses it */
__device__ __forceinline__ void philox(unsigned c0, unsigned c1, unsigned c2, unsigned c3, unsigned k0, unsigned k1,
                                       unsigned out[4]) {
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const unsigned long long p0 = (unsigned long long)0xD2511F53u * c0, p1 = (unsigned long long)0xCD9E8D57u * c2;
    const unsigned n0 = (unsigned)(p1 >> 32) ^ c1 ^ k0, n2 = (unsigned)(p0 >> 32) ^ c3 ^ k1;
    c1 = (unsigned)p1;
    c3 = (unsigned)p0;
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  out[0] = c0; out[1] = c1; out[2] = c2; out[3] = c3;
}

/* A thread takes the 8 columns of one Philox call.  131,072 x 256 bfloat16 with a residual, and the gradient, take 64 us,
   5.2 TB/s: memory bounds it, with ten rounds of products per 8 elements beside.
   WHOLE: rows of whole blocks on boundaries of 16 bytes.  ROWS: at least 8 columns on any boundary; the last block of a row
   reads the last 8 columns, its own behind the `back` that the block in front stores (39,049 x 405 bfloat16:
   13.6 us, 4.7 TB/s; element by element 38 us).  PARTS: less than 8 columns. */
enum Layout { WHOLE, ROWS, PARTS };
template <class T, Layout LAY>
__global__ __launch_bounds__(256) void k_keyed_dropout(long long rows, int cols, const T* x, long long xs, const T* res,
                                                       long long rs, T* y, long long ys, const long long* ids,
                                                       unsigned long long seed, unsigned sub, unsigned count, float up) {
  const unsigned blocks = (unsigned)(cols + 7) / 8;
  const long long n = rows * blocks;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const long long row = i / blocks;
  const unsigned j = (unsigned)(i % blocks);
  const unsigned long long id = ids ? (unsigned long long)ids[row] : (unsigned long long)row;
  const int m = LAY == WHOLE || cols - 8 * (int)j >= 8 ? 8 : cols - 8 * (int)j; /* columns of this block */
  const int back = LAY == ROWS ? 8 - m : 0, c0 = 8 * (int)j - back;
  float xv[8], rv[8];
  if constexpr (LAY != PARTS) {
    Eight<T, LAY == WHOLE>::load(x + row * xs + c0, xv);
    if (res) Eight<T, LAY == WHOLE>::load(res + row * rs + c0, rv);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      xv[e] = e < m ? to_f(x[row * xs + c0 + e]) : 0.0f;
      rv[e] = res && e < m ? to_f(res[row * rs + c0 + e]) : 0.0f;
    }
  }
  unsigned u[4];
  philox(j, (unsigned)id, (unsigned)(id >> 32), sub, (unsigned)seed, (unsigned)(seed >> 32), u);
  unsigned keep = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) keep |= ((e & 1 ? u[e >> 1] >> 16 : u[e >> 1] & 0xffffu) < count ? 1u : 0u) << e;
  keep <<= back;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    float z = keep >> e & 1 ? xv[e] * up : 0.0f; /* a dropped element is 0 whatever it held */
    if (res) z += rv[e];
    xv[e] = z;
  }
  T* const o = y + row * ys + c0;
  if (LAY == WHOLE || (LAY == ROWS && back == 0)) {
    Eight<T, LAY == WHOLE>::store(o, xv);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e >= back && e < back + m) o[e] = from_f<T>(xv[e]);
  }
}

/* ---- host ------------------------------------------------------------------------------------- */

static int bad_arg(const char* msg) { return ur3e_internal_fail(UR3E_EINVAL, msg); }

static int elem_size(int dtype) { return dtype == UR3E_F32 ? 4 : 2; }

static int attn_check(const ur3e_attn_t* a) {
  if (!a) return bad_arg("attention: null argument");
  if (a->dtype < UR3E_F32 || a->dtype > UR3E_F16) return bad_arg("attention: dtype must be 0 (float), 1 (bfloat16) or 2 (half)");
  if (a->b < 0 || a->t < 0 || a->heads < 1 || a->kv_heads < 1) return bad_arg("attention: need b >= 0, t >= 0, heads >= 1, kv_heads >= 1");
  if (a->heads % a->kv_heads) return bad_arg("attention: kv_heads must divide heads");
  if (a->dk < 1 || a->dk > UR3E_ATTN_MAX_DIM || a->dv < 1 || a->dv > UR3E_ATTN_MAX_DIM)
    return bad_arg("attention: dk and dv must be in [1, 128]");
  if ((long long)a->b * a->heads > 4194303) return bad_arg("attention: b * heads must be below 2^22");
  if (a->t > 1 << 30) return bad_arg("attention: t must be at most 2^30");
  /* 32-bit indices in k_attn_group_sum, of groups of four channels (query heads where nothing is shared) */
  const int most = a->dk > a->dv ? a->dk : a->dv;
  if ((a->heads != a->kv_heads || a->dk < 4 || a->dv < 4) &&
      (long long)a->b * a->t * (a->dk < 4 || a->dv < 4 ? a->heads : a->kv_heads) * ((most + 3) / 4) > 0xffffff00LL)
    return bad_arg("attention: too many tokens for shared heads or for less than 4 channels");
  if (a->b == 0) return UR3E_OK;
  if (a->q.st < 0 || a->k.st < 0 || a->v.st < 0 || a->starts_st < 0) return bad_arg("attention: token strides must not be negative");
  if (!a->log_decay) return bad_arg("attention: null log_decay");
  if (a->t > 0 && (!a->q.p || !a->k.p || !a->v.p)) return bad_arg("attention: null q, k or v");
  return UR3E_OK;
}

static int pow2_tiles(int d) { return d <= 16 ? 1 : d <= 32 ? 2 : d <= 64 ? 4 : 8; }

struct Tiles {
  int kt, vt, slabs;
};
/* the state of a wave is kdim x 16 vt floats, at most 64 registers a lane, so vt is at most 2 at 128 key channels */
static Tiles tiles_of(int kdim, int vdim) {
  Tiles p;
  p.kt = pow2_tiles(kdim);
  p.vt = pow2_tiles(vdim);
  const int most = p.kt == 8 ? 2 : 4;
  if (p.vt > most) p.vt = most;
  p.slabs = (vdim + 16 * p.vt - 1) / (16 * p.vt);
  return p;
}

struct Splits {
  int n, len;
};
/* How many waves share a sequence, from the waves of the smallest launch.  Two waves a SIMD (2,048) fill the card,
   and what does not fit beside them waits for a second round, so as many splits as still fit.  Padded sequences
   leave the waves of their padding idle: twice as many, unless the states of the splits, which are written, joined
   and read, would then move more bytes than the tokens.  A split costs a chain of chunks, and its state one more
   link of the chain of the join, so the shortest worth having grows with the square root of the length. */
static Splits splits_of(const ur3e_attn_t* a, int backward) {
  long long waves = (long long)a->b * a->heads * tiles_of(a->dk, a->dv).slabs;
  if (backward && a->dk == a->dv) waves *= 3;
  if (backward && a->dk != a->dv) {
    const long long other = 2LL * a->b * a->heads * tiles_of(a->dv, a->dk).slabs;
    if (other < waves) waves = other;
  }
  Splits p = {1, a->t > 0 ? a->t : 1};
  /* three launches take ~13 us more than one, the time of ~7 chunks */
  if (a->t < (a->dtype == UR3E_F32 ? 128 : 192)) return p;
  auto length = [&](long long n) { return (int)(((a->t + n - 1) / n + 15) / 16 * 16); };
  int least = 32;
  while ((long long)least * least * 4 < a->t) least += 16;
  const long long once = 2048 / waves, again = 4096 / waves;
  int len = once > 1 ? length(once) : a->t;
  if (a->lengths && again > 1) {
    const int even = 8 * a->dk * a->dv / ((a->dk + a->dv) * elem_size(a->dtype)), twice = length(again);
    const int more = twice > even ? twice : (even + 15) / 16 * 16;
    if (more < len) len = more;
  }
  if (len >= a->t) return p;
  p.len = len > least ? len : least;
  p.n = (a->t + p.len - 1) / p.len;
  if (p.n < 2) p = {1, a->t};
  return p;
}

/* the states that enter the splits, and the factors between them */
static size_t split_bytes(const ur3e_attn_t* a, const Splits& p) {
  return p.n > 1 ? (size_t)a->b * a->heads * p.n * (room(a->dk * a->dv) + 1) * sizeof(float) : 0;
}
static void split_use(const ur3e_attn_t* a, const Splits& p, void* ws, Walk& w) {
  if (p.n < 2) return;
  w.ws = (float*)ws;
  w.wf = w.ws + (long long)a->b * a->heads * p.n * room(a->dk * a->dv);
}

/* the rows hold a lane's load (Place::NC is 4 for up to 16 channels) */
static bool whole(int d) { return d >= 4; }

/* what a launch does: the states at the ends of the splits and their join, or the outputs */
enum Phase { STATES, OUTPUTS };

template <class T, int KT, int VT, bool STATE>
static void walk_kernel(const WalkArgs& a, bool fine, dim3 grid, dim3 block, hipStream_t s) {
  /* Two tiles of tokens at a time for 16-bit types, where there is more than one and the registers hold them (2,048 x 512
     tokens x 4 heads, gradients, two tiles at a time and one: 64 channels bfloat16 1.16 and 1.37 ms, half 1.34 and 1.46; 128
     channels bfloat16 4.43 and 4.25) */
  constexpr bool PAIRS = sizeof(T) == 2 && KT < 8;
  if constexpr (PAIRS) {
    if (a.t > 16) {
      if (fine) hipLaunchKernelGGL((k_attn_walk<T, KT, VT, STATE, 2, true>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((k_attn_walk<T, KT, VT, STATE, 2, false>), grid, block, 0, s, a);
      return;
    }
  }
  /* (splits, and with them STATE, are for longer sequences) */
  if constexpr (!STATE || !PAIRS) {
    if (sizeof(T) == 4 || fine) hipLaunchKernelGGL((k_attn_walk<T, KT, VT, STATE, 1, true>), grid, block, 0, s, a);
    else if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((k_attn_walk<T, KT, VT, STATE, 1, false>), grid, block, 0, s, a);
  }
}
template <class T, int KT, int VT> static int walk_launch(WalkArgs& a, Phase phase, hipStream_t s) {
  const long long tasks = (long long)a.b * a.h * a.nw * a.slabs * (phase == STATES ? a.nsplit - 1 : a.nsplit);
  /* The waves that share a sequence's tensors in one workgroup, where they are two or four (128 channels bfloat16: 1.51 ms,
     in workgroups of one wave 1.58).  Not three: two waves fit a SIMD, so a compute unit would hold two such workgroups and
     leave two of its eight places empty (float gradients at 64 channels 2.63 ms, one by one 2.45).  Nor where there is less
     than a wave a SIMD: one by one they spread over all units (16 sequences x 16 tokens, both directions: 14.6 us, 13.3). */
  const int share = a.nw * a.slabs, waves = tasks <= 1024 || share == 3 ? 1 : share <= 4 ? share : 4;
  a.near = (share + waves - 1) / waves;
  constexpr int load = Place<T, VT>::NC;
  a.lent = a.slabs > 1 && a.vdim - (a.slabs - 1) * 16 * VT < load ? load : 0;
  const long long per = 8LL * a.near * waves;
  const dim3 grid((unsigned)((tasks + per - 1) / per * 8 * a.near)), block(64 * waves);
  bool fine = false;
  for (int i = 0; i < a.nw; i++) fine = fine || a.w[i].s_out;
  if (phase == STATES) {
    walk_kernel<T, KT, VT, true>(a, fine, grid, block, s);
    PL_CHK(hipGetLastError());
    const int elems = a.kdim * a.vdim;
    const unsigned bh = (unsigned)(a.b * a.h), nw = (unsigned)a.nw;
    /* From 2^18 elements on the bytes count, below it the chain (64 x 64 states, four elements a thread and the wide one: 2^17
       elements, 64 splits 12.1 and 11.0 us; 2^18, 32 splits 10.9 and 11.6; 2^19, 16 splits 10.7 and 13.8; 2^21, 4 splits 10.6 and
       32.3).  A wave of the wide one for each 32 splits, up to 16. */
    const int join_waves = a.nsplit <= 32 * JOIN_WAVES ? (a.nsplit + 31) / 32 : JOIN_WAVES;
    if ((long long)bh * nw * elems >= 64 * 4096)
      hipLaunchKernelGGL(k_attn_join, dim3((elems + 255) / 256, bh, nw), dim3(64), 0, s, a);
    else
      hipLaunchKernelGGL(k_attn_join_wide, dim3((elems + 63) / 64, bh, nw), dim3(64 * join_waves), 0, s, a);
  } else {
    walk_kernel<T, KT, VT, false>(a, fine, grid, block, s);
  }
  PL_CHK(hipGetLastError());
  return UR3E_OK;
}
template <class T, int KT, int VT> static int walk_tile(WalkArgs& a, Phase phase, hipStream_t s) {
  a.chunk = 16;
  /* a tile's tokens (a chunk's starts) within its 30-bit offsets, else token by token */
  auto far = [](long long st, int e, int tokens = 16) { return st > ((1LL << 30) - 1024) / tokens / e; };
  if (far(a.starts_st, 1, 32)) a.chunk = 1;
  for (int i = 0; i < a.nw; i++) {
    const Walk& w = a.w[i];
    if (far(w.q.st, sizeof(T)) || far(w.k.st, sizeof(T)) || far(w.v.st, sizeof(T)) || far(w.o.st, w.out_f32 ? 4 : sizeof(T))) a.chunk = 1;
  }
  return walk_launch<T, KT, VT>(a, phase, s);
}
template <class T, int KT> static int walk_vt(WalkArgs& a, int vt, Phase phase, hipStream_t s) {
  if (vt == 1) return walk_tile<T, KT, 1>(a, phase, s);
  if (vt == 2) return walk_tile<T, KT, 2>(a, phase, s);
  if constexpr (KT < 8) return walk_tile<T, KT, 4>(a, phase, s);
  return bad_arg("attention: no such tile");
}
template <class T> static int walk_kt(WalkArgs& a, const Tiles& p, Phase phase, hipStream_t s) {
  switch (p.kt) {
    case 1: return walk_vt<T, 1>(a, p.vt, phase, s);
    case 2: return walk_vt<T, 2>(a, p.vt, phase, s);
    case 4: return walk_vt<T, 4>(a, p.vt, phase, s);
    default: return walk_vt<T, 8>(a, p.vt, phase, s);
  }
}
static int walk_run(int dtype, WalkArgs& a, Phase phase, hipStream_t s) {
  Tiles p = tiles_of(a.kdim, a.vdim);
  /* Where the card has room, narrower slabs: a wave's chunk of 16 tokens of 64 x 64 float channels takes 3.3 us, with
     a quarter of the value channels 2.1 us, for keys and scores that four waves then read and form. */
  while (p.vt > 1 && (long long)a.b * a.h * a.nw * p.slabs * a.nsplit <= 1024) {
    p.vt /= 2;
    p.slabs = (a.vdim + 16 * p.vt - 1) / (16 * p.vt);
  }
  a.slabs = p.slabs;
  if (dtype == UR3E_F32) return walk_kt<float>(a, p, phase, s);
  if (dtype == UR3E_BF16) return walk_kt<Bf16>(a, p, phase, s);
  return walk_kt<F16>(a, p, phase, s);
}

static Tok tok_of(const ur3e_tokens_t& x, int hdiv) { return Tok{x.p, x.sb, x.st, x.sh, hdiv}; }

static WalkArgs args_of(const ur3e_attn_t* a, int kdim, int vdim, const Splits& p) {
  WalkArgs w = {};
  w.b = a->b; w.t = a->t; w.h = a->heads; w.kdim = kdim; w.vdim = vdim;
  w.nsplit = p.n; w.split_len = p.len;
  w.log_decay = a->log_decay;
  w.starts = a->starts; w.starts_sb = a->starts_sb; w.starts_st = a->starts_st;
  w.lengths = a->lengths;
  return w;
}

static size_t up256(size_t x) { return (x + 255) / 256 * 256; }

/* The tokens of a call as the walks read them: in place, or as copies behind `used` bytes of the workspace. */
struct Packer {
  const ur3e_attn_t* a;
  char* ws = nullptr;
  size_t used = 0;
  PackArgs args = {};
  int n = 0;
  long long most = 0;
  Tok use(const ur3e_tokens_t& x, int heads, int d, int hdiv) {
    Tok t = tok_of(x, hdiv);
    const int e = elem_size(a->dtype);
    if (whole(d) || a->t == 0) return t;
    PackArgs::One& o = args.x[n++];
    o.src = t;
    o.dst = ws + used;
    o.heads = heads; o.d = d;
    const long long rows = (long long)a->b * a->t * heads;
    if (rows > most) most = rows;
    used += up256((size_t)rows * 8 * e);
    return Tok{o.dst, (long long)a->t * heads * 8, (long long)heads * 8, 8, hdiv};
  }
  int run(hipStream_t s) {
    if (!n) return UR3E_OK;
    args.b = a->b; args.t = a->t; args.lengths = a->lengths;
    const long long blocks = (most + 255) / 256;
    const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20), n);
    if (a->dtype == UR3E_F32) hipLaunchKernelGGL(k_attn_pack<float>, grid, dim3(256), 0, s, args);
    else if (a->dtype == UR3E_BF16) hipLaunchKernelGGL(k_attn_pack<Bf16>, grid, dim3(256), 0, s, args);
    else hipLaunchKernelGGL(k_attn_pack<F16>, grid, dim3(256), 0, s, args);
    PL_CHK(hipGetLastError());
    return UR3E_OK;
  }
};

/* An output that the walks write as float rows of their own: one a query head for gradients of shared heads, eight
   wide for rows that hold no lane's store. */
struct Wide {
  const ur3e_attn_t* a;
  float* p = nullptr;
  int d = 0, grp = 1, width = 0;
  ur3e_tokens_t to = {};
  /* the walk's output: `x` itself or these rows, `used` bytes into the workspace */
  Tok use(const ur3e_tokens_t& x, int channels, int heads_per, char* ws, size_t& used) {
    if (heads_per == 1 && whole(channels)) return tok_of(x, 1);
    d = channels; grp = heads_per; to = x;
    width = whole(d) ? d : 8;
    p = (float*)(ws + used);
    used += up256((size_t)a->b * a->t * a->heads * width * 4);
    return Tok{p, (long long)a->t * a->heads * width, (long long)a->heads * width, width, 1};
  }
};
static int wide_finish(const ur3e_attn_t* a, const Wide* const* wide, int count, hipStream_t s) {
  SumArgs args = {};
  int n = 0;
  unsigned most = 0;
  for (int i = 0; i < count; i++) {
    const Wide& w = *wide[i];
    if (!w.width || a->t == 0) continue;
    SumArgs::One& x = args.x[n++];
    x.src = w.p; x.dst = w.to.p;
    x.sb = w.to.sb; x.st = w.to.st; x.sh = w.to.sh;
    x.hk = a->heads / w.grp; x.grp = w.grp; x.d = w.d; x.width = w.width;
    x.n = (unsigned)((long long)a->b * a->t * x.hk * ((w.d + 3) / 4));
    if (x.n > most) most = x.n;
  }
  if (!n) return UR3E_OK;
  args.t = a->t;
  const unsigned blocks = (most + 255) / 256;
  const dim3 grid(blocks < (1 << 20) ? blocks : 1 << 20, n);
  if (a->dtype == UR3E_F32) hipLaunchKernelGGL(k_attn_group_sum<float>, grid, dim3(256), 0, s, args);
  else if (a->dtype == UR3E_BF16) hipLaunchKernelGGL(k_attn_group_sum<Bf16>, grid, dim3(256), 0, s, args);
  else hipLaunchKernelGGL(k_attn_group_sum<F16>, grid, dim3(256), 0, s, args);
  PL_CHK(hipGetLastError());
  return UR3E_OK;
}

/* The workspace of a call: the states of its splits, its wide outputs, its copied inputs. */
struct ForwardSpace {
  Splits p;
  size_t used;
  Wide out;
  Packer pack;
  Tok q, k, v, o;
  ForwardSpace(const ur3e_attn_t* a, const ur3e_tokens_t& to, void* ws) : p(splits_of(a, 0)), out{a}, pack{a} {
    const int grp = a->heads / a->kv_heads;
    used = up256(split_bytes(a, p));
    o = out.use(to, a->dv, 1, (char*)ws, used);
    pack.ws = (char*)ws; pack.used = used;
    q = pack.use(a->q, a->heads, a->dk, 1); k = pack.use(a->k, a->kv_heads, a->dk, grp); v = pack.use(a->v, a->kv_heads, a->dv, grp);
    used = pack.used;
  }
};
struct BackwardSpace {
  Splits p;
  size_t states, used; /* bytes of one walk's states, of everything */
  Wide wq, wk, wv;
  Packer pack;
  Tok q, k, v, dout, dq, dk, dv;
  BackwardSpace(const ur3e_attn_t* a, const ur3e_tokens_t& g, const ur3e_tokens_t& tq, const ur3e_tokens_t& tk,
                const ur3e_tokens_t& tv, void* ws)
      : p(splits_of(a, 1)), wq{a}, wk{a}, wv{a}, pack{a} {
    const int grp = a->heads / a->kv_heads;
    states = up256(split_bytes(a, p));
    used = 2 * states;
    dq = wq.use(tq, a->dk, 1, (char*)ws, used);
    dk = wk.use(tk, a->dk, grp, (char*)ws, used);
    dv = wv.use(tv, a->dv, grp, (char*)ws, used);
    pack.ws = (char*)ws; pack.used = used;
    q = pack.use(a->q, a->heads, a->dk, 1); k = pack.use(a->k, a->kv_heads, a->dk, grp); v = pack.use(a->v, a->kv_heads, a->dv, grp);
    dout = pack.use(g, a->heads, a->dv, 1);
    used = pack.used;
  }
};

static int space_check(size_t need, const void* ws, size_t bytes) {
  if (bytes < need || (need && !ws)) return bad_arg("attention: workspace too small");
  if ((uintptr_t)ws % 16) return bad_arg("attention: workspace must be on a boundary of 16 bytes");
  return UR3E_OK;
}

extern "C" int ur3e_attn_workspace(const ur3e_attn_t* a, int backward, size_t* bytes) {
  const int rc = attn_check(a);
  if (rc) return rc;
  if (!bytes) return bad_arg("attention: null bytes");
  const ur3e_tokens_t any = {};
  *bytes = a->b == 0 ? 0 : backward ? BackwardSpace(a, any, any, any, any, nullptr).used : ForwardSpace(a, any, nullptr).used;
  return UR3E_OK;
}

extern "C" int ur3e_attn_forward(const ur3e_attn_t* a, const ur3e_tokens_t* out, float* s_out, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  int rc = attn_check(a);
  if (rc) return rc;
  if (a->b == 0) return UR3E_OK;
  if (!out || (a->t > 0 && !out->p)) return bad_arg("attention: null out");
  if (out->st < 0) return bad_arg("attention: token strides must not be negative");
  ForwardSpace ws(a, *out, workspace);
  rc = space_check(ws.used, workspace, workspace_bytes);
  if (rc) return rc;
  hipStream_t s = (hipStream_t)stream;
  rc = ws.pack.run(s);
  if (rc) return rc;
  WalkArgs w = args_of(a, a->dk, a->dv, ws.p);
  w.nw = 1;
  Walk& f = w.w[0];
  f.q = ws.q; f.k = ws.k; f.v = ws.v; f.o = ws.o;
  f.out_f32 = ws.out.width != 0;
  f.s_in = a->s0; f.s_out = s_out;
  f.in_scale = f.p_scale = a->scale; f.w_scale = 1.0f;
  split_use(a, ws.p, workspace, f);
  if (ws.p.n > 1) {
    rc = walk_run(a->dtype, w, STATES, s);
    if (rc) return rc;
  }
  rc = walk_run(a->dtype, w, OUTPUTS, s);
  if (rc) return rc;
  const Wide* wide[] = {&ws.out};
  return wide_finish(a, wide, 1, s);
}

extern "C" int ur3e_attn_backward(const ur3e_attn_t* a, const ur3e_tokens_t* dout, const float* ds_out,
                                  const ur3e_tokens_t* dq, const ur3e_tokens_t* dk, const ur3e_tokens_t* dv, float* ds0,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  int rc = attn_check(a);
  if (rc) return rc;
  if (a->b == 0) return UR3E_OK;
  if (!dout || !dq || !dk || !dv) return bad_arg("attention: null gradient");
  if (a->t > 0 && (!dout->p || !dq->p || !dk->p || !dv->p)) return bad_arg("attention: null gradient");
  if (dout->st < 0 || dq->st < 0 || dk->st < 0 || dv->st < 0) return bad_arg("attention: token strides must not be negative");
  BackwardSpace ws(a, *dout, *dq, *dk, *dv, workspace);
  rc = space_check(ws.used, workspace, workspace_bytes);
  if (rc) return rc;
  hipStream_t s = (hipStream_t)stream;
  rc = ws.pack.run(s);
  if (rc) return rc;
  Walk f = {}, q = {}, k = {}, v = {};
  /* dq = walk(do, v, k) on S^T */
  q.q = ws.dout; q.k = ws.v; q.v = ws.k; q.o = ws.dq;
  q.out_f32 = ws.wq.width != 0;
  q.state_t = 1;
  q.s_in = a->s0;
  q.in_scale = q.p_scale = a->scale; q.w_scale = 1.0f;
  split_use(a, ws.p, workspace, q);
  /* dv = reversed walk(k, q, do) on G */
  v.q = ws.k; v.k = ws.q; v.v = ws.dout; v.o = ws.dv;
  v.out_f32 = ws.wv.width != 0;
  v.s_in = ds_out; v.s_out = ds0;
  v.reversed = 1;
  v.in_scale = 1.0f; v.p_scale = v.w_scale = a->scale;
  split_use(a, ws.p, (char*)workspace + ws.states, v);
  /* dk = reversed walk(v, do, q) on G^T */
  k = v;
  k.q = ws.v; k.k = ws.dout; k.v = ws.q; k.o = ws.dk;
  k.out_f32 = ws.wk.width != 0;
  k.state_t = 1;
  k.s_out = nullptr;
  if (ws.p.n > 1) {
    /* the states of the splits: S of the forward walk, and G, which dk and dv share */
    f.k = ws.k; f.v = ws.v;
    f.s_in = a->s0;
    f.w_scale = 1.0f;
    split_use(a, ws.p, workspace, f);
    WalkArgs w = args_of(a, a->dk, a->dv, ws.p);
    w.w[0] = f; w.w[1] = v;
    w.nw = 2;
    rc = walk_run(a->dtype, w, STATES, s);
    if (rc) return rc;
  }
  WalkArgs w = args_of(a, a->dv, a->dk, ws.p);
  w.w[0] = q; w.w[1] = k; w.w[2] = v;
  w.nw = a->dk == a->dv ? 3 : 2;
  rc = walk_run(a->dtype, w, OUTPUTS, s);
  if (rc) return rc;
  if (w.nw == 2) {
    WalkArgs x = args_of(a, a->dk, a->dv, ws.p);
    x.w[0] = v;
    x.nw = 1;
    rc = walk_run(a->dtype, x, OUTPUTS, s);
    if (rc) return rc;
  }
  const Wide* wide[] = {&ws.wq, &ws.wk, &ws.wv};
  return wide_finish(a, wide, 3, s);
}

extern "C" int ur3e_attn_step(const ur3e_attn_t* a, const ur3e_tokens_t* out, const float* state_in, float* state_out,
                              void* stream) {
  int rc = attn_check(a);
  if (rc) return rc;
  if (a->t != 1) return bad_arg("attention step: t must be 1");
  if (a->lengths) return bad_arg("attention step: lengths must be null");
  if (a->b == 0) return UR3E_OK;
  if (!out || !out->p || !state_in) return bad_arg("attention step: null out or state");
  StepArgs s = {};
  const int grp = a->heads / a->kv_heads;
  s.q = tok_of(a->q, 1); s.k = tok_of(a->k, grp); s.v = tok_of(a->v, grp); s.o = tok_of(*out, 1);
  s.b = a->b; s.h = a->heads; s.kdim = a->dk; s.vdim = a->dv;
  s.scale = a->scale; s.log_decay = a->log_decay;
  s.starts = a->starts; s.starts_sb = a->starts_sb;
  s.s_in = state_in; s.s_out = state_out;
  const bool v4 = a->dv % 4 == 0;
  const int groups = v4 ? a->dv / 4 : a->dv;
  int cl = 0;
  while ((1 << cl) < groups && cl < 6) cl++;
  auto slabs = [&] { return (groups + (1 << cl) - 1) >> cl; };
  /* A wave a SIMD (1,024) where that leaves 64 bytes of a row to a wave, four groups (one env's head of 64 x 64: 4.1 us, a
     group alone 5.5; 256 heads of 128 x 128: 7.2, 8 groups 7.1, 16 groups 8.2, one 19.0) */
  while (cl > 2 && (long long)a->b * a->heads * slabs() < 1024) cl--;
  const dim3 grid((unsigned)(((long long)a->b * a->heads * slabs() + 3) / 4));
  hipStream_t st = (hipStream_t)stream;
  auto run = [&](auto four, auto one) { hipLaunchKernelGGL(v4 ? four : one, grid, dim3(256), 0, st, s, cl, slabs()); };
  if (a->dtype == UR3E_F32) run(k_attn_step<float, 4>, k_attn_step<float, 1>);
  else if (a->dtype == UR3E_BF16) run(k_attn_step<Bf16, 4>, k_attn_step<Bf16, 1>);
  else run(k_attn_step<F16, 4>, k_attn_step<F16, 1>);
  PL_CHK(hipGetLastError());
  return UR3E_OK;
}

template <class T>
static int dropout_launch(long long rows, int cols, const void* x, long long xs, const void* res, long long rs, void* y,
                          long long ys, const long long* ids, unsigned long long seed, unsigned sub, int count, hipStream_t s) {
  const long long n = rows * ((cols + 7) / 8);
  const float up = count ? 65536.0f / (float)count : 0.0f;
  constexpr int E = 16 / (int)sizeof(T);
  auto al = [](const void* p, long long st) { return (uintptr_t)p % 16 == 0 && st % E == 0; };
  const Layout lay = cols < 8 ? PARTS : cols % 8 == 0 && al(x, xs) && al(y, ys) && (!res || al(res, rs)) ? WHOLE : ROWS;
  const dim3 grid((unsigned)((n + 255) / 256));
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, rows, cols, (const T*)x, xs, (const T*)res, rs, (T*)y, ys, ids, seed, sub, (unsigned)count, up);
  };
  if (lay == WHOLE) run(k_keyed_dropout<T, WHOLE>);
  else if (lay == ROWS) run(k_keyed_dropout<T, ROWS>);
  else run(k_keyed_dropout<T, PARTS>);
  PL_CHK(hipGetLastError());
  return UR3E_OK;
}

extern "C" int ur3e_keyed_dropout(int dtype, long long rows, int cols, const void* x, long long x_stride,
                                  const void* residual, long long residual_stride, void* y, long long y_stride,
                                  const long long* row_ids, unsigned long long seed, unsigned int substream,
                                  int keep_count, void* stream) {
  if (dtype < UR3E_F32 || dtype > UR3E_F16) return bad_arg("dropout: dtype must be 0 (float), 1 (bfloat16) or 2 (half)");
  if (rows < 0 || cols < 0) return bad_arg("dropout: need rows >= 0 and cols >= 0");
  if (keep_count < 0 || keep_count > 65536) return bad_arg("dropout: keep_count must be in [0, 65536]");
  if (rows == 0 || cols == 0) return UR3E_OK;
  if (!x || !y) return bad_arg("dropout: null argument");
  if (rows > 0xffffff00LL || rows * (((long long)cols + 7) / 8) > 0xffffff00LL) return bad_arg("dropout: too many elements for one call");
  hipStream_t s = (hipStream_t)stream;
  if (dtype == UR3E_F32) return dropout_launch<float>(rows, cols, x, x_stride, residual, residual_stride, y, y_stride, row_ids, seed, substream, keep_count, s);
  if (dtype == UR3E_BF16) return dropout_launch<Bf16>(rows, cols, x, x_stride, residual, residual_stride, y, y_stride, row_ids, seed, substream, keep_count, s);
  return dropout_launch<F16>(rows, cols, x, x_stride, residual, residual_stride, y, y_stride, row_ids, seed, substream, keep_count, s);
}
