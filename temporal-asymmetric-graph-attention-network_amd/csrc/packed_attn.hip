// Attention over packed sequences (different lengths behind one another, grouped key heads, causal), its backward, and
// the serving form against a cache.  For one sequence and one key head, with the group's G query heads packed as rows
// r = token * G + g:
//   S = scale Q Kᵀ over the visible keys (j <= token + Lk - Lq when causal), P = softmax(S), O = P V
//   dV = Pᵀ dO, dP = dO Vᵀ, dS = P (dP - rowsum(dO O)), dQ = scale dS K, dK = scale dSᵀ Q  (sums over the group's rows)
// One pass over the keys with a running maximum and sum (fp32); a row that sees no key gives zeros.  The backward makes
// P again from the stored log-sum-exp: one kernel over row tiles for dQ, one over key tiles for dK and dV, no atomics,
// every sum in a fixed order.
//
// Matrix cores: 32x32 tiles, bf16 products of 16 (v_mfma_f32_32x32x16_bf16) or fp32 products of 2, accumulated in
// fp32.  A fragment is 8 contraction values of a lane: lane l holds row (or column) l % 32 and the values
// 8 (l / 32) .. + 7 of a run of 16.  Scores are formed transposed (keys in the accumulator's registers, the row in the
// lane), so a row's softmax statistics are one per lane and its reduction is in registers plus one half swap; the
// accumulator's 8 registers of a run of 16 keys are, converted, the second product's operand without any exchange,
// because a contraction may take its keys in any order as long as both operands do: value j of half h is key
// 4 h + j % 4 + 8 (j / 4).  The other operand comes transposed out of LDS in that order (ds_read_tr16 for bf16).
//
// LDS tiles are filled by direct loads (buffer_load ... lds); the descriptor's bound makes rows behind the sequence
// and features behind head_dim zeros.  16-byte chunks are swizzled within a row so that both the row reads (16 rows,
// one chunk) and the transposed reads (4 rows, 64 bytes) touch all banks once.
#include "common.cuh"

namespace tagan {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

#define TAGAN_LDS(T, p) ((__attribute__((address_space(3))) T*)(p))

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LAZY = 8.f;
constexpr int SHORT = 128;   // keys of a history up to which the FINE kernels take two operands

// ------------------------------------------------------------------------------------------------ fragments
template <typename T>
struct Frag;
template <>
struct Frag<uint16_t> {
    union {
        bf16x8 v;
        s16x4 h[2];
        uint32_t u[4];
    };
    __device__ __forceinline__ void zero() { u[0] = u[1] = u[2] = u[3] = 0; }
};
template <>
struct Frag<float> {
    float v[8];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
};

__device__ __forceinline__ void mma(f32x16& c, const Frag<uint16_t>& a, const Frag<uint16_t>& b) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& c, const Frag<float>& a, const Frag<float>& b) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], c, 0, 0, 0);
}

// eight accumulator registers as an operand (bf16: one rounding to nearest even of each probability or its gradient; the
// matrix cores take no wider operand at this rate, and over many keys the roundings average out)
__device__ __forceinline__ void from_acc(Frag<uint16_t>& f, const f32x16& c, int at) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f.u[j] = f2bf2(c[at + 2 * j], c[at + 2 * j + 1]);
}
__device__ __forceinline__ void from_acc(Frag<float>& f, const f32x16& c, int at) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = c[at + j];
}

// and what that rounding took away, as a second operand
__device__ __forceinline__ void rest_of(Frag<uint16_t>& f, const f32x16& c, int at) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float a = c[at + 2 * j], b = c[at + 2 * j + 1];
        const uint32_t u = f2bf2(a, b);
        f.u[j] = f2bf2(a - __uint_as_float(u << 16), b - __uint_as_float(u & 0xffff0000u));
    }
}

__device__ __forceinline__ void load_frag(Frag<uint16_t>& f, const uint16_t* p) {
    const uint4 u = *(const uint4*)p;
    f.u[0] = u.x; f.u[1] = u.y; f.u[2] = u.z; f.u[3] = u.w;
}
__device__ __forceinline__ void load_frag(Frag<float>& f, const float* p) {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    f.v[0] = a.x; f.v[1] = a.y; f.v[2] = a.z; f.v[3] = a.w;
    f.v[4] = b.x; f.v[5] = b.y; f.v[6] = b.z; f.v[7] = b.w;
}
__device__ __forceinline__ float dot(const Frag<uint16_t>& a, const Frag<uint16_t>& b) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        s = fmaf(__uint_as_float(a.u[j] << 16), __uint_as_float(b.u[j] << 16), s);
        s = fmaf(__uint_as_float(a.u[j] & 0xffff0000u), __uint_as_float(b.u[j] & 0xffff0000u), s);
    }
    return s;
}
__device__ __forceinline__ float dot(const Frag<float>& a, const Frag<float>& b) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(a.v[j], b.v[j], s);
    return s;
}

__device__ __forceinline__ void store4(uint16_t* p, float a, float b, float c, float d) {
    *(uint2*)p = make_uint2(f2bf2(a, b), f2bf2(c, d));
}
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
    *(float4*)p = make_float4(a, b, c, d);
}

// ------------------------------------------------------------------------------------------------ LDS tiles
// [rows][D] of T, chunk c of row r at chunk c ^ swz(r)
template <typename T, int D>
struct Tile {
    static constexpr int E = 16 / (int)sizeof(T);      // elements of a chunk
    static constexpr int CPR = D / E;                  // chunks of a row: 2 to 32
    static constexpr int ROW = D * (int)sizeof(T);     // bytes of a row
    // 16 features: the 32-wide transposed reads pass the row's end (and at the last one the tile's); what they bring from
    // there goes to accumulator rows that are never stored
    static constexpr int PAD = D < 32 ? 64 : 0;

    __device__ static __forceinline__ int swz(int r) {
        if constexpr (CPR == 2) return (r >> 3) & 1;
        else if constexpr (CPR == 4) return (r >> 2) & 3;
        else if constexpr (CPR == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
        else return ((r & 3) << 2) | ((r >> 2) & 3);
    }

    static constexpr int RPW = 64 / CPR;               // rows of a wave's load
    static constexpr uint32_t PAST = 0x7ffffff0u;      // an offset behind every bound: the load writes zeros

    // A thread's place in the loads of a tile whose rows are `stride` bytes apart: the row's offset, the chunk's, and
    // their sum where it lies inside head_dim.
    struct Lay {
        uint32_t row, chunk, sum;
    };
    template <int WAVES>
    __device__ static __forceinline__ Lay lay(uint32_t stride, uint32_t bytes) {
        const int r = (WAVES == 1 ? 0 : (int)threadIdx.x >> 6) * RPW + (threadIdx.x & 63) / CPR;
        Lay y;
        y.row = (uint32_t)r * stride;
        y.chunk = (uint32_t)(((threadIdx.x & 63) % CPR) ^ swz(r)) * 16u;
        y.sum = y.chunk < bytes ? y.row + y.chunk : PAST;
        return y;
    }
    // Rows [0, ROWS) of a tile from global rows `stride` bytes apart, `valid` of them and `bytes` of each there.  Steps lie
    // whole swizzle periods apart where a step has 16 rows and more, and share a thread's offset.
    template <int ROWS, int WAVES>
    __device__ static __forceinline__ void fill(char* lds, const T* base, uint32_t stride, int valid, uint32_t bytes,
                                                const Lay& y) {
        constexpr int SR = RPW * WAVES, STEPS = ROWS / SR;
        static_assert(STEPS * SR == ROWS, "a tile is filled by whole wave loads");
        const int wave = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const uint32_t skip = (uint32_t)(s * SR) * stride;
            const int records = valid > s * SR ? (int)((uint32_t)(valid - 1 - s * SR) * stride + bytes) : 0;
            const auto rs = __builtin_amdgcn_make_buffer_rsrc((char*)base + skip, 0, records, 0x00027000);
            uint32_t at = y.sum;
            if constexpr (SR % 16 != 0) {
                const uint32_t c = y.chunk ^ (uint32_t)(swz(s * SR) << 4);
                at = c < bytes ? y.row + c : PAST;
            }
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, TAGAN_LDS(void, lds + (s * WAVES + wave) * 1024), 16, (int)at, 0,
                                                     0, 0);
        }
    }
    // The same of packed rows (token, head of the group), at offsets that `spot` gives for each row of the tile.
    template <int ROWS, int WAVES, class Spot>
    __device__ static __forceinline__ void fill_rows(char* lds, const T* base, uint32_t span, uint32_t bytes, Spot spot) {
        constexpr int SR = RPW * WAVES, STEPS = ROWS / SR;
        static_assert(STEPS * SR == ROWS, "a tile is filled by whole wave loads");
        const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)span, 0x00027000);
        const int wave = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int r = s * SR + (WAVES == 1 ? 0 : (int)threadIdx.x >> 6) * RPW + (threadIdx.x & 63) / CPR;
            const uint32_t c = (uint32_t)(((threadIdx.x & 63) % CPR) ^ swz(r)) * 16u, at = spot(s, r);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, TAGAN_LDS(void, lds + (s * WAVES + wave) * 1024), 16,
                                                     (int)(at != PAST && c < bytes ? at + c : PAST), 0, 0, 0);
        }
    }

    // Where a lane reads, for row (or run) 0 of a tile.  swz is linear in the bits of the row and chunks are whole powers
    // of two, so every other address is one exclusive or with a constant and a constant offset; made anew for each tile,
    // these cost less than the registers that all addresses would take over the loop.
    struct At {
        int row, col;
    };
    __device__ static __forceinline__ At at() {
        int l = threadIdx.x & 63;
        asm volatile("" : "+v"(l));                      // not kept over the loop
        const int h = l >> 5;
        At p;
        if constexpr (sizeof(T) == 2) {
            // transposed: a lane addresses 4 features of one row; within 16 lanes the 4 x 16 block comes back transposed
            const int s = l & 15, r = 4 * h + (s >> 2);
            p.row = (l & 31) * ROW + ((h ^ swz(l & 31)) << 4);
            p.col = r * ROW + (((((l & 16) >> 3) + ((s & 3) >> 1)) ^ swz(r)) << 4) + (s & 1) * 8;
        } else {
            p.row = (l & 31) * ROW + (((2 * h) ^ swz(l & 31)) << 4);
            p.col = 4 * h * ROW + ((((l & 31) >> 2) ^ swz(4 * h)) << 4) + (l & 3) * 4;
        }
        return p;
    }
    // operand of rows row0 + l % 32, features 16 c + 8 (l / 32) .. + 7
    __device__ static __forceinline__ void rows(Frag<T>& f, const char* lds, At p, int row0, int c) {
        if constexpr (sizeof(T) == 2) {
            const uint4 u = *(const uint4*)(lds + (p.row ^ (c << 5)) + row0 * ROW);
            f.u[0] = u.x; f.u[1] = u.y; f.u[2] = u.z; f.u[3] = u.w;
        } else {
            const float4 a = *(const float4*)(lds + (p.row ^ (c << 6)) + row0 * ROW);
            const float4 b = *(const float4*)(lds + (p.row ^ (c << 6) ^ 16) + row0 * ROW);
            f.v[0] = a.x; f.v[1] = a.y; f.v[2] = a.z; f.v[3] = a.w;
            f.v[4] = b.x; f.v[5] = b.y; f.v[6] = b.z; f.v[7] = b.w;
        }
    }
    // transposed operand: features 32 db + l % 32, rows row0 + 4 h + j % 4 + 8 (j / 4)
    __device__ static __forceinline__ void cols(Frag<T>& f, char* lds, At p, int row0, int db) {
        if constexpr (sizeof(T) == 2) {
            char* a = lds + (p.col ^ (db << 6)) + row0 * ROW;
            char* b = lds + (p.col ^ (db << 6) ^ (swz(8) << 4)) + (row0 + 8) * ROW;
            f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(TAGAN_LDS(s16x4, a));
            f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(TAGAN_LDS(s16x4, b));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = (j & 3) + 8 * (j >> 2);
                f.v[j] = *(const float*)(lds + (p.col ^ (db << 7) ^ (swz(r) << 4)) + (row0 + r) * ROW);
            }
        }
    }
};

// Infinities and NaN among the values of a tile of which some row sees only a part: 0 * inf in the product would carry
// them into rows that do not see them.  Such a tile is multiplied with zeros in their place, and after the last tile
// each row adds those that it does see (any weight times an infinity is that infinity).  Elsewhere a weight that is zero
// in fp32 makes NaN of it: either way a row that sees such a value is not finite there.
__device__ __forceinline__ bool wild(float v) { return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u; }
template <typename T>
__device__ __forceinline__ bool tame(uint32_t& w) {
    const uint32_t was = w;
    if (wild(__uint_as_float(w))) w = sizeof(T) == 2 ? w & 0x0000ffffu : 0u;
    if (sizeof(T) == 2 && wild(__uint_as_float(w << 16))) w &= 0xffff0000u;
    return w != was;
}
// the whole workgroup: whether a tile had any, and zeros in their place
template <typename T, int BYTES, int WAVES>
__device__ __forceinline__ bool tame_tile(char* lds) {
    bool any = false;
#pragma unroll 1
    for (int at = threadIdx.x * 16; at < BYTES; at += WAVES * 1024) {
        uint4 u = *(const uint4*)(lds + at);
        const bool x = tame<T>(u.x), y = tame<T>(u.y), z = tame<T>(u.z), w = tame<T>(u.w);
        if (x || y || z || w) {
            *(uint4*)(lds + at) = u;
            any = true;
        }
    }
    return __syncthreads_or(any) != 0;
}
__device__ __forceinline__ float as_float(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float as_float(float v) { return v; }

// every direct load of this wave has arrived, then of the workgroup
__device__ __forceinline__ void tiles_ready() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

__device__ __forceinline__ float half_max(float x) {
    float a, b;
    swap32(x, a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float half_sum(float x) {
    float a, b;
    swap32(x, a, b);
    return a + b;
}

// ------------------------------------------------------------------------------------------------ sequences
struct Strides {
    int64_t b, tok, head;   // elements
};

// n / d by a multiplication for n < 2^31: m = ceil(2^(31 + l) / d), l = ceil(log2 d), is off by less than 2^l / d <= 2
// parts of n / 2^(31 + l) < 2^-l <= 1 / d
struct Div {
    uint32_t d, m;
    int l;
};
Div div_by(int64_t d) {
    Div v = {(uint32_t)d, 0u, 0};
    while ((1ll << v.l) < d) ++v.l;
    v.m = (uint32_t)(((1ull << (31 + v.l)) + (uint64_t)d - 1) / (uint64_t)d);
    return v;
}
__device__ __forceinline__ int quot(int n, const Div& v) {
    return (int)(((uint64_t)(uint32_t)n * v.m) >> (31 + v.l));
}

struct AttnArgs {
    const void *q, *k, *v, *o, *dout;
    void *out, *dq, *dk, *dv;
    uint16_t* rest;     // bf16 training: out in 32 bits minus out, [nq, heads, dim]
    float* lse;
    float2* stat;       // backward: (log-sum-exp, rowsum(dO O)) of each row
    Strides qs, ks, vs, os, dos, dqs, dks, dvs;
    const int32_t *offs_q, *offs_k;   // packed: [n_seq + 1]; null: a cache
    const int32_t* lens;              // cache: [batch] keys of each
    int64_t nq, nk;                   // packed: tokens in all; cache: new tokens and capacity of each
    int32_t n_seq, heads, kv_heads, G, dim, causal, splits, ranked, key_blocks;
    Div by_g, by_kv, by_splits, by_tiles;   // of the group, the key heads, the splits, a cache's tiles to a sequence
    float c;                          // scale * log2(e)
    float scale;
    float* part;                      // splits: sums [token][head][split][D], then (base, total) of each
    int64_t part_rows;                // tokens times heads
};

// One sequence and where its rows lie.  Rows outside every sequence belong to two more that see no key (the run before
// the first offset and the run behind the last), so they get zeros.
struct Seq {
    int q0, k0;        // first token, first key
    int lq, lk, index;
    int past;          // keys before the first query's own; of a cache by its length, fit or not
    int tile;          // tile of this sequence
};

__device__ __forceinline__ int edge(const int32_t* offs, int n_seq, int n, int i) {
    if (i == 0) return 0;
    if (i == n_seq + 2) return n;
    return max(0, min(n, offs[i - 1]));
}

// The sequence of virtual tile vt, its first token and its length: sequence i starts at floor(edge_i * mul / tile) + i,
// which leaves each room for ceil(length * mul / tile) tiles.  64 probes to a step of the search; the last step's probes
// are neighbours and hold both edges.
struct Found {
    int i, begin, length, start;
};
__device__ __forceinline__ Found find_seq(const int32_t* offs, int n_seq, int n, int mul, int tile, int vt) {
    int lo = 0, count = n_seq + 2, hit, e;
    for (;;) {
        const int step = (count + 63) / 64;
        const int i = lo + (int)(threadIdx.x & 63) * step;
        e = edge(offs, n_seq, n, min(i, n_seq + 2));
        hit = max(1, (int)__popcll(__ballot(i < lo + count && e * mul / tile + i <= vt)));
        if (step == 1) break;
        count = min(step, count - (hit - 1) * step);
        lo += (hit - 1) * step;
    }
    Found f;
    f.i = __builtin_amdgcn_readfirstlane(lo + hit - 1);
    f.begin = __builtin_amdgcn_readlane(e, hit - 1);
    const int end = hit < 64 ? __builtin_amdgcn_readlane(e, hit & 63) : edge(offs, n_seq, n, f.i + 1);
    f.length = __builtin_amdgcn_readfirstlane(end) - f.begin;
    f.start = f.begin * mul / tile + f.i;
    return f;
}

// Heaviest tiles first.  With up to 62 sequences (and the two runs outside them) a lane keeps one of them, and every
// block finds its own tile: the rank-th in falling order of work, by bisection on the work W.  at_least(W) counts the tiles
// of the lane's sequence whose work is at least W: its first ones, for no tile has more than the one before.
// A long sequence whose tiles begin last costs the launch a fifth of its time (six histories of 1188 to 4096 tokens, dK
// and dV: 782 us against 640); the 20 wave sums are a few per cent of a long block, so only launches of few blocks do it,
// and the row kernels, whose blocks are shorter, lost 8 % by it (13 prompts of 5 to 2500, longest last, first or in the
// middle: 243, 253 and 247 us).
constexpr int ORDERED = 62;
__device__ __forceinline__ int wave_sum_int(int x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int wave_max_int(int x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x = max(x, __shfl_xor(x, o, 64));
    return __builtin_amdgcn_readfirstlane(x);
}
// most: no tile has more work
template <class AtLeast>
__device__ __forceinline__ bool ranked(int rank, int most, AtLeast at_least, int& seq, int& tile) {
    int lo = 0, hi = most + 1;                 // count(lo) > rank >= count(hi)
    if (wave_sum_int(at_least(0)) <= rank) return false;
    int above = 0;
    while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2, n = wave_sum_int(at_least(mid));
        if (n > rank) lo = mid;
        else {
            hi = mid;
            above = n;
        }
    }
    // the tiles of work lo exactly: in order of the sequences, those of one in order of their numbers
    const int n_hi = at_least(hi), n = at_least(lo) - n_hi;
    int before = n;                            // inclusive sum over the lanes
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(before, o, 64);
        if (lane >= o) before += up;
    }
    const int left = rank - above;
    seq = __ffsll((long long)__ballot(before > left)) - 1;
    tile = __shfl(n_hi, seq, 64) + left - __shfl(before - n, seq, 64);
    seq = __builtin_amdgcn_readfirstlane(seq);
    tile = __builtin_amdgcn_readfirstlane(tile);
    return true;
}

// rows of a query tile: sequence, false where the tile is none
template <int ROWS>
__device__ __forceinline__ bool locate(const AttnArgs& A, int vt, Seq& s) {
    if (A.offs_q == nullptr) {
        s.index = quot(vt, A.by_tiles);
        if (TAGAN_DBAD(s.index >= 0 && s.index < A.n_seq, s.index, A.n_seq)) return false;   // history of a tile
        s.tile = vt - s.index * (int)A.by_tiles.d;
        s.lq = (int)A.nq;
        s.q0 = s.k0 = 0;
        const int len = max(0, A.lens[s.index]);
        s.lk = min((int)A.nk, len);
        s.past = len - s.lq;
        return true;
    }
    const Found f = find_seq(A.offs_q, A.n_seq, (int)A.nq, A.G, ROWS, vt);
    s.q0 = f.begin;
    s.lq = f.length;
    s.tile = vt - f.start;
    if (s.lq <= 0 || s.tile < 0 || s.tile * ROWS >= s.lq * A.G) return false;   // below 0: offsets that descend
    s.index = 0;
    s.k0 = 0;
    s.lk = 0;
    if (f.i >= 1 && f.i <= A.n_seq) {
        if (A.offs_k == A.offs_q && A.nk == A.nq) {
            s.k0 = f.begin;
            s.lk = f.length;
        } else {
            s.k0 = edge(A.offs_k, A.n_seq, (int)A.nk, f.i);
            s.lk = max(0, edge(A.offs_k, A.n_seq, (int)A.nk, f.i + 1) - s.k0);
        }
    }
    s.past = s.lk - s.lq;
    // the sequence that the search found
    return !TAGAN_DBAD(s.q0 >= 0 && s.q0 + s.lq <= A.nq && s.k0 >= 0 && s.k0 + s.lk <= A.nk, s.q0, s.k0);
}

// The rows of a wave and what they see.  Counts of rows (tokens times the group) stay below 2^31.
struct Rows {
    int nrows, r0, row, token, g;
    bool mine;
    int see;                           // keys of this lane's row
    int most, least;                   // keys that some row of the block sees, and that all of its rows see
    int wave_most, wave_least;         // of the wave's 32 rows; wave_least is 0 where rows are missing
};
template <int ROWS>
__device__ __forceinline__ Rows rows_of(const AttnArgs& A, const Seq& sq) {
    const int lane = threadIdx.x & 63, wave = ROWS == 32 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    Rows R;
    R.nrows = sq.lq * A.G;
    R.r0 = sq.tile * ROWS;
    R.row = R.r0 + wave * 32 + (lane & 31);
    R.mine = R.row < R.nrows;
    R.token = quot(R.row, A.by_g);
    R.g = R.row - R.token * A.G;
    const auto keys = [&](int row) { return A.causal ? min(sq.lk, max(0, quot(row, A.by_g) + sq.past + 1)) : sq.lk; };
    R.see = !R.mine ? 0 : (A.causal ? min(sq.lk, max(0, R.token + sq.past + 1)) : sq.lk);
    R.most = keys(min(R.r0 + ROWS, R.nrows) - 1);
    R.least = keys(R.r0);
    const int w0 = R.r0 + wave * 32;
    R.wave_least = w0 + 31 >= R.nrows ? 0 : keys(w0);
    R.wave_most = w0 >= R.nrows ? 0 : keys(min(w0 + 32, R.nrows) - 1);
    return R;
}

// ------------------------------------------------------------------------------------------------ forward
template <typename T, int D, int WAVES>
struct Shape {
    // keys of a tile: 64; 32 for one-wave blocks and for 128 features, whose scores then leave the forward three waves to
    // a SIMD (ragged prompts 345 -> 315 us)
    static constexpr int LEAST = WAVES == 1 || D == 128 ? 32 : 64, ALL = Tile<T, D>::RPW * WAVES;
    static constexpr int KT = LEAST > ALL ? LEAST : ALL;   // a wave load at least to every wave
};

// A wave has 32 rows, a block WAVES times as many, and a tile of KT keys at a time.  A tile of 32 keys of 128 features costs
// a wave 16 matrix instructions of 32 cycles and about 75 vector ones, 16 of them exponentials: the two pipes are near
// balance.  One sequence of 16384 tokens, 16 heads over 2, bf16: 1.00 to 1.13 ms with the card's temperature (0.97 to 1.1
// PFLOP/s; a library product of that size reaches 1.38), matrix pipe busy 52 % of the cycles at 1.9 GHz, no LDS conflicts.
// Four waves share a tile: two waves lost 40 % to the tiles' traffic, eight gained nothing, a third stage lost 3 %.
// STAGES 2: the next tile arrives while this one is multiplied; 1 (short sequences, one-wave blocks): half the LDS, and as
// many more blocks of a CU hide each other's waits.
// FINE (bf16, batches of short histories: few_keys): each probability of a short one as two operands, its bf16 value and
// the rest.
template <typename T, int D, int WAVES, bool SPLIT, int STAGES, bool FINE = false>
__global__ void __launch_bounds__(WAVES * 64, sizeof(T) == 4 && D == 128 ? 1 : 3) k_attn_fwd(AttnArgs A) {
    constexpr int KT = Shape<T, D, WAVES>::KT, NB = KT / 32, NC = D / 16, ND = (D + 31) / 32, ROWS = 32 * WAVES;
    typedef Tile<T, D> TL;
    // two buffers, each an object of its own: reads of one do not wait for the loads of the other
    constexpr int SECOND = STAGES == 2 ? KT * TL::ROW + TL::PAD : 16;
    __shared__ __align__(16) char ks0[KT * TL::ROW + TL::PAD], ks1[SECOND];
    __shared__ __align__(16) char vs0[KT * TL::ROW + TL::PAD], vs1[SECOND];
    const int lane = threadIdx.x & 63, half = lane >> 5;
    int bid = blockIdx.x, split = 0, tiles = quot(gridDim.x, A.by_kv);
    if constexpr (SPLIT) {
        const int rest = quot(bid, A.by_splits);
        split = bid - rest * A.splits;
        bid = rest;
        tiles = quot(tiles, A.by_splits);
    }
    // key heads side by side (with 8 of them each XCD keeps to one), last tiles first: when causal they have the most keys
    const int vt = quot(bid, A.by_kv), hk = bid - vt * A.kv_heads;
    Seq sq;
    if (!locate<ROWS>(A, tiles - 1 - vt, sq)) return;
    const Rows R = rows_of<ROWS>(A, sq);
    int kbeg = 0, kend = R.most;
    if constexpr (SPLIT) {
        const int per = (quot(kend + A.splits - 1, A.by_splits) + KT - 1) / KT * KT;
        kbeg = min((int64_t)kend, (int64_t)split * per);
        kend = min((int64_t)kend, (int64_t)kbeg + per);
    }
    const T* Q = (const T*)A.q + (int64_t)sq.index * A.qs.b + (int64_t)(sq.q0 + R.token) * A.qs.tok +
                 (int64_t)(hk * A.G + R.g) * A.qs.head;
    const T* K = (const T*)A.k + (int64_t)sq.index * A.ks.b + (int64_t)sq.k0 * A.ks.tok + (int64_t)hk * A.ks.head;
    const T* V = (const T*)A.v + (int64_t)sq.index * A.vs.b + (int64_t)sq.k0 * A.vs.tok + (int64_t)hk * A.vs.head;
    const uint32_t bytes = (uint32_t)A.dim * sizeof(T), kstep = (uint32_t)(A.ks.tok * sizeof(T)),
                   vstep = (uint32_t)(A.vs.tok * sizeof(T));
    const auto klay = TL::template lay<WAVES>(kstep, bytes), vlay = TL::template lay<WAVES>(vstep, bytes);

    Frag<T> qf[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        qf[c].zero();
        if (R.mine && 16 * c + 8 * half < A.dim) load_frag(qf[c], Q + 16 * c + 8 * half);
    }
    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    float m = -INFINITY, base = 0.f, l = 0.f;   // largest score of the base, that in powers of two, sum over it

    const bool two = FINE && sq.lk <= SHORT;
    int wild_from = 0x7fffffff;                // first key of the tiles that were tamed
    const typename TL::At at = TL::at();
    const auto load = [&](char* kb, char* vb, int kt) __attribute__((always_inline)) {
        const int valid = min(KT, kend - kt);
        TL::template fill<KT, WAVES>(kb, K + (int64_t)kt * A.ks.tok, kstep, valid, bytes, klay);
        TL::template fill<KT, WAVES>(vb, V + (int64_t)kt * A.vs.tok, vstep, valid, bytes, vlay);
    };
    const auto tile = [&](char* ks, char* vs, int kt) __attribute__((always_inline)) {
        // with two operands in every tile, for the rest of a weight is zero or negative
        if ((two || min(kt + KT, kend) > R.least) && tame_tile<T, KT * TL::ROW, WAVES>(vs)) wild_from = min(wild_from, kt);
        if (kt >= R.wave_most) return;
        f32x16 s[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                Frag<T> kf;
                TL::rows(kf, ks, at, 32 * b, c);
                mma(s[b], kf, qf[c]);
            }
        const bool masked = kt + KT > R.wave_least || kt + KT > kend;
        if (masked) {
            const int lim = min(R.see, kend) - kt - 4 * half;   // keys of this lane below it are visible
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (32 * b + 8 * (i >> 2) + (i & 3) >= lim) s[b][i] = -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
        top = half_max(top);
        // The base of the exponents follows the maximum only where that has grown by more than LAZY powers of two
        // (or had none): weights up to 2^LAZY lose nothing in fp32 sums and bf16 operands, and most tiles then
        // leave the D / 2 output registers alone.
        if (__any(top * A.c > base + LAZY || (m == -INFINITY && top > -INFINITY))) {
            const float next = fmaxf(m, top);
            const float b2 = next == -INFINITY ? 0.f : next * A.c;
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(base - b2);
            m = next;
            base = b2;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
        }
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], A.c, -base));
                sum += s[b][i];
            }
        l += sum;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                Frag<T> pf;
                from_acc(pf, s[b], 8 * x);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    Frag<T> vf;
                    TL::cols(vf, vs, at, 32 * b + 16 * x, d);
                    mma(o[d], vf, pf);
                }
                if constexpr (FINE) {
                    if (!two) continue;
                    rest_of(pf, s[b], 8 * x);
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        Frag<T> vf;
                        TL::cols(vf, vs, at, 32 * b + 16 * x, d);
                        mma(o[d], vf, pf);
                    }
                }
            }
    };
    if constexpr (STAGES == 1) {
        for (int kt = kbeg; kt < kend; kt += KT) {
            __syncthreads();                            // every wave is done with the tile before
            load(ks0, vs0, kt);
            tiles_ready();
            tile(ks0, vs0, kt);
        }
    } else {
        if (kbeg < kend) load(ks0, vs0, kbeg);
        for (int kt = kbeg; kt < kend; kt += 2 * KT) {
            tiles_ready();                              // and every wave is done with the other buffer
            if (kt + KT < kend) load(ks1, vs1, kt + KT);
            tile(ks0, vs0, kt);
            if (kt + KT >= kend) break;
            tiles_ready();
            if (kt + 2 * KT < kend) load(ks0, vs0, kt + 2 * KT);
            tile(ks1, vs1, kt + KT);
        }
    }
#pragma unroll 1
    for (int key = wild_from; key < kend; ++key) {
        const T* value = V + (int64_t)key * A.vs.tok;
        const bool seen = key < R.see;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int at = 32 * d + 8 * (i >> 2) + 4 * half + (i & 3);
                const float x = seen && at < A.dim ? as_float(value[at]) : 0.f;
                if (wild(x)) o[d][i] += x;
            }
    }
    l = half_sum(l);
    if (!R.mine) return;
    if constexpr (SPLIT) {
        // unnormalised sums, and behind those of all rows the maxima (in powers of two) and totals; a row's splits together
        const int64_t at = (sq.index * A.nq + sq.q0 + R.token) * A.heads + hk * A.G + R.g;
        if (TAGAN_DBAD(at < A.part_rows && split < A.splits, at, split)) return;   // place in the workspace
        float* p = A.part + (at * A.splits + split) * D;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                store4(p + 32 * d + 2 * i + 4 * half, o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]);
        if (half == 0) {
            ((float2*)(A.part + A.part_rows * A.splits * D))[at * A.splits + split] = make_float2(base, l);
        }
    } else {
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        T* O = (T*)A.out + (int64_t)sq.index * A.os.b + (int64_t)(sq.q0 + R.token) * A.os.tok +
               (int64_t)(hk * A.G + R.g) * A.os.head;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int at = 32 * d + 2 * i + 4 * half;
                if (at < A.dim)
                    store4(O + at, o[d][i] * inv, o[d][i + 1] * inv, o[d][i + 2] * inv, o[d][i + 3] * inv);
            }
        if constexpr (sizeof(T) == 2) {
            if (A.rest) {
                uint16_t* rest = A.rest + ((int64_t)(sq.q0 + R.token) * A.heads + hk * A.G + R.g) * A.dim;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const int at = 32 * d + 2 * i + 4 * half;
                        float r[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float x = o[d][i + j] * inv;
                            r[j] = x - __uint_as_float(f2bf2(x, 0.f) << 16);
                        }
                        if (at < A.dim) store4(rest + at, r[0], r[1], r[2], r[3]);
                    }
            }
        }
        // +inf where no key is seen: exp2(s - lse) is 0 in the backward
        if (A.lse && half == 0)
            A.lse[(int64_t)(sq.q0 + R.token) * A.heads + hk * A.G + R.g] = l == 0.f ? INFINITY : base + __log2f(l);
    }
}

// A cache's keys are split over blocks that divide the length they find: 64 histories to 8000 tokens, 32 heads over 8, 128
// features, bf16, 1.08 GB of keys and values: 209 us, 5.2 TB/s (a copy reaches 4.7); two of 40 and 70 thousand, 24 rows in
// fp32: 45 us (2.9 TB/s; a wave's 128 fp32 matrix instructions to a tile take as long as its 32 KB).
//
// Joins the splits of a row, a workgroup to 32 features of a row and a thread to a split: the weights of all splits first,
// then the sums, with the splits dealt out to JT / 8 groups of 8 lanes whose partial sums are added in a fixed order.  No
// thread has more than 8 loads in a row, all independent (a chain over 256 splits took 200 us).
constexpr int MAX_SPLITS = 512;
template <typename T, int D, int JT>
__global__ void __launch_bounds__(JT) k_attn_join(AttnArgs A) {
    constexpr int JW = JT / 64, JG = JT / 8, CH = D / 32;
    __shared__ float w[JT], red[JW], tot[JW];
    __shared__ float4 sums[JW][8];
    const int64_t at = blockIdx.x / CH;
    const int ch = blockIdx.x % CH, s = threadIdx.x, wave = s >> 6, lane = s & 63;
    if (TAGAN_DBAD(at < A.part_rows, at, A.part_rows)) return;   // row of the workspace
    float2 ml = make_float2(-INFINITY, 0.f);
    if (s < A.splits) ml = ((const float2*)(A.part + A.part_rows * A.splits * D))[at * A.splits + s];
    const bool some = ml.y != 0.f;             // a split without a visible key has no base
    const float m = lane_max<64>(some ? ml.x : -INFINITY);
    if (lane == 0) red[wave] = m;
    __syncthreads();
    float top = red[0];
#pragma unroll
    for (int i = 1; i < JW; ++i) top = fmaxf(top, red[i]);
    const float x = some ? __builtin_amdgcn_exp2f(ml.x - top) : 0.f;
    w[s] = x;
    const float t = lane_sum<64>(some ? x * ml.y : 0.f);
    if (lane == 0) tot[wave] = t;
    __syncthreads();
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < JW; ++i) l += tot[i];
    const int f = s & 7, g = s >> 3;
    const float* p = A.part + at * A.splits * D + 32 * ch + 4 * f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int i = g; i < A.splits; i += JG) {
        // a split that the row does not see has zeros here; one whose weight is zero may hold an infinity that the row
        // does see, and 0 * inf tells so
        const float4 v = *(const float4*)(p + (int64_t)i * D);
        const float wi = w[i];
        o.x = fmaf(v.x, wi, o.x);
        o.y = fmaf(v.y, wi, o.y);
        o.z = fmaf(v.z, wi, o.z);
        o.w = fmaf(v.w, wi, o.w);
    }
#pragma unroll
    for (int d = 8; d < 64; d <<= 1) {
        o.x += __shfl_xor(o.x, d, 64);
        o.y += __shfl_xor(o.y, d, 64);
        o.z += __shfl_xor(o.z, d, 64);
        o.w += __shfl_xor(o.w, d, 64);
    }
    if (lane < 8) sums[wave][f] = o;
    __syncthreads();
    const int feature = 32 * ch + 4 * f;
    if (s >= 8 || feature >= A.dim) return;
#pragma unroll
    for (int i = 1; i < JW; ++i) {
        const float4 v = sums[i][f];
        o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    const int64_t token = at / A.heads, head = at - token * A.heads, b = token / A.nq;   // packed: one batch of nq tokens
    T* out = (T*)A.out + b * A.os.b + (token - b * A.nq) * A.os.tok + head * A.os.head;
    const float x4[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    store4(out + feature, x4[0], x4[1], x4[2], x4[3]);
    if (A.lse && s == 0 && ch == 0) A.lse[at] = l == 0.f ? INFINITY : top + __log2f(l);
    if constexpr (sizeof(T) == 2) {
        if (A.rest) {
            float r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = x4[j] - __uint_as_float(f2bf2(x4[j], 0.f) << 16);
            store4(A.rest + at * A.dim + feature, r[0], r[1], r[2], r[3]);
        }
    }
}

// ------------------------------------------------------------------------------------------------ backward
// (log-sum-exp, delta = rowsum(dO O)) of each row, D / 8 lanes to a row.  A short row's dP - delta is a small difference
// of large terms: delta takes out to 16 bits and more (its bf16 value and the rest that the forward kept).  Bound by
// memory: 15850 tokens of 16 heads of 128, 195 MB: 31 us (6.3 TB/s, part of it from the caches).
template <typename T, int D>
__global__ void __launch_bounds__(256) k_attn_stat(AttnArgs A) {
    constexpr int L = D / 8;
    const int64_t at = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const int x = threadIdx.x % L * 8;
    if (at >= A.nq * A.heads) return;
    const int64_t token = at / A.heads, head = at - token * A.heads;
    float sum = 0.f;
    if (x < A.dim) {
        Frag<T> g, o;
        load_frag(g, (const T*)A.dout + token * A.dos.tok + head * A.dos.head + x);
        load_frag(o, (const T*)A.o + token * A.os.tok + head * A.os.head + x);
        sum = dot(g, o);
        if constexpr (sizeof(T) == 2) {
            if (A.rest) {
                load_frag(o, A.rest + at * A.dim + x);
                sum += dot(g, o);
            }
        }
    }
    sum = lane_sum<L>(sum);
    if (x == 0) A.stat[at] = make_float2(A.lse[at], sum);
}

// Keys of a tile of the dQ blocks: at least as many as the direct loads of all waves bring
template <typename T, int D, int WAVES>
constexpr int dq_keys() {
    constexpr int KT = WAVES == 1 || (D == 128 && sizeof(T) == 4) ? 32 : 64, ALL = Tile<T, D>::RPW * WAVES;
    return KT > ALL ? KT : ALL;
}

// dQ: rows as in the forward.
template <typename T, int D, int WAVES, int STAGES, bool FINE>
__device__ __forceinline__ void attn_dq(const AttnArgs& A, int block, int blocks, char* ks0, char* ks1, char* vs0,
                                        char* vs1) {
    constexpr int KT = dq_keys<T, D, WAVES>(), NB = KT / 32, NC = D / 16, ND = (D + 31) / 32, ROWS = 32 * WAVES;
    typedef Tile<T, D> TL;
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const int vt = quot(block, A.by_kv), hk = block - vt * A.kv_heads;
    Seq sq;
    if (!locate<ROWS>(A, quot(blocks, A.by_kv) - 1 - vt, sq)) return;
    const Rows R = rows_of<ROWS>(A, sq);
    const int kend = R.most;
    const bool two = FINE && sq.lk <= SHORT;
    const int64_t head = hk * A.G + R.g, tok = sq.q0 + R.token;
    const T* Q = (const T*)A.q + tok * A.qs.tok + head * A.qs.head;
    const T* DO = (const T*)A.dout + tok * A.dos.tok + head * A.dos.head;
    const T* K = (const T*)A.k + (int64_t)sq.k0 * A.ks.tok + (int64_t)hk * A.ks.head;
    const T* V = (const T*)A.v + (int64_t)sq.k0 * A.vs.tok + (int64_t)hk * A.vs.head;
    const uint32_t bytes = (uint32_t)A.dim * sizeof(T), kstep = (uint32_t)(A.ks.tok * sizeof(T)),
                   vstep = (uint32_t)(A.vs.tok * sizeof(T));
    const auto klay = TL::template lay<WAVES>(kstep, bytes), vlay = TL::template lay<WAVES>(vstep, bytes);

    Frag<T> qf[NC], gf[NC];
    float lse = INFINITY, delta = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        qf[c].zero();
        gf[c].zero();
        if (R.mine && 16 * c + 8 * half < A.dim) {
            load_frag(qf[c], Q + 16 * c + 8 * half);
            load_frag(gf[c], DO + 16 * c + 8 * half);
        }
    }
    if (R.mine) {
        const float2 stat = A.stat[tok * A.heads + head];
        lse = stat.x;
        delta = stat.y;
    }
    f32x16 dq[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) dq[d][i] = 0.f;

    const typename TL::At at = TL::at();
    const auto load = [&](char* kb, char* vb, int kt) __attribute__((always_inline)) {
        const int valid = min(KT, kend - kt);
        TL::template fill<KT, WAVES>(kb, K + (int64_t)kt * A.ks.tok, kstep, valid, bytes, klay);
        TL::template fill<KT, WAVES>(vb, V + (int64_t)kt * A.vs.tok, vstep, valid, bytes, vlay);
    };
    const auto tile = [&](char* ks, char* vs, int kt) __attribute__((always_inline)) {
        if (kt >= R.wave_most) return;
        const bool masked = kt + KT > R.wave_least;
        const int lim = R.see - kt - 4 * half;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = dp[i] = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                Frag<T> kf, vf;
                TL::rows(kf, ks, at, 32 * b, c);
                mma(s, kf, qf[c]);
                TL::rows(vf, vs, at, 32 * b, c);
                mma(dp, vf, gf[c]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[i], A.c, -lse));
                s[i] = p * (dp[i] - delta);
            }
            if (masked) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (32 * b + 8 * (i >> 2) + (i & 3) >= lim) s[i] = 0.f;
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                Frag<T> pf;
                from_acc(pf, s, 8 * x);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    Frag<T> kf;
                    TL::cols(kf, ks, at, 32 * b + 16 * x, d);
                    mma(dq[d], kf, pf);
                }
                if constexpr (FINE) {
                    if (!two) continue;
                    rest_of(pf, s, 8 * x);
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        Frag<T> kf;
                        TL::cols(kf, ks, at, 32 * b + 16 * x, d);
                        mma(dq[d], kf, pf);
                    }
                }
            }
        }
    };
    if constexpr (STAGES == 1) {
        for (int kt = 0; kt < kend; kt += KT) {
            __syncthreads();
            load(ks0, vs0, kt);
            tiles_ready();
            tile(ks0, vs0, kt);
        }
    } else {
        if (kend > 0) load(ks0, vs0, 0);
        for (int kt = 0; kt < kend; kt += 2 * KT) {
            tiles_ready();
            if (kt + KT < kend) load(ks1, vs1, kt + KT);
            tile(ks0, vs0, kt);
            if (kt + KT >= kend) break;
            tiles_ready();
            if (kt + 2 * KT < kend) load(ks0, vs0, kt + 2 * KT);
            tile(ks1, vs1, kt + KT);
        }
    }
    if (!R.mine) return;
    T* DQ = (T*)A.dq + tok * A.dqs.tok + head * A.dqs.head;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int at = 32 * d + 2 * i + 4 * half;
            if (at < A.dim)
                store4(DQ + at, dq[d][i] * A.scale, dq[d][i + 1] * A.scale, dq[d][i + 2] * A.scale,
                       dq[d][i + 3] * A.scale);
        }
}

// ------------------------------------------------------------------------------------------------ backward: dK, dV
// dK, dV.  A wave has 32 keys (in its lanes); WK waves side by side have the block's keys and WR of them share the
// rows that see those keys, 32 rows of every tile to each.  The WR partial sums are added in LDS, in order.  Splitting the rows inside
// the block is what bounds the longest block: the first keys of a long causal sequence are seen by every row of the group.
template <typename T, int D, int WK, int WR>
constexpr int dkv_rows() {          // rows of a tile: 32 to a row wave, and enough for a chunk to every lane of the loads
    constexpr int LEAST = 1024 * WK * WR / Tile<T, D>::ROW;
    return 32 * WR > LEAST ? 32 * WR : LEAST;
}
template <typename T, int D, int WK, int WR, int STAGES, bool FINE>
__device__ __forceinline__ void attn_dkv(const AttnArgs& A, int block, char* qs0, char* gs0, char* qs1, char* gs1,
                                         char* st0, char* st1, char* vl) {
    typedef Tile<T, D> TL;
    constexpr int WAVES = WK * WR, NC = D / 16, ND = (D + 31) / 32, KEYS = 32 * WK;
    constexpr int QT = dkv_rows<T, D, WK, WR>(), TILE = QT * TL::ROW;
    constexpr bool VL = D == 128;   // the keys' own v: in LDS where the accumulators and k leave no registers for it
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, wk = wave % WK, wr = wave / WK;
    const int vt = quot(block, A.by_kv), hk = block - vt * A.kv_heads, nk = (int)A.nk;
    int i, tile, k0, lk;
    if (A.ranked) {
        int slq = 0, slk = 0;
        if (lane < A.n_seq + 2) {
            slk = max(0, edge(A.offs_k, A.n_seq, nk, lane + 1) - edge(A.offs_k, A.n_seq, nk, lane));
            if (lane >= 1 && lane <= A.n_seq)
                slq = max(0, edge(A.offs_q, A.n_seq, (int)A.nq, lane + 1) - edge(A.offs_q, A.n_seq, (int)A.nq, lane));
        }
        const int tiles = (slk + KEYS - 1) / KEYS, most = wave_max_int(slq);
        // tile t is seen by lq - max(0, t KEYS - past) tokens (all of them when not causal), 0 at least
        const bool found = ranked(vt, most, [&](int w) {
            if (w <= 0) return tiles;
            if (slq < w) return 0;
            const int span = slk - w;          // lq - w + past
            return !A.causal ? tiles : span < 0 ? 0 : min(tiles, span / KEYS + 1);
        }, i, tile);
        if (!found) return;
        k0 = edge(A.offs_k, A.n_seq, nk, i);
        lk = edge(A.offs_k, A.n_seq, nk, i + 1) - k0;
    } else {
        const Found f = find_seq(A.offs_k, A.n_seq, nk, 1, KEYS, vt);
        i = f.i;
        tile = vt - f.start;
        k0 = f.begin;
        lk = f.length;
    }
    const int key0 = tile * KEYS;
    if (lk <= 0 || tile < 0 || key0 >= lk) return;   // below 0: offsets that descend
    int q0 = 0, lq = 0;
    if (i >= 1 && i <= A.n_seq) {
        const bool same = A.offs_k == A.offs_q && A.nk == A.nq;
        q0 = same ? k0 : edge(A.offs_q, A.n_seq, (int)A.nq, i);
        lq = same ? lk : max(0, edge(A.offs_q, A.n_seq, (int)A.nq, i + 1) - q0);
    }
    if (TAGAN_DBAD(k0 >= 0 && k0 + lk <= nk && q0 >= 0 && q0 + lq <= A.nq, k0, q0)) return;   // what the search found
    const int G = A.G, past = lk - lq, key = key0 + wk * 32 + (lane & 31);
    const bool mine = key < lk;
    const uint32_t bytes = (uint32_t)A.dim * sizeof(T);
    const T* K = (const T*)A.k + (int64_t)(k0 + key) * A.ks.tok + (int64_t)hk * A.ks.head;
    const T* V = (const T*)A.v + (int64_t)(k0 + key) * A.vs.tok + (int64_t)hk * A.vs.head;
    Frag<T> kf[NC], vf[VL ? 1 : NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        kf[c].zero();
        if constexpr (!VL) vf[c].zero();
        if (mine && 16 * c + 8 * half < A.dim) {
            load_frag(kf[c], K + 16 * c + 8 * half);
            if constexpr (!VL) load_frag(vf[c], V + 16 * c + 8 * half);
        }
    }
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int x = 0; x < 16; ++x) dk[d][x] = dv[d][x] = 0.f;

    // Tiles of whole tokens, so that a row's (token, head of the group) is the same in every tile and its offset is kept:
    // QT / G tokens; groups wider than a tile take as many tiles to a token, the last of them part empty.
    const bool wide = G > QT;
    const int tokens = wide ? 1 : QT / G, pieces = wide ? (G + QT - 1) / QT : 1;
    const uint32_t qtok = (uint32_t)(A.qs.tok * sizeof(T)), qhead = (uint32_t)(A.qs.head * sizeof(T)),
                   gtok = (uint32_t)(A.dos.tok * sizeof(T)), ghead = (uint32_t)(A.dos.head * sizeof(T));
    constexpr int SR = TL::RPW * WAVES, STEPS = QT / SR;
    uint32_t qat[STEPS], gat[STEPS];
    int rt[STEPS];                                     // token of the row in a tile; many where the row is none
    const int myrow = (WAVES == 1 ? 0 : (int)threadIdx.x >> 6) * TL::RPW + (threadIdx.x & 63) / TL::CPR;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int r = myrow + s * SR, t = wide ? 0 : quot(r, A.by_g), g = r - t * G;
        rt[s] = t < tokens ? t : 1 << 30;
        qat[s] = t < tokens ? (uint32_t)t * qtok + (uint32_t)g * qhead : TL::PAST;
        gat[s] = t < tokens ? (uint32_t)t * gtok + (uint32_t)g * ghead : TL::PAST;
    }
    // (log-sum-exp, delta) of 32 rows to a wave
    const int srow = wave * 32 + (lane >> 1), stok = wide ? 0 : quot(srow, A.by_g);
    const uint32_t sat = ((uint32_t)stok * (uint32_t)A.heads + (uint32_t)(srow - stok * G)) * 8 + (lane & 1) * 4;
    static_assert(QT / 32 <= WAVES, "a wave loads the statistics of 32 rows");

    // tile n: tokens [t0, t0 + tokens), from head g0 of the group on
    const int tbeg = A.causal ? max(0, key0 - past) : 0;       // the first token that sees the block's first key
    const int ntiles = tbeg < lq ? (lq - tbeg + tokens - 1) / tokens * pieces : 0;
    const auto load = [&](char* qs, char* gs, char* st, int n) __attribute__((always_inline)) {
        const int step = wide ? n / pieces : n, t0 = tbeg + step * tokens, g0 = wide ? (n - step * pieces) * QT : 0;
        const int there = min(tokens, lq - t0), heads = min(QT, G - g0);       // tokens, and heads of a wide token
        const int64_t tok = q0 + t0, head = (int64_t)hk * G + g0;
        const bool part = wide ? heads < QT : there < tokens;
        const auto have = [&](int s, int r) __attribute__((always_inline)) {
            return !part || (wide ? r < heads : rt[s] < there);
        };
        const uint32_t qspan = (uint32_t)(there - 1) * qtok + (uint32_t)((wide ? heads : G) - 1) * qhead + bytes;
        const uint32_t gspan = (uint32_t)(there - 1) * gtok + (uint32_t)((wide ? heads : G) - 1) * ghead + bytes;
        TL::template fill_rows<QT, WAVES>(qs, (const T*)A.q + tok * A.qs.tok + head * A.qs.head, qspan, bytes,
                                          [&](int s, int r) __attribute__((always_inline)) {
                                              return have(s, r) ? qat[s] : TL::PAST;
                                          });
        TL::template fill_rows<QT, WAVES>(gs, (const T*)A.dout + tok * A.dos.tok + head * A.dos.head, gspan, bytes,
                                          [&](int s, int r) __attribute__((always_inline)) {
                                              return have(s, r) ? gat[s] : TL::PAST;
                                          });
        // zeros where a row is none: its q and dO are zeros, so the weight 1 that zeros give adds nothing
        if (wave < QT / 32) {
            const float2* base = A.stat + tok * A.heads + head;
            const auto rs = __builtin_amdgcn_make_buffer_rsrc(
                (void*)base, 0, ((there - 1) * A.heads + (wide ? heads : G)) * 8, 0x00027000);
            const bool is = stok < tokens && (wide ? srow < heads : stok < there);
            const int to = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(wave) * 256;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, TAGAN_LDS(void, st + to), 4, (int)(is ? sat : TL::PAST), 0, 0, 0);
        }
    };
    const auto part = [&](char* qs, char* gs, const char* st, int n, int q) __attribute__((always_inline)) {
        const typename TL::At at = TL::at();
        const int t0 = tbeg + (wide ? n / pieces : n) * tokens;
        const bool masked = A.causal && key0 + wk * 32 + 31 > t0 + past;
        // rows of this lane below it do not see its key; a wide token's rows are of one token
        const int lim = !masked ? -1 : wide ? (key > t0 + past ? QT : -1) : (key - past - t0) * G - q - 4 * half;
        f32x16 s, dp;
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] = dp[x] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            Frag<T> f;
            TL::rows(f, qs, at, q, c);
            mma(s, f, kf[c]);
            TL::rows(f, gs, at, q, c);
            if constexpr (VL) TL::rows(vf[0], vl, at, wk * 32, c);
            mma(dp, f, vf[VL ? 0 : c]);
        }
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
            const float4* sp = (const float4*)(st + (q + 2 * x + 4 * half) * 8);
            const float4 a = sp[0], b = sp[1];
            const float lx[4] = {a.x, a.z, b.x, b.z}, dx[4] = {a.y, a.w, b.y, b.w};
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[x + y], A.c, -lx[y]));
                s[x + y] = p;
                dp[x + y] = p * (dp[x + y] - dx[y]);
            }
        }
        if (masked) {
#pragma unroll
            for (int x = 0; x < 16; ++x)
                if (8 * (x >> 2) + (x & 3) < lim) s[x] = dp[x] = 0.f;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            Frag<T> pf, sf;
            from_acc(pf, s, 8 * x);
            from_acc(sf, dp, 8 * x);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                Frag<T> f;
                TL::cols(f, gs, at, q + 16 * x, d);
                mma(dv[d], f, pf);
                TL::cols(f, qs, at, q + 16 * x, d);
                mma(dk[d], f, sf);
            }
            if constexpr (FINE) {
                if (lk > SHORT) continue;
                rest_of(pf, s, 8 * x);
                rest_of(sf, dp, 8 * x);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    Frag<T> f;
                    TL::cols(f, gs, at, q + 16 * x, d);
                    mma(dv[d], f, pf);
                    TL::cols(f, qs, at, q + 16 * x, d);
                    mma(dk[d], f, sf);
                }
            }
        }
    };
    if constexpr (VL) {
        if (ntiles > 0)
            TL::template fill<KEYS, WAVES>(vl, (const T*)A.v + (int64_t)(k0 + key0) * A.vs.tok + (int64_t)hk * A.vs.head,
                                       (uint32_t)(A.vs.tok * sizeof(T)), min(KEYS, lk - key0), bytes,
                                       TL::template lay<WAVES>((uint32_t)(A.vs.tok * sizeof(T)), bytes));
    }
    const auto rows = [&](char* qs, char* gs, const char* st, int n) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < QT; q += 32 * WR) part(qs, gs, st, n, q + 32 * wr);
    };
    if constexpr (STAGES == 1) {
        for (int n = 0; n < ntiles; ++n) {
            __syncthreads();
            load(qs0, gs0, st0, n);
            tiles_ready();
            rows(qs0, gs0, st0, n);
        }
    } else {
        if (ntiles > 0) load(qs0, gs0, st0, 0);
        for (int n = 0; n < ntiles; n += 2) {
            tiles_ready();
            if (n + 1 < ntiles) load(qs1, gs1, st1, n + 1);
            rows(qs0, gs0, st0, n);
            if (n + 1 >= ntiles) break;
            tiles_ready();
            if (n + 2 < ntiles) load(qs0, gs0, st0, n + 2);
            rows(qs1, gs1, st1, n + 1);
        }
    }
    if constexpr (WR > 1) {
        // 64 lanes x 16 ND floats of a wave to a slot of the tiles: one tensor after the other
        constexpr int SLOT = 64 * 16 * ND * 4, PER = TILE / SLOT;
        static_assert(STAGES == 2 && 4 * PER >= (WR - 1) * WK, "the tiles hold the waves' sums");
        const auto slot = [&](int w) __attribute__((always_inline)) {
            const int n = (w - 1) * WK + wk, t = n / PER;
            return (float*)((t == 0 ? qs0 : t == 1 ? gs0 : t == 2 ? qs1 : gs1) + n % PER * SLOT) + 4 * lane;
        };
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            f32x16* acc = which == 0 ? dv : dk;
            __syncthreads();
            if (wr > 0) {
                float* at = slot(wr);
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int x = 0; x < 16; x += 4)
                        *(float4*)(at + (16 * d + x) * 64) =
                            make_float4(acc[d][x], acc[d][x + 1], acc[d][x + 2], acc[d][x + 3]);
            }
            __syncthreads();
            if (wr == 0) {
#pragma unroll
                for (int w = 1; w < WR; ++w) {
                    const float* at = slot(w);
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int x = 0; x < 16; x += 4) {
                            const float4 v = *(const float4*)(at + (16 * d + x) * 64);
                            acc[d][x] += v.x; acc[d][x + 1] += v.y; acc[d][x + 2] += v.z; acc[d][x + 3] += v.w;
                        }
                }
            }
        }
    }
    if (!mine || wr > 0) return;
    T* DK = (T*)A.dk + (int64_t)(k0 + key) * A.dks.tok + (int64_t)hk * A.dks.head;
    T* DV = (T*)A.dv + (int64_t)(k0 + key) * A.dvs.tok + (int64_t)hk * A.dvs.head;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
            const int at = 32 * d + 2 * x + 4 * half;
            if (at < A.dim) {
                store4(DK + at, dk[d][x] * A.scale, dk[d][x + 1] * A.scale, dk[d][x + 2] * A.scale,
                       dk[d][x + 3] * A.scale);
                store4(DV + at, dv[d][x], dv[d][x + 1], dv[d][x + 2], dv[d][x + 3]);
            }
        }
}

// waves to a SIMD that the accumulators and k, v leave room for
template <typename T, int D, int WK>
constexpr int bwd_waves() {
    return D * sizeof(T) == 512 ? 1 : D == 16 && WK == 1 ? 4 : 2;
}
// Both in one launch, the key blocks first: they are the longer ones, and the row blocks fill the CUs that they leave.
// Six histories to 4096 tokens, 16 heads over 4, 128 features, bf16: 0.84 to 0.92 ms for seven products (two are made
// twice so that no sum needs atomics), 0.75 to 0.82 PFLOP/s; apart they took 0.99.  1200 fp32 histories to 64 tokens, 8
// heads of 16: 89 us, matrix pipe busy 45 %.
template <typename T, int D, int WK, int WR, int STAGES, bool FINE>
__global__ void __launch_bounds__(WK* WR * 64, (bwd_waves<T, D, WK>())) k_attn_bwd(AttnArgs A) {
    typedef Tile<T, D> TL;
    constexpr int WAVES = WK * WR, QT = dkv_rows<T, D, WK, WR>(), KT = dq_keys<T, D, WAVES>();
    constexpr int TILE = (QT > KT ? QT : KT) * TL::ROW + TL::PAD, SECOND = STAGES == 2 ? TILE : 16;
    __shared__ __align__(16) char qs0[TILE], gs0[TILE], qs1[SECOND], gs1[SECOND], st0[QT * 8], st1[QT * 8];
    __shared__ __align__(16) char vl[D == 128 ? 32 * WK * TL::ROW : 16];
    const int block = (int)blockIdx.x;
    if (block < A.key_blocks) attn_dkv<T, D, WK, WR, STAGES, FINE>(A, block, qs0, gs0, qs1, gs1, st0, st1, vl);
    else attn_dq<T, D, WAVES, STAGES, FINE>(A, block - A.key_blocks, (int)gridDim.x - A.key_blocks, qs0, qs1, gs0, gs1);
}

// ------------------------------------------------------------------------------------------------ launches
constexpr int MAX_DIM = 128, MAX_GROUP = 512;
constexpr int64_t MAX_TOKENS = 0x7fffffff - 1024;   // a tile's end behind the last one is counted in 31 bits
constexpr int64_t MAX_ROWS = 1ll << 40;             // tokens times heads: 16 TB of the smallest; their bytes stay in 64 bits

bool aligned(const void* p, int64_t a, int64_t b, int64_t c, int es) {
    return !((uintptr_t)p & 15) && (a * es) % 16 == 0 && (b * es) % 16 == 0 && (c * es) % 16 == 0;
}

int check_shape(const char* what, int dtype, int64_t heads, int64_t kv_heads, int32_t dim, float scale) {
    TAGAN_REQUIRE(dtype == TAGAN_F32 || dtype == TAGAN_BF16, TAGAN_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
    TAGAN_REQUIRE(kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0 && heads / kv_heads <= MAX_GROUP,
                  TAGAN_ERR_ARG, "%s: %lld heads over %lld key heads (a multiple, up to %d)", what, (long long)heads,
                  (long long)kv_heads, MAX_GROUP);
    TAGAN_REQUIRE(dim >= 8 && dim <= MAX_DIM && dim % 8 == 0, TAGAN_ERR_UNSUPPORTED,
                  "%s: head_dim %d (a multiple of 8 up to %d)", what, dim, MAX_DIM);
    // scale log2(e) has to be a finite fp32 number too
    TAGAN_REQUIRE(scale >= 0x1p-126f && scale <= 0x1p127f, TAGAN_ERR_ARG, "%s: scale has to lie in 2^-126 to 2^127", what);
    return TAGAN_OK;
}

// Strides that a tile's 32-bit offsets and 16-byte loads can take.  An axis of one step is never stepped over: its stride
// is anything.
int check_tensor(const char* what, const char* name, const void* p, Strides& s, int64_t nb, int64_t nt, int64_t nh,
                 int32_t dim, int es) {
    TAGAN_REQUIRE(p, TAGAN_ERR_ARG, "%s: %s is null", what, name);
    if (nb <= 1) s.b = 0;
    if (nt <= 1) s.tok = dim;
    if (nh <= 1) s.head = dim;
    TAGAN_REQUIRE(aligned(p, s.b, s.tok, s.head, es), TAGAN_ERR_ARG,
                  "%s: %s has to lie on 16 bytes, its strides too", what, name);
    TAGAN_REQUIRE(s.tok >= dim && s.tok <= (1 << 21) && s.head >= 0 && s.head <= (1ll << 40) && s.b >= 0, TAGAN_ERR_ARG,
                  "%s: %s has token stride %lld, head stride %lld", what, name, (long long)s.tok, (long long)s.head);
    return TAGAN_OK;
}

#define TAGAN_BY_DIM(T, dim, F)                                    \
    ((dim) <= 32 ? F<T, 32> : (dim) <= 64 ? F<T, 64> : F<T, 128>)
// with a tile of its own for the framework's 16 features, half the products of 32
#define TAGAN_BY_DIM16(T, dim, F) ((dim) <= 16 ? F<T, 16> : TAGAN_BY_DIM(T, dim, F))

// bf16, up to 64 keys to an average history: the FINE kernels, which take each probability and each gradient of a score as
// two operands in histories of up to 128 keys (and as one in a longer one beside them).  The roundings of few terms do not
// average out, and dP - rowsum(dO O) is a small difference that the forward's probabilities enter.  Errors over that of one
// rounding of the result, out / dQ / dK / dV, one operand and two: 240 histories of 1 to 4 tokens, 8 heads of 16: 1.08 /
// 1.51 / 1.51 / 1.21 and 1.00 each; single dQ and dK of the smallest batches 2.4 and 1.00; at 100 keys one operand gives
// 1.20 / 1.45 / 1.44 / 1.36, at 300 1.25 / 1.45 / 1.44 / 1.38.  Times: 1200 histories to 64 tokens, 8 heads of 16: forward 23
// and 25 us, backward 64 and 69; 16 heads over 4 of 64: 58 and 60, 239 and 258; 400 of 50 tokens, 32 heads over 4 of 128:
// 110 and 113, 412 and 451.  The same choice in the kernels of long batches cost those 2 % (128 features, six histories to
// 4096) to 14 % (16 features, 16 of 1000).
bool few_keys(const AttnArgs& A) { return A.nk <= (int64_t)64 * A.n_seq; }

// a launch counts its threads in 32 bits
bool fits_grid(int64_t blocks, int64_t threads) { return blocks <= 0xffffffffll / threads && blocks <= 0x7fffffff; }

template <typename T, int D, int WK, int WR, int STAGES>
int launch_bwd(AttnArgs A, hipStream_t s) {
    const int64_t keys = A.nk > 0 ? (A.nk / (32 * WK) + A.n_seq + 2) * A.kv_heads : 0;
    const int64_t rows = A.nq > 0 ? (A.nq * A.G / (32 * WK * WR) + A.n_seq + 2) * A.kv_heads : 0;
    TAGAN_REQUIRE(fits_grid(keys + rows, 64 * WK * WR), TAGAN_ERR_UNSUPPORTED, "packed_attn_bwd: too many tiles");
    A.ranked = A.n_seq >= 2 && A.n_seq <= ORDERED && keys < 16 * 256;
    A.key_blocks = (int32_t)keys;
    bool fine = false;
    if constexpr (sizeof(T) == 2) {
        fine = few_keys(A);
        if (fine) k_attn_bwd<T, D, WK, WR, STAGES, true><<<(unsigned)(keys + rows), 64 * WK * WR, 0, s>>>(A);
    }
    if (!fine) k_attn_bwd<T, D, WK, WR, STAGES, false><<<(unsigned)(keys + rows), 64 * WK * WR, 0, s>>>(A);
    TAGAN_CHECK_LAUNCH("packed_attn_bwd");
    return TAGAN_OK;
}

template <typename T, int D>
int run_bwd(const AttnArgs& A, hipStream_t s) {
    if (A.nq > 0) {
        const int64_t blocks = (A.nq * A.heads + 2048 / D - 1) / (2048 / D);
        TAGAN_REQUIRE(fits_grid(blocks, 256), TAGAN_ERR_UNSUPPORTED, "packed_attn_bwd: too many rows");
        k_attn_stat<T, D><<<(unsigned)blocks, 256, 0, s>>>(A);
        TAGAN_CHECK_LAUNCH("packed_attn_bwd (row sums)");
    }
    // One-wave blocks where a sequence has few rows and keys.  Two row waves where blocks are few and the longest of them
    // decides, and for 256-byte rows, whose accumulators leave two waves to a SIMD in any case; with 4 blocks to a CU and
    // more, smaller ones keep the CUs busier (48 histories to 512 tokens, 64 features, dK and dV: 84 us against 111).  fp32
    // at 128 features: one wave's registers fill a SIMD.
    if (A.nq * A.G + A.nk < (int64_t)128 * A.n_seq) return launch_bwd<T, D, 1, 1, 1>(A, s);
    if constexpr (sizeof(T) == 4 && D == 128) return launch_bwd<T, D, 4, 1, 2>(A, s);
    else {
        if constexpr (D * sizeof(T) < 256)
            if ((A.nk / 128 + A.n_seq + 2) * A.kv_heads >= 4 * 256) return launch_bwd<T, D, 4, 1, 2>(A, s);
        return launch_bwd<T, D, 4, 2, 2>(A, s);
    }
}

// Splits of the key axis where rows are few: enough one-wave blocks for 16 to a CU, and at least `least` keys of the longest
// axis to each (the lengths themselves are on the device; a split divides the length it finds there).
int key_splits(int64_t blocks, bool one, int64_t keys, int64_t least) {
    const int64_t want = ((one ? 4096 : 1024) + blocks - 1) / (blocks > 0 ? blocks : 1);
    const int64_t most = (keys + least - 1) / least;
    const int64_t n = want < most ? want : most;
    return (int)(n < 1 ? 1 : n > MAX_SPLITS ? MAX_SPLITS : n);
}
bool few_rows(int64_t rows) { return rows < 64; }   // of a sequence: one-wave blocks, four waves would mostly idle
int64_t cache_blocks(int64_t batch, int64_t rows, int64_t kv_heads) {
    return batch * kv_heads * (few_rows(rows) ? (rows + 31) / 32 : (rows + 127) / 128);
}
int cache_splits(int64_t batch, int64_t rows, int64_t kv_heads, int64_t capacity) {
    return key_splits(cache_blocks(batch, rows, kv_heads), few_rows(rows), capacity, 64);
}
// Packed sequences: blocks by the rows of an average sequence, splits by its keys, at least 256 to each.  A block takes
// about `key` ns to a key (measured); where that comes to 20 us the axis is split, into as many as write their sums in a
// quarter of that time (written and read at 3 TB/s), 64 MB at most.  Unsplit and split, 128 features: 16 x 8 tokens on 8192
// keys, bf16, 8 heads over 2: 330 and 38 us; one causal history of 4096, a head: bf16 102 and 31 us, fp32 538 and 68 us;
// two of 1024, 8 heads, bf16, stay unsplit: 33 and 46 us.
int64_t packed_blocks(int64_t n_seq, int64_t nq, int64_t G, int64_t kv_heads) {
    return (nq * G / (nq * G < 64 * n_seq ? 32 : 128) + n_seq + 2) * kv_heads;
}
int packed_splits(int dtype, int64_t n_seq, int64_t nq, int64_t nk, int64_t heads, int64_t kv_heads, int D) {
    if (n_seq < 1 || nq < 1 || nk < 1) return 1;
    const int64_t G = heads / kv_heads, keys = nk / n_seq, row = heads * nq * (D + 2) * 4;
    const bool one = nq * G < 64 * n_seq;
    const int64_t key = (dtype == TAGAN_F32 ? 10 + D : 6 + D / 7) * (one ? 3 : 2) / 2, ns = keys * key;
    if (ns < 20000) return 1;
    const int64_t bytes = ns * 375, most = 64ll << 20, budget = (bytes < most ? bytes : most) / row;
    const int n = key_splits(packed_blocks(n_seq, nq, G, kv_heads), one, keys, 256);
    return n < budget ? n : budget < 2 ? 1 : (int)budget;
}

template <typename T, int D>
int launch_splits(const AttnArgs& A, int64_t blocks, bool one, const char* what, hipStream_t s) {
    const int64_t joins = A.part_rows * (D / 32);
    TAGAN_REQUIRE(fits_grid(blocks * A.splits, one ? 64 : 256) && fits_grid(joins, 512), TAGAN_ERR_UNSUPPORTED,
                  "%s: too many rows", what);
    const unsigned grid = (unsigned)(blocks * A.splits);
    // 32 keys and values of 128 fp32 features are 32 KB: twice that would leave two waves to a CU
    if (one) k_attn_fwd<T, D, 1, true, sizeof(T) == 4 && D == 128 ? 1 : 2><<<grid, 64, 0, s>>>(A);
    else k_attn_fwd<T, D, 4, true, 2><<<grid, 256, 0, s>>>(A);
    TAGAN_CHECK_LAUNCH(what);
    static_assert(MAX_SPLITS <= 512, "a thread to a split");
    if (A.splits <= 64) k_attn_join<T, D, 64><<<(unsigned)joins, 64, 0, s>>>(A);
    else k_attn_join<T, D, 512><<<(unsigned)joins, 512, 0, s>>>(A);
    TAGAN_CHECK_LAUNCH(what);
    return TAGAN_OK;
}

template <typename T, int D>
int run_fwd(const AttnArgs& A, hipStream_t s) {
    const bool one = A.nq * A.G < (int64_t)64 * A.n_seq;
    const int64_t blocks = packed_blocks(A.n_seq, A.nq, A.G, A.kv_heads);
    TAGAN_REQUIRE(fits_grid(blocks, one ? 64 : 256), TAGAN_ERR_UNSUPPORTED, "packed_attn_fwd: too many tiles");
    if constexpr (sizeof(T) == 2)
        if (few_keys(A)) {
            if (one) k_attn_fwd<T, D, 1, false, 1, true><<<(unsigned)blocks, 64, 0, s>>>(A);
            else k_attn_fwd<T, D, 4, false, 2, true><<<(unsigned)blocks, 256, 0, s>>>(A);
            TAGAN_CHECK_LAUNCH("packed_attn_fwd");
            return TAGAN_OK;
        }
    if (one) k_attn_fwd<T, D, 1, false, 1><<<(unsigned)blocks, 64, 0, s>>>(A);
    else k_attn_fwd<T, D, 4, false, 2><<<(unsigned)blocks, 256, 0, s>>>(A);
    TAGAN_CHECK_LAUNCH("packed_attn_fwd");
    return TAGAN_OK;
}
template <typename T, int D>
int run_fwd_splits(const AttnArgs& A, hipStream_t s) {
    return launch_splits<T, D>(A, packed_blocks(A.n_seq, A.nq, A.G, A.kv_heads), A.nq * A.G < (int64_t)64 * A.n_seq,
                               "packed_attn_fwd", s);
}

template <typename T, int D>
int run_cached(const AttnArgs& A, hipStream_t s) {
    const int64_t rows = A.nq * A.G, blocks = cache_blocks(A.n_seq, rows, A.kv_heads);
    const bool one = few_rows(rows);
    if (A.splits > 1) return launch_splits<T, D>(A, blocks, one, "cached_attn", s);
    TAGAN_REQUIRE(fits_grid(blocks, one ? 64 : 256), TAGAN_ERR_UNSUPPORTED, "cached_attn: too many rows");
    if (one) k_attn_fwd<T, D, 1, false, 1><<<(unsigned)blocks, 64, 0, s>>>(A);
    else k_attn_fwd<T, D, 4, false, 2><<<(unsigned)blocks, 256, 0, s>>>(A);
    TAGAN_CHECK_LAUNCH("cached_attn");
    return TAGAN_OK;
}

int padded_dim(int32_t dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

}  // namespace
}  // namespace tagan

using namespace tagan;

extern "C" {

size_t tagan_packed_attn_fwd_workspace(int32_t n_seq, int64_t nq, int64_t nk, int32_t heads, int32_t kv_heads,
                                       int32_t head_dim) {
    if (kv_heads < 1 || heads < kv_heads || head_dim < 1 || head_dim > MAX_DIM) return 0;
    if (nq > MAX_TOKENS || nk > MAX_TOKENS || nq > MAX_ROWS / heads) return 0;   // the forward refuses them
    const int n = packed_splits(TAGAN_F32, n_seq, nq, nk, heads, kv_heads, padded_dim(head_dim));   // bf16 splits no more
    return n == 1 ? 0 : (size_t)n * (size_t)nq * (size_t)heads * (size_t)(padded_dim(head_dim) + 2) * 4;
}

int tagan_packed_attn_fwd(int dtype, int32_t n_seq, int64_t nq, int64_t nk, int32_t heads, int32_t kv_heads,
                          int32_t head_dim, const void* q, int64_t q_tok, int64_t q_head, const void* k, int64_t k_tok,
                          int64_t k_head, const void* v, int64_t v_tok, int64_t v_head, const int32_t* offsets_q,
                          const int32_t* offsets_k, int causal, float scale, void* out, int64_t o_tok, int64_t o_head,
                          float* lse, void* rest, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_shape("packed_attn_fwd", dtype, heads, kv_heads, head_dim, scale);
    if (rc != TAGAN_OK) return rc;
    TAGAN_REQUIRE(n_seq >= 0 && nq >= 0 && nk >= 0 && nq <= MAX_TOKENS && nk <= MAX_TOKENS,
                  TAGAN_ERR_ARG, "packed_attn_fwd: %d sequences, %lld and %lld tokens", n_seq, (long long)nq, (long long)nk);
    TAGAN_REQUIRE(nq * (heads / kv_heads) <= MAX_TOKENS && nq <= MAX_ROWS / heads, TAGAN_ERR_UNSUPPORTED,
                  "packed_attn_fwd: %lld tokens of %d heads",
                  (long long)nq, heads);
    if (nq == 0) return TAGAN_OK;
    TAGAN_REQUIRE(offsets_q && offsets_k, TAGAN_ERR_ARG, "packed_attn_fwd: null offsets");
    const int es = dtype == TAGAN_F32 ? 4 : 2;
    AttnArgs A = {};
    A.q = q; A.k = k; A.v = v; A.out = out; A.lse = lse; A.rest = (uint16_t*)rest;
    TAGAN_REQUIRE(!rest || (dtype == TAGAN_BF16 && ((uintptr_t)rest & 15) == 0), TAGAN_ERR_ARG,
                  "packed_attn_fwd: rest is of bf16 and lies on 16 bytes");
    A.qs = {0, q_tok, q_head};
    A.ks = {0, k_tok, k_head};
    A.vs = {0, v_tok, v_head};
    A.os = {0, o_tok, o_head};
    if ((rc = check_tensor("packed_attn_fwd", "q", q, A.qs, 1, nq, heads, head_dim, es)) != TAGAN_OK) return rc;
    if (nk > 0) {
        if ((rc = check_tensor("packed_attn_fwd", "k", k, A.ks, 1, nk, kv_heads, head_dim, es)) != TAGAN_OK) return rc;
        if ((rc = check_tensor("packed_attn_fwd", "v", v, A.vs, 1, nk, kv_heads, head_dim, es)) != TAGAN_OK) return rc;
    }
    if ((rc = check_tensor("packed_attn_fwd", "out", out, A.os, 1, nq, heads, head_dim, es)) != TAGAN_OK) return rc;
    A.offs_q = offsets_q; A.offs_k = offsets_k;
    A.nq = nq; A.nk = nk; A.n_seq = n_seq;
    A.heads = heads; A.kv_heads = kv_heads; A.G = heads / kv_heads; A.dim = head_dim;
    A.causal = causal != 0;
    A.by_g = div_by(A.G);
    A.by_kv = div_by(kv_heads);
    A.scale = scale; A.c = scale * LOG2E;
    hipStream_t s = as_stream(stream);
    const size_t need = tagan_packed_attn_fwd_workspace(n_seq, nq, nk, heads, kv_heads, head_dim);
    TAGAN_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0)),
                  TAGAN_ERR_WORKSPACE, "packed_attn_fwd: workspace of %zu bytes, %zu are needed on 16", workspace_bytes, need);
    A.splits = need ? packed_splits(dtype, n_seq, nq, nk, heads, kv_heads, padded_dim(head_dim)) : 1;
    if (A.splits > 1) {
        A.by_splits = div_by(A.splits);
        A.part = (float*)workspace;
        A.part_rows = nq * heads;
        return dtype == TAGAN_F32 ? TAGAN_BY_DIM(float, head_dim, run_fwd_splits)(A, s)
                                  : TAGAN_BY_DIM(uint16_t, head_dim, run_fwd_splits)(A, s);
    }
    return dtype == TAGAN_F32 ? TAGAN_BY_DIM16(float, head_dim, run_fwd)(A, s)
                              : TAGAN_BY_DIM16(uint16_t, head_dim, run_fwd)(A, s);
}

size_t tagan_packed_attn_bwd_workspace(int64_t nq, int32_t heads) {
    return nq > 0 && heads > 0 ? (size_t)nq * (size_t)heads * 8 : 0;
}

int tagan_packed_attn_bwd(int dtype, int32_t n_seq, int64_t nq, int64_t nk, int32_t heads, int32_t kv_heads,
                          int32_t head_dim, const void* q, int64_t q_tok, int64_t q_head, const void* k, int64_t k_tok,
                          int64_t k_head, const void* v, int64_t v_tok, int64_t v_head, const int32_t* offsets_q,
                          const int32_t* offsets_k, int causal, float scale, const void* out, int64_t o_tok,
                          int64_t o_head, const float* lse, const void* rest, const void* dout, int64_t do_tok, int64_t do_head, void* dq,
                          int64_t dq_tok, int64_t dq_head, void* dk, int64_t dk_tok, int64_t dk_head, void* dv,
                          int64_t dv_tok, int64_t dv_head, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_shape("packed_attn_bwd", dtype, heads, kv_heads, head_dim, scale);
    if (rc != TAGAN_OK) return rc;
    TAGAN_REQUIRE(n_seq >= 0 && nq >= 0 && nk >= 0 && nq <= MAX_TOKENS && nk <= MAX_TOKENS,
                  TAGAN_ERR_ARG, "packed_attn_bwd: %d sequences, %lld and %lld tokens", n_seq, (long long)nq, (long long)nk);
    TAGAN_REQUIRE(nq * (heads / kv_heads) <= MAX_TOKENS && nq <= MAX_ROWS / heads, TAGAN_ERR_UNSUPPORTED,
                  "packed_attn_bwd: %lld tokens of %d heads",
                  (long long)nq, heads);
    if (nq == 0 && nk == 0) return TAGAN_OK;
    TAGAN_REQUIRE(offsets_q && offsets_k, TAGAN_ERR_ARG, "packed_attn_bwd: null offsets");
    TAGAN_REQUIRE(workspace_bytes >= tagan_packed_attn_bwd_workspace(nq, heads) && (nq == 0 || (workspace && lse)),
                  TAGAN_ERR_WORKSPACE, "packed_attn_bwd: workspace of %zu bytes", workspace_bytes);
    const int es = dtype == TAGAN_F32 ? 4 : 2;
    AttnArgs A = {};
    A.q = q; A.k = k; A.v = v; A.o = out; A.dout = dout;
    A.dq = dq; A.dk = dk; A.dv = dv;
    A.lse = (float*)lse; A.stat = (float2*)workspace; A.rest = (uint16_t*)rest;
    TAGAN_REQUIRE(!rest || (dtype == TAGAN_BF16 && ((uintptr_t)rest & 15) == 0), TAGAN_ERR_ARG,
                  "packed_attn_bwd: rest is of bf16 and lies on 16 bytes");
    TAGAN_REQUIRE(((uintptr_t)workspace & 7) == 0, TAGAN_ERR_ARG, "packed_attn_bwd: the workspace has to lie on 8 bytes");
    A.qs = {0, q_tok, q_head};
    A.ks = {0, k_tok, k_head};
    A.vs = {0, v_tok, v_head};
    A.os = {0, o_tok, o_head};
    A.dos = {0, do_tok, do_head};
    A.dqs = {0, dq_tok, dq_head};
    A.dks = {0, dk_tok, dk_head};
    A.dvs = {0, dv_tok, dv_head};
    const struct { const char* name; const void* p; Strides& s; int64_t n; int32_t h; } all[] = {
        {"q", q, A.qs, nq, heads}, {"out", out, A.os, nq, heads}, {"dout", dout, A.dos, nq, heads},
        {"dq", dq, A.dqs, nq, heads}, {"k", k, A.ks, nk, kv_heads}, {"v", v, A.vs, nk, kv_heads},
        {"dk", dk, A.dks, nk, kv_heads}, {"dv", dv, A.dvs, nk, kv_heads}};
    for (const auto& x : all)
        if (x.n > 0 && (rc = check_tensor("packed_attn_bwd", x.name, x.p, x.s, 1, x.n, x.h, head_dim, es)) != TAGAN_OK)
            return rc;
    A.offs_q = offsets_q; A.offs_k = offsets_k;
    A.nq = nq; A.nk = nk; A.n_seq = n_seq;
    A.heads = heads; A.kv_heads = kv_heads; A.G = heads / kv_heads; A.dim = head_dim;
    A.causal = causal != 0; A.splits = 1;
    A.by_g = div_by(A.G);
    A.by_kv = div_by(kv_heads);
    A.scale = scale; A.c = scale * LOG2E;
    // a tile of packed rows spans (32 / G + 2) tokens and G heads in 31 bits
    TAGAN_REQUIRE((A.qs.head > A.dos.head ? A.qs.head : A.dos.head) * A.G * es < (1ll << 30), TAGAN_ERR_UNSUPPORTED,
                  "packed_attn_bwd: head strides %lld and %lld", (long long)q_head, (long long)do_head);
    hipStream_t s = as_stream(stream);
    return dtype == TAGAN_F32 ? TAGAN_BY_DIM16(float, head_dim, run_bwd)(A, s)
                              : TAGAN_BY_DIM16(uint16_t, head_dim, run_bwd)(A, s);
}

size_t tagan_cached_attn_workspace(int64_t batch, int32_t new_len, int64_t capacity, int32_t heads, int32_t kv_heads,
                                   int32_t head_dim) {
    if (batch <= 0 || new_len <= 0 || kv_heads < 1 || heads < kv_heads || head_dim < 1 || head_dim > MAX_DIM) return 0;
    const int64_t rows = (int64_t)new_len * (heads / kv_heads);
    if (batch > 0x7fffffff || batch * new_len > MAX_ROWS / heads) return 0;      // cached_attn refuses them
    const int n = cache_splits(batch, rows, kv_heads, capacity);
    return n == 1 ? 0 : (size_t)n * (size_t)batch * (size_t)(kv_heads * rows) * (size_t)(padded_dim(head_dim) + 2) * 4;
}

int tagan_cached_attn(int dtype, int64_t batch, int32_t new_len, int64_t capacity, int32_t heads, int32_t kv_heads,
                      int32_t head_dim, const void* q, int64_t q_b, int64_t q_tok, int64_t q_head, const void* k_cache,
                      int64_t k_b, int64_t k_tok, int64_t k_head, const void* v_cache, int64_t v_b, int64_t v_tok,
                      int64_t v_head, const int32_t* lens, float scale, void* out, int64_t o_b, int64_t o_tok,
                      int64_t o_head, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_shape("cached_attn", dtype, heads, kv_heads, head_dim, scale);
    if (rc != TAGAN_OK) return rc;
    TAGAN_REQUIRE(batch >= 0 && batch <= 0x7fffffff && new_len >= 0 && capacity >= 0 && capacity <= MAX_TOKENS,
                  TAGAN_ERR_ARG, "cached_attn: batch %lld new_len %d capacity %lld", (long long)batch, new_len,
                  (long long)capacity);
    if (batch == 0 || new_len == 0) return TAGAN_OK;
    TAGAN_REQUIRE((int64_t)new_len * (heads / kv_heads) <= MAX_TOKENS && batch * new_len <= MAX_ROWS / heads,
                  TAGAN_ERR_UNSUPPORTED, "cached_attn: %lld x %d new tokens of %d heads", (long long)batch, new_len, heads);
    TAGAN_REQUIRE(lens, TAGAN_ERR_ARG, "cached_attn: null lens");
    const int es = dtype == TAGAN_F32 ? 4 : 2;
    AttnArgs A = {};
    A.q = q; A.k = k_cache; A.v = v_cache; A.out = out;
    A.qs = {q_b, q_tok, q_head};
    A.ks = {k_b, k_tok, k_head};
    A.vs = {v_b, v_tok, v_head};
    A.os = {o_b, o_tok, o_head};
    if ((rc = check_tensor("cached_attn", "q", q, A.qs, batch, new_len, heads, head_dim, es)) != TAGAN_OK) return rc;
    if (capacity > 0) {
        if ((rc = check_tensor("cached_attn", "k_cache", k_cache, A.ks, batch, capacity, kv_heads, head_dim, es)) != TAGAN_OK) return rc;
        if ((rc = check_tensor("cached_attn", "v_cache", v_cache, A.vs, batch, capacity, kv_heads, head_dim, es)) != TAGAN_OK) return rc;
    }
    if ((rc = check_tensor("cached_attn", "out", out, A.os, batch, new_len, heads, head_dim, es)) != TAGAN_OK) return rc;
    A.lens = lens;
    A.nq = new_len; A.nk = capacity; A.n_seq = (int32_t)batch;
    A.heads = heads; A.kv_heads = kv_heads; A.G = heads / kv_heads; A.dim = head_dim;
    A.causal = 1;
    A.by_g = div_by(A.G);
    A.by_kv = div_by(kv_heads);
    A.scale = scale; A.c = scale * LOG2E;
    const int64_t rows = (int64_t)new_len * A.G;
    A.splits = cache_splits(batch, rows, kv_heads, capacity);
    A.by_splits = div_by(A.splits);
    A.by_tiles = div_by(few_rows(rows) ? (rows + 31) / 32 : (rows + 127) / 128);
    A.part = (float*)workspace;
    A.part_rows = batch * new_len * heads;
    const size_t need = tagan_cached_attn_workspace(batch, new_len, capacity, heads, kv_heads, head_dim);
    TAGAN_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0)),
                  TAGAN_ERR_WORKSPACE, "cached_attn: workspace of %zu bytes, %zu are needed on 16", workspace_bytes, need);
    hipStream_t s = as_stream(stream);
    return dtype == TAGAN_F32 ? TAGAN_BY_DIM(float, head_dim, run_cached)(A, s)
                              : TAGAN_BY_DIM(uint16_t, head_dim, run_cached)(A, s);
}

}  // extern "C"
