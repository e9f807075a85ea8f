// Rotary positions: every pair (a, b) of a head's first `rot` features is turned by the angle t = position * freq of
// the pair, (a, b) -> scale * (a cos t - b sin t, a sin t + b cos t); the features behind them pass as they are.  The
// gradient of a turn is the turn back (sign of sin) with the same scale.  Serving: the same turn of new tokens at
// positions lens[b] + i, with k and v written behind the cached rows in the same launch.
//
// Angles: position * freq is formed in fp64 (a position of 10^6 has an fp32 angle error of 0.06 rad), reduced there to
// half turns in [-1, 1], and only that remainder goes to fp32 sinpi / cospi (|error of the angle| <= pi 2^-25).  A
// block of tokens evaluates its tokens x rot/2 angles once into LDS and reuses them over all heads of q and k.
//
// Bound: HBM, two moves of every element: 24001 tokens of 32 + 8 heads of 128, bf16, 492 MB: 97 us, 5.1 TB/s (a copy
// reaches 4.7); a serving step of 48 tokens: 6 us.  A thread keeps one item (16 B of a head: a vector of each half, or a
// vector of neighbouring pairs) and steps over the heads of the block's tokens, so there is no index division in the
// loop (18889 tokens of 9 heads: 29 us; 47 with one token after the other).
// Small heads stay below that: 400000 tokens of 8 + 8 heads of 16, bf16, all turned 1.7 TB/s (240 us); with 8 of the 16 turned
// a half is no whole vector, and the form with one element to a thread moves 1.2 TB/s (340 us).
#include "common.cuh"

namespace tagan {
namespace {

constexpr int RB = 256;            // threads of a block
constexpr int ROT_MAX_DIM = 256;   // one item per thread in the scalar form
constexpr int ROT_MAX_HEADS = 1 << 28;   // a block counts the heads of its tokens, and a step behind them, in 31 bits

struct RotTensor {
    const void* in;
    void* out;
    int64_t ib, it, ih, ob, ot, oh;   // strides in elements: batch, token, head
    int32_t heads;
};

struct RotArgs {
    RotTensor x[3];             // q, k (turned), v (moved); heads = 0 where absent
    const void* pos;            // [tokens], pos_type; null: lens[b] + t
    const int32_t* lens;
    const double* freq;         // [rot / 2]
    int64_t tokens;             // batch * per
    int32_t per, pos_type, dim, rot, interleaved;
    int64_t capacity;           // rows of a cache (lens form): rows outside [0, capacity) are not written
    float scale, sign;
};

template <typename S>
__device__ __forceinline__ void unpack(const uint4& u, float* v) {
    if constexpr (sizeof(S) == 4) {
        v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y);
        v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
    } else {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
template <typename S>
__device__ __forceinline__ uint4 pack(const float* v) {
    if constexpr (sizeof(S) == 4)
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    else
        return make_uint4(f2bf2(v[0], v[1]), f2bf2(v[2], v[3]), f2bf2(v[4], v[5]), f2bf2(v[6], v[7]));
}
// one element of the scalar form
__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(uint16_t* p, float v) { *p = (uint16_t)f2bf2(v, 0.f); }

__device__ __forceinline__ double rot_position(const RotArgs& A, int64_t n) {
    if (A.pos == nullptr) return (double)((int64_t)A.lens[n / A.per] + n % A.per);
    switch (A.pos_type) {
        case TAGAN_POS_I32: return (double)((const int32_t*)A.pos)[n];
        case TAGAN_POS_I64: return (double)((const int64_t*)A.pos)[n];
        case TAGAN_POS_F32: return (double)((const float*)A.pos)[n];
        default: return ((const double*)A.pos)[n];
    }
}

// TOK tokens to a block; VEC: 16-byte items, else one element (of each half) per item
template <typename S, bool VEC, int TOK>
__global__ void __launch_bounds__(RB) k_rotary(RotArgs A) {
    constexpr int E = VEC ? 16 / (int)sizeof(S) : 1;   // elements of an item's vector
    __shared__ float2 cs[TOK * (ROT_MAX_DIM / 2)];
    __shared__ int64_t in_at[3][TOK], out_at[3][TOK];
    const int half = A.rot / 2;
    const int64_t n0 = (int64_t)blockIdx.x * TOK;
    const int ntok = (int)min((int64_t)TOK, A.tokens - n0);
    for (int i = threadIdx.x; i < ntok * half; i += RB) {
        const int t = i / half, p = i - t * half;
        const double a = rot_position(A, n0 + t) * A.freq[p];
        double u = a * 0.31830988618379067154;   // half turns
        u -= 2.0 * rint(0.5 * u);
        float s, c;
        sincospif((float)u, &s, &c);
        cs[i] = make_float2(c * A.scale, s * A.scale * A.sign);
    }
    // where each token's heads lie; an output of -1 is not written
    if (threadIdx.x < 3 * TOK) {
        const int which = threadIdx.x / TOK, t = threadIdx.x % TOK;
        if (t < ntok) {
            const RotTensor& X = A.x[which];
            const int64_t n = n0 + t, b = n / A.per, ti = n - b * A.per;
            int64_t row = ti;
            if (A.pos == nullptr && which > 0) row += A.lens[b];   // a cache row
            in_at[which][t] = b * X.ib + ti * X.it;
            out_at[which][t] = A.pos == nullptr && which > 0 && (row < 0 || row >= A.capacity) ? -1 : b * X.ob + row * X.ot;
        }
    }
    __syncthreads();
    // items of a head: the turned ones first, then those that are moved
    const int nrot = A.interleaved ? (VEC ? A.rot / E : half) : half / E;
    const int ntail = (A.dim - A.rot) / E, nall = A.dim / E;
    for (int which = 0; which < 3; ++which) {
        const RotTensor& X = A.x[which];
        if (X.heads == 0) continue;
        const int items = which == 2 ? nall : nrot + ntail;
        const int step = RB / items, rows = ntok * X.heads;   // rows: heads of all tokens
        if ((int)threadIdx.x >= step * items) continue;
        const int item = threadIdx.x % items;
        int at, second = -1, pair = 0;             // first feature, the other half's, first pair
        if (which == 2) at = item * E;
        else if (item >= nrot) at = A.rot + (item - nrot) * E;
        else if (!A.interleaved) { at = item * E; second = half + at; pair = at; }
        else if constexpr (VEC) { at = item * E; second = at; pair = at / 2; }
        else { at = 2 * item; second = at + 1; pair = item; }
        const auto token = [&](int r) {
            int t = 0;
#pragma unroll
            for (int i = 1; i < TOK; ++i) t += r >= i * X.heads;
            return t;
        };
        // U rows at a time, all loads before the first store (outputs may be the inputs, so the compiler keeps their
        // order): 117 -> 97 us for 24001 tokens of 40 heads
        constexpr int U = VEC ? 4 : 1;
        for (int r0 = threadIdx.x / items; r0 < rows; r0 += U * step) {
            if constexpr (VEC) {
                uint4 a[U], b[U];
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    const int r = r0 + j * step, t = token(r);
                    if (r >= rows) continue;
                    const S* src = (const S*)X.in + in_at[which][t] + (r - t * X.heads) * X.ih;
                    a[j] = *(const uint4*)(src + at);
                    if (second > at) b[j] = *(const uint4*)(src + second);
                }
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    const int r = r0 + j * step, t = token(r);
                    if (r >= rows || out_at[which][t] < 0) continue;
                    S* dst = (S*)X.out + out_at[which][t] + (r - t * X.heads) * X.oh;
                    if (second < 0) {
                        *(uint4*)(dst + at) = a[j];
                        continue;
                    }
                    const float2* w = cs + t * half + pair;
                    float x[E], y[E];
                    unpack<S>(a[j], x);
                    if (!A.interleaved) {
                        unpack<S>(b[j], y);
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const float c = w[e].x, s = w[e].y, xv = x[e], yv = y[e];
                            x[e] = xv * c - yv * s;
                            y[e] = xv * s + yv * c;
                        }
                        *(uint4*)(dst + second) = pack<S>(y);
                    } else {
#pragma unroll
                        for (int e = 0; e < E; e += 2) {
                            const float c = w[e / 2].x, s = w[e / 2].y, xv = x[e], yv = x[e + 1];
                            x[e] = xv * c - yv * s;
                            x[e + 1] = xv * s + yv * c;
                        }
                    }
                    *(uint4*)(dst + at) = pack<S>(x);
                }
            } else {
                const int t = token(r0), h = r0 - t * X.heads;
                if (out_at[which][t] < 0) continue;
                const S* src = (const S*)X.in + in_at[which][t] + h * X.ih;
                S* dst = (S*)X.out + out_at[which][t] + h * X.oh;
                if (second < 0) {
                    dst[at] = src[at];
                } else {
                    const float2* w = cs + t * half + pair;
                    const float xv = ld1(src + at), yv = ld1(src + second), c = w->x, s = w->y;
                    st1(dst + at, xv * c - yv * s);
                    st1(dst + second, xv * s + yv * c);
                }
            }
        }
    }
}

bool vec_ok(const RotArgs& A, int es) {
    const int E = 16 / es;
    if (A.dim % E || A.rot % E || (!A.interleaved && (A.rot / 2) % E)) return false;
    for (const RotTensor& X : A.x) {
        if (X.heads == 0) continue;
        if (((uintptr_t)X.in | (uintptr_t)X.out) & 15) return false;
        if ((X.ib | X.it | X.ih | X.ob | X.ot | X.oh) % E) return false;
    }
    return true;
}

template <typename S>
int run_rotary(const RotArgs& A, hipStream_t s, const char* what) {
    // four tokens to a block once that still leaves 8 blocks to each of the 256 CUs; one otherwise (a serving step's
    // few tokens spread over as many CUs)
    const bool four = A.tokens >= 4 * 2048;
    const int64_t blocks = four ? (A.tokens + 3) / 4 : A.tokens;
    TAGAN_REQUIRE(blocks <= 0xffffffffll / RB, TAGAN_ERR_UNSUPPORTED,   // a launch counts its threads in 32 bits
                  "%s: %lld tokens", what, (long long)A.tokens);
    if (vec_ok(A, (int)sizeof(S))) {
        if (four) k_rotary<S, true, 4><<<(unsigned)blocks, RB, 0, s>>>(A);
        else k_rotary<S, true, 1><<<(unsigned)blocks, RB, 0, s>>>(A);
    } else {
        if (four) k_rotary<S, false, 4><<<(unsigned)blocks, RB, 0, s>>>(A);
        else k_rotary<S, false, 1><<<(unsigned)blocks, RB, 0, s>>>(A);
    }
    TAGAN_CHECK_LAUNCH(what);
    return TAGAN_OK;
}

int check_dims(const char* what, int dtype, int32_t heads, int32_t kv_heads, int32_t dim, int32_t rot, float scale) {
    TAGAN_REQUIRE(dtype == TAGAN_F32 || dtype == TAGAN_BF16, TAGAN_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
    TAGAN_REQUIRE(heads >= 0 && kv_heads >= 0 && heads + kv_heads > 0, TAGAN_ERR_ARG, "%s: heads %d, %d", what, heads,
                  kv_heads);
    TAGAN_REQUIRE(heads <= ROT_MAX_HEADS && kv_heads <= ROT_MAX_HEADS, TAGAN_ERR_UNSUPPORTED,
                  "%s: heads %d, %d (up to %d)", what, heads, kv_heads, ROT_MAX_HEADS);
    TAGAN_REQUIRE(dim >= 1 && dim <= ROT_MAX_DIM, TAGAN_ERR_UNSUPPORTED, "%s: head_dim %d (1 to %d)", what, dim,
                  ROT_MAX_DIM);
    TAGAN_REQUIRE(rot >= 2 && rot <= dim && rot % 2 == 0, TAGAN_ERR_ARG, "%s: %d of %d features turned", what, rot,
                  dim);
    TAGAN_REQUIRE(isfinite(scale), TAGAN_ERR_ARG, "%s: scale", what);
    return TAGAN_OK;
}

}  // namespace
}  // namespace tagan

using namespace tagan;

extern "C" {

int tagan_rotary(int dtype, int64_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t rot,
                 const void* q, int64_t q_tok, int64_t q_head, const void* k, int64_t k_tok, int64_t k_head,
                 const void* positions, int32_t pos_type, const double* inv_freq, float scale, int interleaved,
                 int inverse, void* q_out, int64_t qo_tok, int64_t qo_head, void* k_out, int64_t ko_tok,
                 int64_t ko_head, void* stream) {
    const int rc = check_dims("rotary", dtype, heads, kv_heads, head_dim, rot, scale);
    if (rc != TAGAN_OK) return rc;
    TAGAN_REQUIRE(tokens >= 0, TAGAN_ERR_ARG, "rotary: %lld tokens", (long long)tokens);
    TAGAN_REQUIRE(pos_type >= TAGAN_POS_I32 && pos_type <= TAGAN_POS_F64, TAGAN_ERR_UNSUPPORTED,
                  "rotary: position type %d", pos_type);
    if (tokens == 0) return TAGAN_OK;
    TAGAN_REQUIRE(positions && inv_freq && (heads == 0 || (q && q_out)) && (kv_heads == 0 || (k && k_out)),
                  TAGAN_ERR_ARG, "rotary: null pointer");
    RotArgs A = {};
    A.x[0] = {q, q_out, 0, q_tok, q_head, 0, qo_tok, qo_head, heads};
    A.x[1] = {k, k_out, 0, k_tok, k_head, 0, ko_tok, ko_head, kv_heads};
    A.pos = positions;
    A.freq = inv_freq;
    A.tokens = tokens;
    A.per = 0x7fffffff;
    TAGAN_REQUIRE(tokens < A.per, TAGAN_ERR_UNSUPPORTED, "rotary: %lld tokens", (long long)tokens);
    A.pos_type = pos_type;
    A.dim = head_dim;
    A.rot = rot;
    A.interleaved = interleaved != 0;
    A.scale = scale;
    A.sign = inverse ? -1.f : 1.f;
    return dtype == TAGAN_F32 ? run_rotary<float>(A, as_stream(stream), "rotary")
                              : run_rotary<uint16_t>(A, as_stream(stream), "rotary");
}

int tagan_rotary_append(int dtype, int64_t batch, int32_t new_len, int32_t heads, int32_t kv_heads, int32_t head_dim,
                        int32_t rot, const void* q, int64_t q_b, int64_t q_tok, int64_t q_head, const void* k,
                        int64_t k_b, int64_t k_tok, int64_t k_head, const void* v, int64_t v_b, int64_t v_tok,
                        int64_t v_head, const int32_t* lens, const double* inv_freq, float scale, int interleaved,
                        void* q_out, int64_t qo_b, int64_t qo_tok, int64_t qo_head, void* k_cache, int64_t kc_b,
                        int64_t kc_tok, int64_t kc_head, void* v_cache, int64_t vc_b, int64_t vc_tok, int64_t vc_head,
                        int64_t capacity, void* stream) {
    const int rc = check_dims("rotary_append", dtype, heads, kv_heads, head_dim, rot, scale);
    if (rc != TAGAN_OK) return rc;
    TAGAN_REQUIRE(heads > 0 && kv_heads > 0 && batch >= 0 && new_len >= 0 && capacity >= 0, TAGAN_ERR_ARG,
                  "rotary_append: batch %lld new_len %d capacity %lld", (long long)batch, new_len, (long long)capacity);
    if (batch == 0 || new_len == 0) return TAGAN_OK;
    TAGAN_REQUIRE(q && k && v && lens && inv_freq && q_out && k_cache && v_cache, TAGAN_ERR_ARG,
                  "rotary_append: null pointer");
    TAGAN_REQUIRE(batch <= 0x7fffffff / new_len, TAGAN_ERR_UNSUPPORTED, "rotary_append: %lld x %d tokens",
                  (long long)batch, new_len);
    RotArgs A = {};
    A.x[0] = {q, q_out, q_b, q_tok, q_head, qo_b, qo_tok, qo_head, heads};
    A.x[1] = {k, k_cache, k_b, k_tok, k_head, kc_b, kc_tok, kc_head, kv_heads};
    A.x[2] = {v, v_cache, v_b, v_tok, v_head, vc_b, vc_tok, vc_head, kv_heads};
    A.lens = lens;
    A.freq = inv_freq;
    A.tokens = batch * new_len;
    A.per = new_len;
    A.dim = head_dim;
    A.rot = rot;
    A.interleaved = interleaved != 0;
    A.capacity = capacity;
    A.scale = scale;
    A.sign = 1.f;
    return dtype == TAGAN_F32 ? run_rotary<float>(A, as_stream(stream), "rotary_append")
                              : run_rotary<uint16_t>(A, as_stream(stream), "rotary_append");
}

}  // extern "C"
