// MI355X (gfx950) loss operators: token log-probabilities from logits with their gradient, the clipped policy
// loss with a KL term (from log-probabilities, or straight from the logits) and the preference loss.  C ABI in
// include/rlx_adamw.h.
//
// The work is streams of logits over HBM with one exponential per element; there is nothing for the matrix cores.
// Measured rates below are bytes that have to move (each read once, each written once) over the time on the GPU, inputs
// changing from call to call so that nothing is left in the caches.
//
// Softmax statistics.  With k = log2(e) / temperature a row's softmax is 2^(z k) / sum 2^(z k).  A lane keeps
//     ref = an integer, sum = sum 2^(z k - ref), dot = sum 2^(z k - ref) (z k - ref),
// where ref is about the largest z k so far, rounded up.  z k - ref is one fused multiply-add (rounded once, so the
// size of z k itself costs nothing), and because references are integers, bringing two partial results to a common
// reference multiplies by a power of two: joining lanes, wavefronts or workgroups rounds nothing but the additions.
// References are kept within +-2^29, so that logits of -inf and of a type's lowest value simply contribute 0.  Rows
// whose own values lie out there (every logit the lowest value, +inf, NaN) come out with a sum of 0, infinity or NaN;
// such rows, and only they, are computed again with the row's maximum subtracted first.
//
// The target's own term is kept apart from the sums over the others (`rest`): where the target has most of the
// probability, log p = -log(1 + rest / own) and 1 - p = rest / sum keep their relative precision, which a sum that has
// swallowed both no longer holds (it left log p = -0.0007 off by 2e-4 of itself).

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>

#include "rlx_adamw.h"
#include "rlx_internal.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at any 2-byte boundary: rows of an odd vocabulary start anywhere (gfx950 writes these as one 128-bit access)
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
constexpr float kLn2Hi = 45426.0f / 65536.0f;             // ln 2 cut to 15 bits: an integer below 2^9 times this is exact
constexpr float kLn2Lo = (float)(0.693147180559945309417 - 45426.0 / 65536.0);
constexpr float kRefMost = 536870912.0f;                  // 2^29
constexpr float kMostLse = 16384.0f;                      // beyond, an lse is too coarse to take logits from
constexpr float kLeastD = -1e30f;                         // keeps 0 * (-inf) out of sums of p log p

struct Logits {             // rlx_logits as the kernels take it
    char* data;
    int64_t row_stride, group_stride;      // elements
    uint32_t group_rows, rows;
    int32_t vocab;
};

__device__ __forceinline__ int64_t row_at(const Logits& x, uint32_t r) {
    if (x.group_rows >= x.rows) return (int64_t)r * x.row_stride;
    const uint32_t g = r / x.group_rows;
    return (int64_t)g * x.group_stride + (int64_t)(r - g * x.group_rows) * x.row_stride;
}

// --- the three logit types: PER elements in 16 bytes -----------------------------------------------------------------

__device__ __forceinline__ uint32_t max_f16x2(uint32_t a, uint32_t b) {       // of NaN and a number: the number
    uint32_t r;
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// Element `at` of eight 16-bit ones becomes the half of `least`.
__device__ __forceinline__ void drop_half(u32x4& v, int at, uint32_t least) {
    const uint32_t keep = at & 1 ? 0x0000ffffu : 0xffff0000u;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i == at >> 1) v[i] = (v[i] & keep) | (least & ~keep);
}

struct F16 {
    static constexpr int PER = 8, SIZE = 2;
    static constexpr uint32_t kLeast = 0xfc00fc00u;                             // -inf, twice
    static __device__ __forceinline__ void drop(u32x4& v, int at) { drop_half(v, at, kLeast); }
    typedef uint32_t Top;                                                       // two running maxima
    static __device__ __forceinline__ Top no_top() { return kLeast; }
    static __device__ __forceinline__ void add_top(Top& t, u32x4 v) {
        t = max_f16x2(max_f16x2(t, max_f16x2(v[0], v[1])), max_f16x2(v[2], v[3]));
    }
    static __device__ __forceinline__ float top_of(Top t) {
        const f16x2 h = __builtin_bit_cast(f16x2, t);
        return fmaxf((float)h[0], (float)h[1]);
    }
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = v[i];
            const f16x2 h = __builtin_bit_cast(f16x2, w);
            f[2 * i] = (float)h[0];
            f[2 * i + 1] = (float)h[1];
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {        // round to nearest even
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f16x2 h = {(_Float16)f[2 * i], (_Float16)f[2 * i + 1]};
            v[i] = __builtin_bit_cast(uint32_t, h);
        }
        return v;
    }
    static __device__ __forceinline__ float one(const char* p, int64_t i) {
        return (float)((const RLX_GLOBAL _Float16*)p)[i];
    }
    static __device__ __forceinline__ void put(char* p, int64_t i, float f) { ((RLX_GLOBAL _Float16*)p)[i] = (_Float16)f; }
};

struct BF16 {
    static constexpr int PER = 8, SIZE = 2;
    static constexpr uint32_t kLeast = 0xff80ff80u;
    static __device__ __forceinline__ void drop(u32x4& v, int at) { drop_half(v, at, kLeast); }
    typedef float Top;
    static __device__ __forceinline__ Top no_top() { return -INFINITY; }
    static __device__ __forceinline__ void add_top(Top& t, u32x4 v) {
        float f[PER];
        unpack(v, f);
#pragma unroll
        for (int i = 0; i < PER; i++) t = fmaxf(t, f[i]);
    }
    static __device__ __forceinline__ float top_of(Top t) { return t; }
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = v[i];
            f[2 * i] = __builtin_bit_cast(float, w << 16);
            f[2 * i + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f32x2 two = {f[2 * i], f[2 * i + 1]};
            const bf16x2 h = __builtin_convertvector(two, bf16x2);
            v[i] = __builtin_bit_cast(uint32_t, h);
        }
        return v;
    }
    static __device__ __forceinline__ float one(const char* p, int64_t i) {
        const uint32_t w = ((const RLX_GLOBAL uint16_t*)p)[i];
        return __builtin_bit_cast(float, w << 16);
    }
    static __device__ __forceinline__ void put(char* p, int64_t i, float f) { ((RLX_GLOBAL __bf16*)p)[i] = (__bf16)f; }
};

struct F32 {
    static constexpr int PER = 4, SIZE = 4;
    static constexpr uint32_t kLeast = 0xff800000u;
    static __device__ __forceinline__ void drop(u32x4& v, int at) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i == at) v[i] = kLeast;
    }
    typedef float Top;
    static __device__ __forceinline__ Top no_top() { return -INFINITY; }
    static __device__ __forceinline__ void add_top(Top& t, u32x4 v) {
        float f[PER];
        unpack(v, f);
#pragma unroll
        for (int i = 0; i < PER; i++) t = fmaxf(t, f[i]);
    }
    static __device__ __forceinline__ float top_of(Top t) { return t; }
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = v[i];
            f[i] = __builtin_bit_cast(float, w);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[4]) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __builtin_bit_cast(uint32_t, f[i]);
        return v;
    }
    static __device__ __forceinline__ float one(const char* p, int64_t i) { return ((const RLX_GLOBAL float*)p)[i]; }
    static __device__ __forceinline__ void put(char* p, int64_t i, float f) { ((RLX_GLOBAL float*)p)[i] = f; }
};

__device__ __forceinline__ u32x4 load16(const char* p) { return *(const RLX_GLOBAL u32x4_any*)(const RLX_GLOBAL char*)p; }
__device__ __forceinline__ u32x4 load16_once(const char* p) {            // data that is not read again
    return __builtin_nontemporal_load((const RLX_GLOBAL u32x4_any*)(const RLX_GLOBAL char*)p);
}
__device__ __forceinline__ void store16_once(char* p, u32x4 v) {
    __builtin_nontemporal_store(v, (RLX_GLOBAL u32x4_any*)(RLX_GLOBAL char*)p);
}
__device__ __forceinline__ void store16(char* p, u32x4 v) { *(RLX_GLOBAL u32x4_any*)(RLX_GLOBAL char*)p = v; }
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }     // 1 ulp

// --- reductions over a wavefront -------------------------------------------------------------------------------------
// Data-parallel-primitive moves: shifts by 1, 2, 4 and 8 inside rows of 16 lanes leave a row's total in its last lane,
// two broadcasts carry it over the four rows.  Lane 63 holds the result, which every lane gets.  Lanes that a move does
// not reach add `none`.  The order of the additions is fixed.

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t none, uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)x, CTRL, ROWS, 0xf, false);
}

template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(float none, float x) {
    return __builtin_bit_cast(float, moved<CTRL, ROWS>(__builtin_bit_cast(uint32_t, none), __builtin_bit_cast(uint32_t, x)));
}

template <int CTRL, int ROWS, typename T8>
__device__ __forceinline__ T8 moved8(T8 x) {               // 8 bytes; lanes not reached get 0
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint64_t lo = moved<CTRL, ROWS>(0u, (uint32_t)b), hi = moved<CTRL, ROWS>(0u, (uint32_t)(b >> 32));
    return __builtin_bit_cast(T8, lo | (hi << 32));
}

template <int LANES>                                        // of lanes 0 .. LANES - 1 (16 or 64)
__device__ __forceinline__ float last_lane(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), LANES - 1));
}

template <int LANES>
__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, moved<0x111, 0xf>(x, x));
    x = fmaxf(x, moved<0x112, 0xf>(x, x));
    x = fmaxf(x, moved<0x114, 0xf>(x, x));
    x = fmaxf(x, moved<0x118, 0xf>(x, x));
    if constexpr (LANES == 64) {
        x = fmaxf(x, moved<0x142, 0xa>(x, x));
        x = fmaxf(x, moved<0x143, 0xc>(x, x));
    }
    return last_lane<LANES>(x);
}

template <int LANES>
__device__ __forceinline__ float wave_sum(float x) {
    x += moved<0x111, 0xf>(0.0f, x);
    x += moved<0x112, 0xf>(0.0f, x);
    x += moved<0x114, 0xf>(0.0f, x);
    x += moved<0x118, 0xf>(0.0f, x);
    if constexpr (LANES == 64) {
        x += moved<0x142, 0xa>(0.0f, x);
        x += moved<0x143, 0xc>(0.0f, x);
    }
    return last_lane<LANES>(x);
}

template <typename T8>                                      // double or int64_t
__device__ __forceinline__ T8 wave_sum8(T8 x) {
    x += moved8<0x111, 0xf>(x);
    x += moved8<0x112, 0xf>(x);
    x += moved8<0x114, 0xf>(x);
    x += moved8<0x118, 0xf>(x);
    x += moved8<0x142, 0xa>(x);
    x += moved8<0x143, 0xc>(x);
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 63);
    const uint64_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), 63);
    return __builtin_bit_cast(T8, lo | (hi << 32));
}

// Makes the compiler forget what it knows about a value: without this it keeps the unpacked FP32 form of a held group
// from one pass over the registers to the next, which takes twice the registers.
__device__ __forceinline__ void forget(u32x4& v) { asm volatile("" : "+v"(v)); }

// A row is its whole 16-byte groups, counted from its first element wherever that lies, and the fewer than PER elements
// behind them, one per lane.  (Counted from the first 16-byte boundary, a sum's order would depend on the address.)

// Loads N groups per lane, STEP apart; what lies behind the last group comes as -inf.  The loads are unconditional
// (lanes without a group read the last one again): a load under a condition makes the compiler wait for it before it
// issues the next, which took the policy loss of 8,000 rows of 32,000 FP16 from 136 to 246 us.  ONCE: past the
// caches, for rows that start on a 16-byte boundary (statistics of 4,096 x 151,936 FP16: 187 against 199 us); groups of
// other rows share cache lines, which would be fetched twice.
template <typename T, int N, int STEP, bool ONCE>
__device__ __forceinline__ void load_groups(u32x4 (&held)[N], const char* row, int first, int groups) {
    if (groups == 0) {                        // fewer elements than a group: nothing may be read
#pragma unroll
        for (int n = 0; n < N; n++) held[n] = u32x4{T::kLeast, T::kLeast, T::kLeast, T::kLeast};
        return;
    }
    if constexpr (ONCE || T::SIZE == 4) {
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int g = first + n * STEP < groups ? first + n * STEP : groups - 1;
            held[n] = ONCE ? load16_once(row + (int64_t)g * 16) : load16(row + (int64_t)g * 16);
        }
    } else {
        // Rows of an odd vocabulary start in the middle of a word, and a 16-byte load from there is slow (policy loss of 2,250
        // rows of 50,257 BF16: 113 against 95 us).  So the words that hold the group are loaded, four and the one with its
        // last element (the fourth again if the row starts with a word), and shifted into place.  No word is read that
        // holds none of the group's bytes; its other half may be another row's, and is dropped.
        const uint32_t off = (uint32_t)(uintptr_t)row & 2;
        const char* words = row - off;
        uint32_t tail[N];
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int g = first + n * STEP < groups ? first + n * STEP : groups - 1;
            const char* at = words + (int64_t)g * 16;
            held[n] = load16(at);
            tail[n] = *(const RLX_GLOBAL uint32_t*)(const RLX_GLOBAL char*)(at + 12 + 2 * off);
        }
#pragma unroll
        for (int n = 0; n < N; n++) {
            const u32x4 w = held[n];
            held[n] = u32x4{__builtin_amdgcn_alignbyte(w[1], w[0], off), __builtin_amdgcn_alignbyte(w[2], w[1], off),
                            __builtin_amdgcn_alignbyte(w[3], w[2], off), __builtin_amdgcn_alignbyte(tail[n], w[3], off)};
        }
    }
#pragma unroll
    for (int n = 0; n < N; n++)
        if (first + n * STEP >= groups) held[n] = u32x4{T::kLeast, T::kLeast, T::kLeast, T::kLeast};
}

// Takes the target out of the groups that the lanes of a workgroup hold (first group of lane 0: `from`).
template <typename T, int N, int STEP>
__device__ __forceinline__ void drop_target(u32x4 (&held)[N], int from, int target) {
    const int group = target / T::PER - from;                   // the same in all lanes
#pragma unroll
    for (int n = 0; n < N; n++)
        if (group >= n * STEP && group < (n + 1) * STEP && (int)threadIdx.x == group - n * STEP) T::drop(held[n], target % T::PER);
}

// --- statistics of a row ---------------------------------------------------------------------------------------------

struct Stat {
    float ref, sum, dot;
};
constexpr Stat kNoStat = {-kRefMost, 0.0f, 0.0f};

__device__ __forceinline__ float reference_of(float top, float k) {
    return fminf(fmaxf(__builtin_ceilf(top * k), -kRefMost), kRefMost);
}

template <bool DOT>
__device__ __forceinline__ Stat joined(Stat a, Stat b) {
    const float ref = fmaxf(a.ref, b.ref), da = a.ref - ref, db = b.ref - ref;
    const float fa = exp2_of(da), fb = exp2_of(db);
    return {ref, a.sum * fa + b.sum * fb, DOT ? fa * (a.dot + da * a.sum) + fb * (b.dot + db * b.sum) : 0.0f};
}

// Joins the statistics of the first LANES lanes of a wavefront: the largest reference first, then plain sums.
template <bool DOT, int LANES>
__device__ __forceinline__ Stat join_wave(Stat s) {
    Stat r;
    r.ref = wave_max<LANES>(s.ref);
    const float d = s.ref - r.ref, f = exp2_of(d);              // a power of two: exact
    r.sum = wave_sum<LANES>(s.sum * f);
    r.dot = DOT ? wave_sum<LANES>(f * (s.dot + d * s.sum)) : 0.0f;
    return r;
}

// Joins the statistics of all lanes of a workgroup (up to 16 wavefronts); every lane gets the result.  `shared` may be
// used again only behind another barrier.
template <bool DOT, int BLOCK>
__device__ __forceinline__ Stat join_block(Stat s, Stat* shared) {
    static_assert(BLOCK <= 1024, "one entry per wavefront, at most 16");
    s = join_wave<DOT, 64>(s);
    if constexpr (BLOCK > 64) {
        if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = s;
        __syncthreads();
        const int lane = threadIdx.x & 63;
        s = lane < BLOCK / 64 ? shared[lane] : kNoStat;
        s = join_wave<DOT, 16>(s);
    }
    return s;
}

// What the row's softmax is computed from: 2^((z - shift) k - ref) / (rest + hot), hot being the target's term and rest and
// dot the sums over the others.
struct Row {
    float shift, ref, rest, dot, hot;
    __device__ __forceinline__ float sum() const { return rest + hot; }
};

// A row from the statistics of all logits but the target's, and that one.
__device__ __forceinline__ Row row_of(const Stat& s, float zt, float k) {
    Row r;
    r.shift = 0.0f;
    r.ref = fmaxf(s.ref, reference_of(zt, k));
    const float d = s.ref - r.ref, f = exp2_of(d);              // a power of two: exact
    r.rest = s.sum * f;
    r.dot = f * (s.dot + d * s.sum);
    r.hot = exp2_of(__builtin_fmaf(zt, k, -r.ref));
    return r;
}

template <int BLOCK>
__device__ __forceinline__ float max_block(float v, float* shared) {
    v = wave_max<64>(v);
    if constexpr (BLOCK > 64) {
        if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
        __syncthreads();
        const int lane = threadIdx.x & 63;
        v = wave_max<16>(lane < BLOCK / 64 ? shared[lane] : -INFINITY);
    }
    return v;
}

// Calls f(index, element) for all elements of a row, six loads of a lane on the way at once (one: a batch of NaN takes twice as long;
// eight: the row kernels' registers spill around the call).
template <typename T, int BLOCK, typename Fn>
__device__ __forceinline__ void for_elements(const char* row, int vocab, Fn f) {
    int j = threadIdx.x;
    for (; j < vocab - 5 * BLOCK; j += 6 * BLOCK) {
        float z[6];
#pragma unroll
        for (int i = 0; i < 6; i++) z[i] = T::one(row, j + i * BLOCK);
#pragma unroll
        for (int i = 0; i < 6; i++) f(j + i * BLOCK, z[i]);
    }
    for (; j < vocab; j += BLOCK) f(j, T::one(row, j));
}

// The rare rows: maximum first, then the sums with it subtracted, one element at a time.
template <typename T, int BLOCK>
__device__ __attribute__((noinline)) Row row_by_maximum(const char* row, int vocab, int target, float k, Stat* shared) {
    float top = -INFINITY;
    for_elements<T, BLOCK>(row, vocab, [&](int, float z) { top = fmaxf(top, z); });
    __syncthreads();                                  // `shared` held the row's first result
    top = max_block<BLOCK>(top, (float*)shared);
    __syncthreads();
    Stat s = {0.0f, 0.0f, 0.0f};
    for_elements<T, BLOCK>(row, vocab, [&](int j, float z) {
        const float d = (z - top) * k, e = exp2_of(d);
        s.sum += j == target ? 0.0f : e;
        s.dot = j == target ? s.dot : __builtin_fmaf(e, fmaxf(d, kLeastD), s.dot);
    });
    s = join_block<true, BLOCK>(s, shared);
    return {top, 0.0f, s.sum, s.dot, exp2_of((T::one(row, target) - top) * k)};
}

__device__ __forceinline__ bool ordinary(float sum) { return sum > 0.0f && sum < INFINITY; }

struct RowValues {
    float lse, logp, entropy, log2_sum;
};

// lse, log-probability of a target with logit zt, and entropy (nats).  The sum's exponent is folded into the integer
// reference, so that what is rounded is of the size of the result.
__device__ __forceinline__ RowValues row_values(const Row& row, float zt, float k, float inv_t) {
    int e;
    const float sum = row.sum(), mant = frexpf(sum, &e);
    const float ref = row.ref + (float)e, lm = log2f(mant);
    RowValues v;
    v.log2_sum = (float)e + lm;
    v.lse = __builtin_fmaf(ref, kLn2Hi, __builtin_fmaf(ref, kLn2Lo, kLn2 * lm));
    if (row.shift != 0.0f) v.lse = row.shift * inv_t + v.lse;
    v.logp = row.hot > row.rest ? 0.0f - log1pf(row.rest / row.hot) : (__builtin_fmaf(zt - row.shift, k, -ref) - lm) * kLn2;
    // - p log p of the target, and of the others: log2 p = d - log2 sum
    const float own = row.hot > 0.0f ? row.hot * v.logp : 0.0f;
    v.entropy = (0.0f - (own + (row.dot - row.rest * v.log2_sum) * kLn2)) / sum;
    return v;
}

__device__ __forceinline__ int64_t target_at(const void* targets, int wide, int64_t r) {
    return wide ? ((const RLX_GLOBAL int64_t*)targets)[r] : (int64_t)((const RLX_GLOBAL int32_t*)targets)[r];
}

// Statistics of up to N groups that a lane holds in registers, and of one loose logit (-inf: none).
template <typename T, int N, bool DOT>
__device__ __forceinline__ Stat held_statistics(u32x4 (&held)[N], float loose, float k) {
    typename T::Top top = T::no_top();
#pragma unroll
    for (int n = 0; n < N; n++) T::add_top(top, held[n]);
    Stat s = {reference_of(fmaxf(T::top_of(top), loose), k), 0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < N; n++) {
        float z[T::PER];
        forget(held[n]);
        T::unpack(held[n], z);
#pragma unroll
        for (int i = 0; i < T::PER; i++) {
            const float d = __builtin_fmaf(z[i], k, -s.ref), e = exp2_of(d);
            s.sum += e;
            if constexpr (DOT) s.dot = __builtin_fmaf(e, fmaxf(d, kLeastD), s.dot);
        }
    }
    const float d = __builtin_fmaf(loose, k, -s.ref), e = exp2_of(d);
    s.sum += e;
    if constexpr (DOT) s.dot = __builtin_fmaf(e, fmaxf(d, kLeastD), s.dot);
    return s;
}

// The gradient of a row: 2^d (b0 + b1 d) with d = (z - shift) k - ref, and `hot` at the target.
struct RowGrad {
    float shift, ref, b0, b1, hot;
};

// g: gradient of logp; c: gradient of the entropy (both with 1/temperature in them).
__device__ __forceinline__ RowGrad row_gradient(const Row& row, const RowValues& v, float g, float c) {
    const float inv = 1.0f / row.sum();
    RowGrad q;
    q.shift = row.shift;
    q.ref = row.ref;
    // log p = ln2 (d - log2 sum), so p (g + c (log p + H)) = p (g + c (H - ln2 log2 sum) + c ln2 d)
    q.b0 = -inv * (g + c * (v.entropy - kLn2 * v.log2_sum));
    q.b1 = -inv * (c * kLn2);
    q.hot = g * (row.rest * inv);                              // g (1 - p)
    if (row.hot > 0.0f) q.hot -= c * (row.hot * inv) * (v.logp + v.entropy);
    return q;
}

template <bool DOT>
__device__ __forceinline__ float grad_of(const RowGrad& q, float z, float k) {
    const float d = __builtin_fmaf(z, k, -q.ref), e = exp2_of(d);
    if constexpr (DOT) return e * __builtin_fmaf(q.b1, fmaxf(d, kLeastD), q.b0);
    else return e * q.b0;
}

template <bool DOT>
__device__ __forceinline__ float grad_by_maximum(const RowGrad& q, float z, float k) {
    const float d = (z - q.shift) * k, e = exp2_of(d);
    if constexpr (DOT) return e * __builtin_fmaf(q.b1, fmaxf(d, kLeastD), q.b0);
    else return e * q.b0;
}

// Writes `value` over a whole row (zeros of an ignored one, NaN of one with a bad target).
template <typename T, int BLOCK>
__device__ void fill_row(char* out, int vocab, float value) {
    constexpr int PER = T::PER;
    const int groups = vocab / PER;
    float f[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) f[i] = value;
    const u32x4 v = T::pack(f);
    for (int g = threadIdx.x; g < groups; g += BLOCK) store16(out + (int64_t)g * 16, v);
    const int j = groups * PER + threadIdx.x;
    if (j < vocab) T::put(out, j, value);
}

// The gradient of one group, with the target's own if it is in it (at < 0 or >= PER: it is not).
template <typename T, bool DOT>
__device__ __forceinline__ u32x4 grad_group(const RowGrad& q, u32x4 v, float k, int at) {
    float z[T::PER];
    T::unpack(v, z);
#pragma unroll
    for (int i = 0; i < T::PER; i++) z[i] = grad_of<DOT>(q, z[i], k);
    if ((unsigned)at < (unsigned)T::PER) {
#pragma unroll
        for (int i = 0; i < T::PER; i++)
            if (i == at) z[i] = q.hot;
    }
    return T::pack(z);
}

// A rare row's gradient: elements from .. to, one at a time.
template <typename T, int BLOCK, bool DOT>
__device__ __attribute__((noinline)) void rare_gradient(RowGrad q, const char* row, char* out, int from, int to,
                                                        float k, int target) {
    for (int j = from + threadIdx.x; j < to; j += BLOCK) {
        const float d = grad_by_maximum<DOT>(q, T::one(row, j), k);
        T::put(out, j, j == target ? q.hot : d);
    }
}

// --- kernels over logits ---------------------------------------------------------------------------------------------

struct RowOutputs {
    float *logp, *lse, *entropy;
};

__device__ __forceinline__ void put_values(const RowOutputs& o, uint32_t r, const RowValues& v) {
    o.logp[r] = v.logp;
    o.lse[r] = v.lse;
    if (o.entropy) o.entropy[r] = v.entropy;
}

// Statistics of one chunk of a row (BLOCK * NG groups) per workgroup: consecutive workgroups read consecutive memory, so
// that the addresses in flight stay a narrow window, and a few rows still fill the chip.  A row of one chunk is
// finished here, with `o`; the chunks of longer rows are added up by the joining launch.
// Bound by HBM reads: 4,096 rows of 151,936 FP16 take 180 us in 32 KiB chunks (6.9 TB/s; the vector units are busy for 115
// of them), 190 in 16 KiB, 333 in 4 KiB, 206 with a workgroup walking its row.
template <typename T, int BLOCK, int NG, bool DOT, bool ONCE>
__global__ __launch_bounds__(BLOCK) void chunk_statistics_kernel(Logits x, const void* __restrict__ targets, int wide,
                                                                 const uint8_t* __restrict__ mask, float k, float inv_t,
                                                                 RowOutputs o, Stat* __restrict__ partials,
                                                                 float* __restrict__ target_logits,
                                                                 uint32_t* __restrict__ ticket, uint32_t first) {
    __shared__ Stat shared[BLOCK / 64];
    const uint32_t r = first + blockIdx.y, c = blockIdx.x;
    const int tid = threadIdx.x;
    if (ticket && r == 0 && c == 0 && tid == 0) *ticket = 0;       // for the launch that follows
    const int64_t t = target_at(targets, wide, r);
    if (t < 0 || t >= x.vocab || (mask && mask[r] == 0)) {
        const float v = t < 0 ? 0.0f : NAN;
        if (o.logp && tid == 0) put_values(o, r, {v, v, v, v});
        return;
    }
    const char* row = x.data + row_at(x, r) * T::SIZE;
    const int groups = x.vocab / T::PER, at = (int)c * BLOCK * NG + tid, j = groups * T::PER + tid;
    u32x4 held[NG];
    load_groups<T, NG, BLOCK, ONCE>(held, row, at, groups);
    drop_target<T, NG, BLOCK>(held, (int)c * BLOCK * NG, (int)t);
    const float loose = c == 0 && j < x.vocab && j != (int)t ? T::one(row, j) : -INFINITY;
    const bool finish = o.logp != nullptr;
    const float zt = finish || (target_logits && c == 0) ? T::one(row, t) : 0.0f;
    Stat s = held_statistics<T, NG, DOT>(held, loose, k);
    s = join_block<DOT, BLOCK>(s, shared);
    if (finish) {
        Row rv = row_of(s, zt, k);
        if (!ordinary(rv.sum())) rv = row_by_maximum<T, BLOCK>(row, x.vocab, (int)t, k, shared);
        if (tid == 0) put_values(o, r, row_values(rv, zt, k, inv_t));
    } else if (tid == 0) {
        partials[(int64_t)r * gridDim.x + c] = s;
        if (target_logits && c == 0) target_logits[r] = zt;
    }
}

// A row's statistics from its chunks, by every wavefront for itself.
template <bool DOT>
__device__ __forceinline__ Stat join_chunks(const Stat* __restrict__ partials, int chunks) {
    const int lane = threadIdx.x & 63;
    Stat s = lane < chunks ? partials[lane] : kNoStat;
    for (int c = lane + 64; c < chunks; c += 64) s = joined<DOT>(s, partials[c]);
    return join_wave<DOT, 64>(s);
}

constexpr int kChunkBlock = 256, kJoinBlock = 256, kJoinRows = kJoinBlock / 64;

// A row per wavefront (a workgroup per row took 2 to 4 us longer for 4,096 and 8,192 rows); the rare rows of a workgroup are
// done again by all of it, one after the other.
template <typename T, bool DOT>
__global__ __launch_bounds__(kJoinBlock) void token_logprob_join_kernel(Logits x, const void* __restrict__ targets, int wide,
                                                                        float k, float inv_t,
                                                                        const Stat* __restrict__ partials, int chunks,
                                                                        RowOutputs o, uint32_t first, uint32_t rows) {
    __shared__ Stat shared[kJoinBlock / 64];
    __shared__ int again[kJoinRows];
    const uint32_t wave = threadIdx.x >> 6, in_launch = blockIdx.x * kJoinRows + wave, r = first + in_launch;
    const bool head = (threadIdx.x & 63) == 0;
    bool rare = false;
    if (in_launch < rows) {
        const int64_t t = target_at(targets, wide, r);
        if (t < 0 || t >= x.vocab) {
            const float v = t < 0 ? 0.0f : NAN;
            if (head) put_values(o, r, {v, v, v, v});
        } else {
            const float zt = T::one(x.data + row_at(x, r) * T::SIZE, t);
            const Row rv = row_of(join_chunks<DOT>(partials + (int64_t)r * chunks, chunks), zt, k);
            rare = !ordinary(rv.sum());
            if (head && !rare) put_values(o, r, row_values(rv, zt, k, inv_t));
        }
    }
    if (head) again[wave] = rare ? 1 : 0;
    __syncthreads();
    for (uint32_t w = 0; w < kJoinRows; w++) {
        if (!again[w]) continue;
        const uint32_t rr = first + blockIdx.x * kJoinRows + w;
        const char* row = x.data + row_at(x, rr) * T::SIZE;
        const int64_t t = target_at(targets, wide, rr);
        const Row rv = row_by_maximum<T, kJoinBlock>(row, x.vocab, (int)t, k, shared);
        if (threadIdx.x == 0) put_values(o, rr, row_values(rv, T::one(row, t), k, inv_t));
    }
}

// dx from the saved lse (and entropy), 4 KiB of a row per workgroup.  Bound by HBM, reads and writes: 4,096 rows of 151,936
// BF16, a quarter of them ignored, 335 us = 6.5 TB/s (8 KiB per workgroup 357, 16 KiB 372, a workgroup per row 437); rows
// that do not start on 16 bytes do better with half the lanes and two groups each (50,257 BF16: 143 against 156 us).
// p = exp(z - lse) is formed as 2^((z/T - lse) log2 e), the difference first; what it inherits is the rounding of lse and of
// the temperature's reciprocal, a few u |lse| of p (u = 2^-24) and, at a target, as much over 1 - p of 1 - p.  Where log p of the target is given, its own gradient
// comes from that and keeps the precision of 1 - p.  Rows whose lse is so large that even log V drowns in its rounding (nothing but
// the type's lowest value), or that overflowed, are worked out again from their logits.
template <typename T, int BLOCK, int NG, bool DOT, bool ONCE>
__global__ __launch_bounds__(BLOCK) void token_logprob_backward_kernel(
    Logits x, Logits dx, const void* __restrict__ targets, int wide, float k, float inv_t, const float* __restrict__ lse,
    const float* __restrict__ entropy, const float* __restrict__ logp, const float* __restrict__ dlogp,
    const float* __restrict__ dentropy, uint32_t first) {
    constexpr int PER = T::PER;
    __shared__ Stat shared[BLOCK / 64];
    const uint32_t r = first + blockIdx.y;
    const int tid = threadIdx.x;
    const int64_t t = target_at(targets, wide, r);
    const char* row = x.data + row_at(x, r) * T::SIZE;
    char* out = dx.data + row_at(dx, r) * T::SIZE;
    const float g = dlogp[r], c = DOT ? dentropy[r] : 0.0f, l = lse[r], h = DOT ? entropy[r] : 0.0f;
    const bool bad = t >= x.vocab, none = t < 0 || (!bad && g == 0.0f && c == 0.0f);
    const int groups = x.vocab / PER, at = (int)blockIdx.x * BLOCK * NG + tid, j = groups * PER + tid;
    const bool has_loose = blockIdx.x == 0 && j < x.vocab;
    if (bad || none) {
        const float value = bad ? NAN : 0.0f;
        float f[PER];
#pragma unroll
        for (int i = 0; i < PER; i++) f[i] = value;
        const u32x4 v = T::pack(f);
#pragma unroll
        for (int n = 0; n < NG; n++)
            if (at + n * BLOCK < groups) store16_once(out + (int64_t)(at + n * BLOCK) * 16, v);
        if (has_loose) T::put(out, j, value);
        return;
    }
    const float gs = g * inv_t, cs = c * inv_t;
    const int target = (int)t;
    if (fabsf(l) >= kMostLse) {
        if (blockIdx.x != 0) return;                        // the first workgroup does the row by itself: dx may be x
        const Row rv = row_by_maximum<T, BLOCK>(row, x.vocab, target, k, shared);
        const RowValues v = row_values(rv, T::one(row, t), k, inv_t);
        __syncthreads();                                    // every lane has read what is overwritten now
        rare_gradient<T, BLOCK, DOT>(row_gradient(rv, v, gs, cs), row, out, 0, x.vocab, k, target);
        return;
    }
    auto grad = [&](float z) {
        const float lp = __builtin_fmaf(z, inv_t, -l), p = exp2_of(lp * kLog2e);
        if constexpr (DOT) return -p * __builtin_fmaf(cs, fmaxf(lp, kLeastD) + h, gs);
        else return -p * gs;
    };
    auto grad_hot = [&](float z) {                          // the target's: 1 - p = -expm1(log p)
        const float lp = logp ? logp[r] : __builtin_fmaf(z, inv_t, -l);
        float d = -gs * expm1f(lp);
        if constexpr (DOT) d -= exp2_of(lp * kLog2e) * cs * (fmaxf(lp, kLeastD) + h);
        return d;
    };
    u32x4 held[NG];
    load_groups<T, NG, BLOCK, ONCE>(held, row, at, groups);
    const float loose = has_loose ? T::one(row, j) : 0.0f;
#pragma unroll
    for (int n = 0; n < NG; n++) {
        float z[PER];
        T::unpack(held[n], z);
        const int in = target - (at + n * BLOCK) * PER;
        float hot = 0.0f;
        if ((unsigned)in < (unsigned)PER) {
#pragma unroll
            for (int e = 0; e < PER; e++)
                if (e == in) hot = grad_hot(z[e]);
        }
#pragma unroll
        for (int e = 0; e < PER; e++) z[e] = grad(z[e]);
        if ((unsigned)in < (unsigned)PER) {
#pragma unroll
            for (int e = 0; e < PER; e++)
                if (e == in) z[e] = hot;
        }
        if (at + n * BLOCK < groups) store16_once(out + (int64_t)(at + n * BLOCK) * 16, T::pack(z));
    }
    if (has_loose) {
        T::put(out, j, j == target ? grad_hot(loose) : grad(loose));
    }
}

// --- sequences, weights, per-token losses --------------------------------------------------------------------------------

struct Batch {              // sequences of a packed or padded batch of tokens
    const uint8_t* mask;
    const int32_t* cu;
    int64_t tokens, n_seqs;
};

// First token and length of a sequence, kept inside the arrays whatever the offsets hold.
__device__ __forceinline__ void sequence_at(const Batch& b, int64_t s, int64_t& begin, int64_t& end) {
    if (b.cu) {
        begin = ((const RLX_GLOBAL int32_t*)b.cu)[s];
        end = ((const RLX_GLOBAL int32_t*)b.cu)[s + 1];
        begin = begin < 0 ? 0 : begin > b.tokens ? b.tokens : begin;
        end = end < begin ? begin : end > b.tokens ? b.tokens : end;
    } else {
        const int64_t n = b.tokens / b.n_seqs;
        begin = s * n;
        end = begin + n;
    }
}

// How many of the offsets lo .. hi - 1 (ascending) and all in front of them are at most t, given that it is lo .. hi.
template <typename Ptr>
__device__ __forceinline__ int64_t offsets_up_to(Ptr cu, int64_t lo, int64_t hi, int64_t t) {
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (cu[mid] <= t) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// The same by a whole wavefront for one t: 64 offsets at a time, so two or three dependent loads instead of ten.
__device__ __forceinline__ int64_t wave_offsets_up_to(const RLX_GLOBAL int32_t* cu, int64_t lo, int64_t hi, int64_t t) {
    const int lane = threadIdx.x & 63;
    while (lo < hi) {
        const int64_t step = (hi - lo + 63) >> 6, at = lo + (lane + 1) * step - 1;
        const int64_t n = __builtin_popcountll(__ballot(at < hi && cu[at < hi ? at : hi - 1] <= t));
        lo = lo + n * step < hi ? lo + n * step : hi;
        hi = lo + step - 1 < hi ? lo + step - 1 : hi;
    }
    return lo;
}

struct Policy {             // rlx_policy_args as the kernels take it
    const float *old_logp, *ref_logp, *advantages, *entropy;
    Batch batch;
    double log_high, log_low;      // borders of the clip
    double high, low;              // 1 + clip_high, 1 - clip_low
    double norm;
    float kl_coef, entropy_coef, grad_scale;
    int reduction, per_token;
};

// What a token, a workgroup or a batch adds to the statistics.
struct Terms {
    double policy, kl, entropy;      // weighted
    double clipped, ratio;
    int64_t count;
};

// exp(x), exp(x) - 1 and exp(x) - 1 - x in FP64, within 2^-41, 2^-39 and 2^-37 of themselves.  x = n ln 2 + r with
// |r| <= ln 2 / 2, and exp(r) = 1 + r + r^2 q(r) with q the Taylor series up to r^10 (the first term left out is below 2^-42).
// For n = 0 the last two are r + r^2 q and r^2 q as they stand, where differences of exp(x) would lose everything.
// The factors of the series are scalar operands: left to itself the compiler puts each into a pair of vector registers, and
// policy_loss_kernel has 82 of them, not 68.
struct Exp {
    double e, less1, less_x;
};

__device__ __forceinline__ Exp exp_of(double x) {
    const double top = x > 2000.0 ? 2000.0 : x, in = top < -2000.0 ? -2000.0 : top;      // NaN stays
    const double n = __builtin_rint(in * 1.4426950408889634), r = __builtin_fma(n, -0.6931471805599453, in);
    double q = 1.0 / 3628800.0;
    for (const double c : {1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0, 1.0 / 120.0, 1.0 / 24.0, 1.0 / 6.0, 0.5})
        asm("v_fma_f64 %0, %1, %2, %3" : "=v"(q) : "v"(q), "v"(r), "s"(c));
    q *= r * r;
    const double rq = r + q;
    Exp o;
    o.e = __builtin_amdgcn_ldexp(1.0 + rq, (int)n);
    const double far = o.e - 1.0;
    o.less1 = n == 0.0 ? rq : far;
    o.less_x = n == 0.0 ? q : far == (double)INFINITY ? far : far - x;
    return o;
}

// What follows from the log-probabilities is computed in FP64 and rounded once, as a gradient or as a sum.  (Differences of
// FP32 values are exact there, so the side of the clip's border is, too.)  With weights, products and exponentials in FP32,
// up to a quarter of the gradients were off by more than that, by up to three roundings; it took 16.8 us for 1.6 M tokens, and
// 19.0 this way.
struct TokenLoss {
    double policy, kl, ratio, slope;     // slope: gradient of the token's loss by its log-probability
    bool clipped;
};

// old and ref are used only where the batch has them.
__device__ __forceinline__ TokenLoss token_loss(const Policy& a, float logp, float old, float ref, float advantage) {
    TokenLoss o;
    const double lr = a.old_logp ? (double)logp - (double)old : 0.0, adv = (double)advantage;
    o.clipped = advantage >= 0.0f ? lr > a.log_high : lr < a.log_low;
    o.ratio = exp_of(lr).e;
    // min(rho A, clip(rho) A) without the product of an infinite rho and A = 0
    o.policy = -(adv * (o.clipped ? (advantage >= 0.0f ? a.high : a.low) : o.ratio));
    o.slope = o.clipped ? 0.0 : -(adv * o.ratio);
    o.kl = 0.0;
    if (a.ref_logp) {
        const Exp x = exp_of((double)ref - (double)logp);
        o.kl = x.less_x;
        if (a.kl_coef != 0.0f) o.slope -= (double)a.kl_coef * x.less1;
    }
    return o;
}

__device__ __forceinline__ double weight_of(const Policy& a, int64_t count) {
    if (a.reduction == RLX_LOSS_SUM) return a.norm;
    if (count < 1) count = 1;              // only with offsets that do not ascend
    if (a.reduction == RLX_LOSS_TOKEN_MEAN) return a.norm / (double)count;
    return a.norm / ((double)a.batch.n_seqs * (double)count);
}

// Sums of N values over a workgroup; every lane gets them.  `shared` (N per wavefront) may be used again only behind
// another barrier.
template <int BLOCK, int N, typename T8>
__device__ __forceinline__ void sum_block(T8 (&v)[N], T8* shared) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = wave_sum8(v[i]);
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < N; i++) shared[(threadIdx.x >> 6) * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = shared[i];
    for (int w = 1; w < BLOCK / 64; w++)
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += shared[w * N + i];
}

template <int BLOCK>
__device__ __forceinline__ int64_t sum_block(int64_t v, int64_t* shared) {
    int64_t one[1] = {v};
    sum_block<BLOCK, 1>(one, shared);
    return one[0];
}

template <int BLOCK>
__device__ __forceinline__ Terms sum_terms(const Terms& t, double* shared, int64_t* shared_n) {
    double v[5] = {t.policy, t.kl, t.entropy, t.clipped, t.ratio};
    sum_block<BLOCK, 5>(v, shared);
    return {v[0], v[1], v[2], v[3], v[4], sum_block<BLOCK>(t.count, shared_n)};
}

constexpr int kTokenBlock = 256;

__device__ __forceinline__ bool counts(const Batch& b, const void* targets, int wide, int64_t t) {
    if (b.mask && ((const RLX_GLOBAL uint8_t*)b.mask)[t] == 0) return false;
    return !targets || target_at(targets, wide, t) >= 0;
}

typedef uint32_t u32x4_bytes __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32_bytes __attribute__((aligned(1)));

__device__ __forceinline__ u32x4 load_mask16(const uint8_t* p) { return *(const RLX_GLOBAL u32x4_bytes*)(const RLX_GLOBAL uint8_t*)p; }
__device__ __forceinline__ uint32_t load_mask4(const uint8_t* p) { return *(const RLX_GLOBAL u32_bytes*)(const RLX_GLOBAL uint8_t*)p; }

// Bytes of a word that are not 0, as their top bits.
__device__ __forceinline__ uint32_t nonzero_bytes(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w) & 0x80808080u; }

__device__ __forceinline__ int masked_in(u32x4 v) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) n += __builtin_popcount(nonzero_bytes(v[i]));
    return n;
}

constexpr int64_t kMostInline = 1024;         // sequences whose counts a wavefront adds up by itself

// How many tokens of each sequence count; with `info` also, per token, its sequence, or -1 if it is ignored.
__global__ __launch_bounds__(kTokenBlock) void sequence_counts_kernel(Batch b, const void* __restrict__ targets, int wide,
                                                                      int32_t* __restrict__ out, int32_t* __restrict__ info) {
    __shared__ int64_t shared[kTokenBlock / 64];
    for (int64_t s = blockIdx.x; s < b.n_seqs; s += gridDim.x) {
        int64_t begin, end, n = 0;
        sequence_at(b, s, begin, end);
        if (info) {
            for (int64_t t = begin + threadIdx.x; t < end; t += kTokenBlock) {
                const bool in = counts(b, targets, wide, t);
                n += in ? 1 : 0;
                info[t] = in ? (int32_t)s : -1;
            }
        } else if (!b.mask) {
            n = threadIdx.x == 0 ? end - begin : 0;
        } else {
            int64_t t = begin + threadIdx.x * 16;
            for (; t + 16 <= end; t += kTokenBlock * 16) n += masked_in(load_mask16(b.mask + t));
            for (int64_t u = t; u < end && u < t + 16; u++) n += ((const RLX_GLOBAL uint8_t*)b.mask)[u] != 0;
        }
        n = sum_block<kTokenBlock>(n, shared);
        if (threadIdx.x == 0) out[s] = (int32_t)n;
        __syncthreads();
    }
    for (int64_t s = b.n_seqs + threadIdx.x; blockIdx.x == 0 && s < kMostInline; s += kTokenBlock) out[s] = 0;
    if (info && b.cu) {                       // in front of the first and behind the last sequence
        int64_t lo, hi, unused;
        sequence_at(b, 0, lo, unused);
        sequence_at(b, b.n_seqs - 1, unused, hi);
        const int64_t step = (int64_t)gridDim.x * kTokenBlock, at = (int64_t)blockIdx.x * kTokenBlock + threadIdx.x;
        for (int64_t t = at; t < lo; t += step) info[t] = -1;
        for (int64_t t = hi + at; t < b.tokens; t += step) info[t] = -1;
    }
}

// The counts of all sequences, by one wavefront: kMostInline of them, those behind the last sequence 0, in one go (a loop
// over 512 counts, a load at a time, took 6 us).
__device__ __forceinline__ int64_t batch_count(const int32_t* __restrict__ seq_counts) {
    const RLX_GLOBAL u32x4* at = (const RLX_GLOBAL u32x4*)seq_counts + (threadIdx.x & 63);
    const u32x4 a = at[0], b = at[64], c = at[128], d = at[192];
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) n += a[i] + b[i] + c[i] + d[i];
    return wave_sum8((int64_t)n);
}

// Leaves the sum in place of the first count, for batches of more sequences.
__global__ __launch_bounds__(1024) void total_count_kernel(int32_t* __restrict__ seq_counts, int64_t n_seqs) {
    __shared__ int64_t shared[16];
    int64_t n = 0;
    for (int64_t s = threadIdx.x; s < n_seqs; s += 1024) n += seq_counts[s];
    n = sum_block<1024>(n, shared);
    if (threadIdx.x == 0) seq_counts[0] = (int32_t)n;
}

// What the weight of a token of sequence s divides by, by one wavefront.
__device__ __forceinline__ int64_t count_for(const Policy& a, const int32_t* __restrict__ seq_counts, int64_t s) {
    if (a.reduction == RLX_LOSS_SUM) return 1;
    if (a.reduction == RLX_LOSS_SEQUENCE_MEAN) return seq_counts[s];
    return a.batch.n_seqs > kMostInline ? (int64_t)seq_counts[0] : batch_count(seq_counts);
}

// Four consecutive floats at any 4-byte boundary.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ f32x4_any load4(const float* p) { return *(const RLX_GLOBAL f32x4_any*)(const RLX_GLOBAL float*)p; }
__device__ __forceinline__ void store4(float* p, f32x4_any v) { *(RLX_GLOBAL f32x4_any*)(RLX_GLOBAL float*)p = v; }

// Four consecutive tokens of the per-token arrays.  Every load is unconditional (arrays that the batch does not have are
// stood for by logp): one under a condition would be waited for before the next is issued.
struct Tokens4 {
    f32x4_any logp, old, ref, entropy, advantage;
    uint32_t in;                   // top bit of byte i: token i is not masked
};

// Tokens t .. t + 3, which must lie in the arrays.
__device__ __forceinline__ Tokens4 load_tokens(const Policy& a, const float* logp, int64_t t) {
    Tokens4 o;
    o.logp = load4(logp + t);
    o.old = load4((a.old_logp ? a.old_logp : logp) + t);
    o.ref = load4((a.ref_logp ? a.ref_logp : logp) + t);
    o.entropy = load4((a.entropy ? a.entropy : logp) + t);
    o.advantage = load4((a.per_token ? a.advantages : logp) + t);
    const uint32_t in = load_mask4(a.batch.mask ? a.batch.mask + t : (const uint8_t*)(logp + t));
    o.in = a.batch.mask ? nonzero_bytes(in) : 0x80808080u;
    if (!a.entropy) o.entropy = f32x4_any{0.0f, 0.0f, 0.0f, 0.0f};
    return o;
}

// Bits of a quad at `at` whose tokens lie in from .. to - 1.
__device__ __forceinline__ uint32_t tokens_within(int64_t at, int64_t from, int64_t to) {
    uint32_t in = 0x80808080u;
    if (from > at) in = from - at >= 4 ? 0 : in << (8 * (from - at));
    if (to < at + 4) in &= to <= at ? 0 : 0x80808080u >> (8 * (at + 4 - to));
    return in;
}

// What a lane adds up over its few tokens.
struct LaneTerms {
    double policy, kl, entropy, ratio;     // the first three weighted
    int clipped, count;
};

// A token's weight as it is used: in the loss, in the gradients of logp and of the entropy.
struct Weight {
    double loss, logp;
    float entropy;
};

__device__ __forceinline__ Weight weights(const Policy& a, int64_t count) {
    const double w = weight_of(a, count), g = w * (double)a.grad_scale;
    return {w, g, (float)(g * -(double)a.entropy_coef)};
}

// One token's share of the loss; returns its gradient.
__device__ __forceinline__ float add_token(const Policy& a, const Weight& w, float logp, float old, float ref, float entropy,
                                           float advantage, LaneTerms& v) {
    const TokenLoss o = token_loss(a, logp, old, ref, advantage);
    v.policy += w.loss * o.policy;
    v.kl += w.loss * o.kl;
    v.entropy += w.loss * (double)entropy;
    v.ratio += o.ratio;
    v.clipped += o.clipped ? 1 : 0;
    v.count++;
    return (float)(w.logp * o.slope);
}

__device__ __forceinline__ Terms terms_of(const LaneTerms& v) {
    return {v.policy, v.kl, v.entropy, (double)v.clipped, v.ratio, v.count};
}

// --- the workgroup of a launch that finishes last ------------------------------------------------------------------------
// Every workgroup publishes its terms with device-scope stores, waits until they have arrived and takes a ticket; the one
// that draws the last ticket adds all terms up, in their order, with device-scope loads.  Tickets decide who adds, never in
// which order.  The launch in front clears the counter.  For launches of up to kFewRows workgroups that take part.

__device__ __forceinline__ void publish8(void* p, double x) {
    __hip_atomic_store((uint64_t*)p, __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ double published8(const void* p) {
    return __builtin_bit_cast(double, __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Publishes terms[block] and says, to every lane, whether this workgroup is the last of `blocks`.
__device__ __forceinline__ bool last_with(const Terms& t, Terms* terms, uint32_t block, uint32_t blocks, uint32_t* ticket,
                                          int* shared) {
    if (threadIdx.x < 64) {
        if (threadIdx.x == 0) {
            publish8(&terms[block].policy, t.policy);
            publish8(&terms[block].kl, t.kl);
            publish8(&terms[block].entropy, t.entropy);
            publish8(&terms[block].clipped, t.clipped);
            publish8(&terms[block].ratio, t.ratio);
            publish8(&terms[block].count, __builtin_bit_cast(double, t.count));
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // they have arrived before the ticket is taken
        if (threadIdx.x == 0) {
            *shared = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == blocks;
        }
    }
    __syncthreads();
    const bool last = *shared != 0;
    if (last) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    return last;
}

// The sum of all published terms, by the last workgroup.
template <int BLOCK>
__device__ __forceinline__ Terms sum_published(const Terms* terms, uint32_t blocks, double* shared, int64_t* shared_n) {
    Terms v = {0.0, 0.0, 0.0, 0.0, 0.0, 0};
    for (uint32_t i = threadIdx.x; i < blocks; i += BLOCK) {
        v.policy += published8(&terms[i].policy);
        v.kl += published8(&terms[i].kl);
        v.entropy += published8(&terms[i].entropy);
        v.clipped += published8(&terms[i].clipped);
        v.ratio += published8(&terms[i].ratio);
        v.count += __builtin_bit_cast(int64_t, published8(&terms[i].count));
    }
    return sum_terms<BLOCK>(v, shared, shared_n);
}

__device__ void write_stats(const Terms& v, float kl_coef, float entropy_coef, rlx_policy_stats* stats) {
    double loss = v.policy;
    if (kl_coef != 0.0f) loss += (double)kl_coef * v.kl;
    if (entropy_coef != 0.0f) loss -= (double)entropy_coef * v.entropy;
    const double m = v.count > 0 ? (double)v.count : 1.0;
    *stats = {(float)loss, (float)v.policy, (float)v.kl, (float)v.entropy, (float)(v.clipped / m), (float)(v.ratio / m),
              v.count};
}

constexpr int kTokensPerBlock = 4 * kTokenBlock;

// Policy loss over log-probabilities (of at least four tokens): a workgroup takes kTokensPerBlock tokens, a lane four in a
// row; the quads of the lanes at the end of the arrays move back into them.  The sequences of a workgroup's first
// and last token are searched once; only where they differ does a lane search between them.
// 1.6 M tokens with every input (46 MB): 19 us; the memory alone takes 9, and as all wavefronts are resident at once (72
// registers or fewer), it overlaps little with the arithmetic.  A token per lane took 37.  (The partial terms are added by a
// launch of its own, 4 us: with tickets, as few rows do it, 1,562 workgroups took 14 us longer.)
__global__ __launch_bounds__(kTokenBlock) void policy_loss_kernel(Policy a, const float* __restrict__ logp,
                                                                  const int32_t* __restrict__ seq_counts,
                                                                  float* __restrict__ dlogp, float* __restrict__ dentropy,
                                                                  Terms* __restrict__ partials) {
    __shared__ int64_t shared_n[kTokenBlock / 64];
    __shared__ double shared[5 * kTokenBlock / 64];
    const RLX_GLOBAL int32_t* cu = (const RLX_GLOBAL int32_t*)a.batch.cu;
    const int64_t n_seqs = a.batch.n_seqs, tokens = a.batch.tokens, begin = (int64_t)blockIdx.x * kTokensPerBlock;
    const int64_t own = begin + threadIdx.x * 4, t0 = own + 4 <= tokens ? own : tokens - 4;
    const int64_t end = begin + kTokensPerBlock < tokens ? begin + kTokensPerBlock : tokens;
    Tokens4 x = load_tokens(a, logp, t0);
    x.in &= tokens_within(t0, own, tokens);
    // offsets up to a token: its sequence is one less (0: in front of the first, n_seqs + 1: behind the last)
    uint32_t lo, hi, len = 1;
    if (cu) {
        lo = (uint32_t)wave_offsets_up_to(cu, 0, n_seqs + 1, begin);
        hi = (uint32_t)wave_offsets_up_to(cu, lo, n_seqs + 1, end - 1);
    } else {
        len = (uint32_t)(tokens / n_seqs);
        lo = (uint32_t)begin / len + 1;
        hi = (uint32_t)(end - 1) / len + 1;
    }
    const int64_t total = a.reduction == RLX_LOSS_TOKEN_MEAN ? count_for(a, seq_counts, 0) : 1;
    uint32_t at = lo, weighed = 0;
    if (lo != hi) at = cu ? (uint32_t)offsets_up_to(cu, lo, hi, t0) : (uint32_t)t0 / len + 1;
    Weight w = {0.0, 0.0, 0.0f};
    float advantage = 0.0f;
    LaneTerms v = {0.0, 0.0, 0.0, 0.0, 0, 0};
    f32x4_any g = {0.0f, 0.0f, 0.0f, 0.0f}, dh = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (cu) {
            while (at < hi && cu[at] <= t0 + i) at++;
        } else if (lo != hi) {
            at = ((uint32_t)t0 + i) / len + 1;
        }
        if ((x.in >> (8 * i) & 0x80u) && at >= 1 && at <= n_seqs) {
            if (weighed != at) {
                weighed = at;
                w = weights(a, a.reduction == RLX_LOSS_SEQUENCE_MEAN ? (int64_t)seq_counts[at - 1] : total);
                if (!a.per_token) advantage = a.advantages[at - 1];
            }
            g[i] = add_token(a, w, x.logp[i], x.old[i], x.ref[i], x.entropy[i], a.per_token ? x.advantage[i] : advantage, v);
            dh[i] = w.entropy;
        }
    }
    if (t0 == own) {
        store4(dlogp + t0, g);
        if (dentropy) store4(dentropy + t0, dh);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (t0 + i < own) continue;
            dlogp[t0 + i] = g[i];
            if (dentropy) dentropy[t0 + i] = dh[i];
        }
    }
    const Terms sum = sum_terms<kTokenBlock>(terms_of(v), shared, shared_n);
    if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

// The whole of a small batch in one launch of one workgroup: counts in LDS (integers, so that the order of their
// additions says nothing), then losses, gradients and statistics.  A lane takes the tokens tid, tid + BLOCK, ...
constexpr int kSmallPerLane = 4, kSmallTokens = 512 * kSmallPerLane, kSmallSeqs = 1024;

template <int BLOCK>
__global__ __launch_bounds__(BLOCK) void policy_loss_small_kernel(Policy a, const float* __restrict__ logp,
                                                                  float* __restrict__ dlogp, float* __restrict__ dentropy,
                                                                  rlx_policy_stats* __restrict__ stats) {
    __shared__ double shared[5 * BLOCK / 64];
    __shared__ int64_t shared_n[BLOCK / 64], shared_m[BLOCK / 64];
    __shared__ int32_t offsets[kSmallSeqs + 1], in_seq[kSmallSeqs];
    const int n_seqs = (int)a.batch.n_seqs, tokens = (int)a.batch.tokens, tid = threadIdx.x;
    float lp[kSmallPerLane], old[kSmallPerLane], ref[kSmallPerLane], entropy[kSmallPerLane], adv[kSmallPerLane];
    int at[kSmallPerLane];
    bool in[kSmallPerLane];
    if (tokens > 0) {
#pragma unroll
        for (int i = 0; i < kSmallPerLane; i++) {           // unconditional loads, the last token's behind the end
            const int t = tid + i * BLOCK < tokens ? tid + i * BLOCK : tokens - 1;
            lp[i] = logp[t];
            old[i] = (a.old_logp ? a.old_logp : logp)[t];
            ref[i] = (a.ref_logp ? a.ref_logp : logp)[t];
            entropy[i] = (a.entropy ? a.entropy : logp)[t];
            adv[i] = (a.per_token ? a.advantages : logp)[t];
            const uint8_t m = a.batch.mask ? a.batch.mask[t] : *(const uint8_t*)(logp + t);
            in[i] = tid + i * BLOCK < tokens && (!a.batch.mask || m != 0);
        }
    }
    // more sequences than fit (only with fewer than four tokens): counted by token, offsets left in place
    const bool many = n_seqs > kSmallSeqs;
    const int slots = many ? 4 : n_seqs, len = n_seqs ? tokens / n_seqs : 0;
    if (!many)
        for (int s = tid; s <= n_seqs; s += BLOCK) offsets[s] = a.batch.cu ? ((const RLX_GLOBAL int32_t*)a.batch.cu)[s] : s * len;
    for (int s = tid; s < slots; s += BLOCK) in_seq[s] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSmallPerLane; i++) {
        at[i] = -1;
        if (tokens > 0 && in[i]) {
            const int t = tid + i * BLOCK;
            const int s = (int)(many ? offsets_up_to((const RLX_GLOBAL int32_t*)a.batch.cu, 0, n_seqs + 1, t)
                                     : offsets_up_to(offsets, 0, n_seqs + 1, t)) - 1;
            if (s >= 0 && s < n_seqs) {
                at[i] = s;
                if (!many) atomicAdd(&in_seq[s], 1);
                if (!a.per_token) adv[i] = a.advantages[s];
            }
        }
    }
    if (many) {                                     // the tokens are lanes 0 .. 2 of the first wavefront
        if (tid < 64) {
            const int s0 = __builtin_amdgcn_readlane(at[0], 0), s1 = __builtin_amdgcn_readlane(at[0], 1);
            const int s2 = __builtin_amdgcn_readlane(at[0], 2);
            if (tid < 4) in_seq[tid] = at[0] < 0 ? 0 : (s0 == at[0]) + (s1 == at[0]) + (s2 == at[0]);
        }
    }
    __syncthreads();
    int64_t total = 0;
    if (a.reduction == RLX_LOSS_TOKEN_MEAN) {
        // of the few tokens of many sequences: each once
        for (int s = tid; s < slots; s += BLOCK) total += many ? (in_seq[s] > 0 ? 1 : 0) : in_seq[s];
        total = sum_block<BLOCK>(total, shared_m);
    }
    LaneTerms v = {0.0, 0.0, 0.0, 0.0, 0, 0};
#pragma unroll
    for (int i = 0; i < kSmallPerLane; i++) {
        const int t = tid + i * BLOCK;
        if (t >= tokens) continue;
        f32x2 d = {0.0f, 0.0f};
        if (at[i] >= 0) {
            const Weight w = weights(a, a.reduction == RLX_LOSS_SEQUENCE_MEAN ? (int64_t)in_seq[many ? tid : at[i]] : total);
            d[0] = add_token(a, w, lp[i], old[i], ref[i], a.entropy ? entropy[i] : 0.0f, adv[i], v);
            d[1] = w.entropy;
        }
        dlogp[t] = d[0];
        if (dentropy) dentropy[t] = d[1];
    }
    const Terms sum = sum_terms<BLOCK>(terms_of(v), shared, shared_n);
    if (tid == 0) write_stats(sum, a.kl_coef, a.entropy_coef, stats);
}

constexpr int kStatsBlock = 512;

// Adds the partial terms, in a fixed order, and writes the statistics.
__global__ __launch_bounds__(kStatsBlock) void policy_stats_kernel(const Terms* __restrict__ partials, int64_t n,
                                                                   float kl_coef, float entropy_coef,
                                                                   rlx_policy_stats* __restrict__ stats) {
    __shared__ double shared[5 * kStatsBlock / 64];
    __shared__ int64_t shared_n[kStatsBlock / 64];
    Terms v = {0.0, 0.0, 0.0, 0.0, 0.0, 0};
    for (int64_t i = threadIdx.x; i < n; i += kStatsBlock) {
        const Terms p = partials[i];
        v.policy += p.policy;
        v.kl += p.kl;
        v.entropy += p.entropy;
        v.clipped += p.clipped;
        v.ratio += p.ratio;
        v.count += p.count;
    }
    v = sum_terms<kStatsBlock>(v, shared, shared_n);
    if (threadIdx.x == 0) write_stats(v, kl_coef, entropy_coef, stats);
}

struct RowTerms {
    RowGrad grad;
    RowValues values;
    Terms terms;
};

// Everything that a row's loss and gradient need besides its statistics.  m: count that the weight divides by.
template <bool DOT>
__device__ __forceinline__ RowTerms row_terms(const Policy& a, const Row& row, float zt, float old, float ref, float advantage,
                                              int64_t m, float k, float inv_t) {
    RowTerms o;
    const double w = weight_of(a, m);
    o.values = row_values(row, zt, k, inv_t);
    const TokenLoss l = token_loss(a, o.values.logp, old, ref, advantage);
    const double ws = w * (double)a.grad_scale * (double)inv_t;
    o.grad = row_gradient(row, o.values, (float)(ws * l.slope), DOT ? (float)-(ws * (double)a.entropy_coef) : 0.0f);
    o.terms = {w * l.policy, w * l.kl, w * (double)o.values.entropy, l.clipped ? 1.0 : 0.0, l.ratio, 1};
    return o;
}

// Policy loss from logits: one workgroup per row, the row held in registers between its statistics and its gradient
// (NG 16-byte groups per lane; a vocabulary beyond BLOCK * NG groups has its rest read a second time, from the
// last-level cache mostly).  A row of 151,936 halves is 304 KB: it fits the 512 KB of registers of a compute unit, not its
// 160 KB of LDS.  Every logit is read once and every gradient written once (FETCH_SIZE 1.54 GB, WRITE_SIZE 1.94 GB at 6,360
// rows of 151,936 FP16, a fifth of them masked), which takes 663 us = 5.2 TB/s; reading the rows twice took 990, and
// statistics and gradient as launches of their own 22 % more (4,096 unmasked rows: 479 and 586 us).
// Bound by the memory system on this pattern of one long row per compute unit: without any arithmetic the same accesses
// take 640 us, and workgroups that stay and load the next row while they write the present one gained nothing (272
// against 274 us at 90,000 FP16).  With the gradient over the logits the same memory is read and written: 10 to 15 % more time
// (4,096 rows of 151,936 FP16 492 and 539 us).  FP32 rows of 151,936 are held by half and their rest read twice: 2,048 of them
// 552 us, 4.5 TB/s.  DOT, the entropy's part of the gradient, is left out where there is none: 1,974 rows of 151,936 FP16 246
// against 252 us, BF16 248 against 255; within 2 % either way at 12,000 to 76,000.
template <typename T, int BLOCK, int NG, bool DOT, bool ONCE>
__global__ __launch_bounds__(BLOCK) void policy_loss_row_kernel(
    Logits x, Logits dx, const void* __restrict__ targets, int wide, float k, float inv_t, Policy a,
    const int32_t* __restrict__ seq_counts, const int32_t* __restrict__ info, float* __restrict__ logp,
    float* __restrict__ entropy, Terms* __restrict__ partials, uint32_t first) {
    __shared__ Stat shared[BLOCK / 64];
    __shared__ Stat shared_rare[BLOCK / 64];
    __shared__ RowGrad shared_grad;
    const uint32_t r = first + blockIdx.x;
    const int tid = threadIdx.x;
    const char* row = x.data + row_at(x, r) * T::SIZE;
    char* out = dx.data + row_at(dx, r) * T::SIZE;
    int64_t s = info[r];
    const int64_t t = target_at(targets, wide, r);
    if (s < 0 || t >= x.vocab) {
        const float value = s < 0 ? 0.0f : NAN;
        fill_row<T, BLOCK>(out, x.vocab, value);
        if (tid == 0) {
            logp[r] = value;
            if (entropy) entropy[r] = value;
            partials[r] = {value, value, value, value, value, s < 0 ? 0 : 1};
        }
        return;
    }
    s = s < a.batch.n_seqs ? s : a.batch.n_seqs - 1;
    const int groups = x.vocab / T::PER, j = groups * T::PER + tid, target = (int)t;
    u32x4 held[NG];
    load_groups<T, NG, BLOCK, ONCE>(held, row, tid, groups);
    drop_target<T, NG, BLOCK>(held, 0, target);
    const float loose = j < x.vocab && j != target ? T::one(row, j) : -INFINITY;
    const float zt = T::one(row, t), advantage = a.advantages[a.per_token ? (int64_t)r : s];
    const float old = a.old_logp ? a.old_logp[r] : 0.0f, ref = a.ref_logp ? a.ref_logp[r] : 0.0f;

    Stat st = held_statistics<T, NG, true>(held, loose, k);
    for (int g = NG * BLOCK + tid; g < groups; g += BLOCK) {
        u32x4 more[1] = {load16(row + (int64_t)g * 16)};
        if (g == target / T::PER) T::drop(more[0], target % T::PER);
        st = joined<true>(st, held_statistics<T, 1, true>(more, -INFINITY, k));
    }
    st = join_block<true, BLOCK>(st, shared);
    Row rv = row_of(st, zt, k);
    if (!ordinary(rv.sum())) rv = row_by_maximum<T, BLOCK>(row, x.vocab, target, k, shared_rare);
    // the row's few scalars by one wavefront: every wavefront doing the same would hold up the compute unit as long
    if (tid < 64) {
        const RowTerms o = row_terms<DOT>(a, rv, zt, old, ref, advantage, count_for(a, seq_counts, s), k, inv_t);
        if (tid == 0) {
            shared_grad = o.grad;
            logp[r] = o.values.logp;
            if (entropy) entropy[r] = o.values.entropy;
            partials[r] = o.terms;
        }
    }
    __syncthreads();
    const RowGrad q = shared_grad;
    if (q.shift != 0.0f) {
        rare_gradient<T, BLOCK, DOT>(q, row, out, 0, x.vocab, k, target);
        return;
    }
#pragma unroll
    for (int n = 0; n < NG; n++) {
        const int g = n * BLOCK + tid;
        forget(held[n]);
        const u32x4 v = grad_group<T, DOT>(q, held[n], k, target - g * T::PER);
        if (g < groups) store16_once(out + (int64_t)g * 16, v);
    }
    for (int g = NG * BLOCK + tid; g < groups; g += BLOCK)
        store16_once(out + (int64_t)g * 16, grad_group<T, DOT>(q, load16(row + (int64_t)g * 16), k, target - g * T::PER));
    if (j < x.vocab) {
        const float d = grad_of<DOT>(q, loose, k);
        T::put(out, j, j == target ? q.hot : d);
    }
}

// --- the loss of few rows: chunks of a row in workgroups of their own ------------------------------------------------------

constexpr int kFewGroups = 2;                // 16-byte groups per lane of such a chunk (8 KiB)

// How many rows of begin .. end - 1 count, by one wavefront.
__device__ __forceinline__ int64_t count_rows(const Batch& b, const void* targets, int wide, int64_t begin, int64_t end) {
    int64_t n = 0;
    for (int64_t t = begin; t < end; t += 64) {
        const int64_t u = t + (threadIdx.x & 63);
        n += __builtin_popcountll(__ballot(u < end && counts(b, targets, wide, u)));
    }
    return n;
}

// The launch behind chunk_statistics_kernel<256, kFewGroups>: every workgroup joins its row's chunks, works out the row's
// loss for itself and writes its chunk of the gradient; the first chunk's workgroup also writes the row's values.
// The last of those to finish adds up the rows, in their order.
// The logits of the targets come from the first launch: here another workgroup may have overwritten them.
template <typename T, bool DOT>
__global__ __launch_bounds__(kChunkBlock) void policy_loss_few_kernel(
    Logits x, Logits dx, const void* __restrict__ targets, int wide, float k, float inv_t, Policy a,
    const Stat* __restrict__ partials, const float* __restrict__ target_logits, float* __restrict__ logp,
    float* __restrict__ entropy, Terms* __restrict__ terms, uint32_t* __restrict__ ticket,
    rlx_policy_stats* __restrict__ stats) {
    constexpr int PER = T::PER;
    __shared__ Stat shared[kChunkBlock / 64];
    __shared__ double sums[5 * kChunkBlock / 64];
    __shared__ int64_t sums_n[kChunkBlock / 64];
    __shared__ int last_shared;
    const uint32_t r = blockIdx.y, c = blockIdx.x;
    const int tid = threadIdx.x, groups = x.vocab / PER, at = (int)c * kChunkBlock * kFewGroups + tid;
    const int j = groups * PER + tid;                        // the loose elements go with the first chunk
    const bool has_loose = c == 0 && j < x.vocab;
    const char* row = x.data + row_at(x, r) * T::SIZE;
    char* out = dx.data + row_at(dx, r) * T::SIZE;
    const RLX_GLOBAL int32_t* cu = (const RLX_GLOBAL int32_t*)a.batch.cu;
    const int64_t t = target_at(targets, wide, r), n_seqs = a.batch.n_seqs, len = cu ? 1 : a.batch.tokens / n_seqs;
    const int64_t s = (cu ? wave_offsets_up_to(cu, 0, n_seqs + 1, r) : r / len + 1) - 1;
    const bool in = s >= 0 && s < n_seqs && counts(a.batch, targets, wide, r), bad = in && t >= x.vocab;
    RowTerms o;
    o.values.logp = o.values.entropy = bad ? NAN : 0.0f;
    o.terms = {0.0, 0.0, 0.0, 0.0, 0.0, 0};
    if (bad) o.terms = {NAN, NAN, NAN, NAN, NAN, 1};
    if (!in || bad) {
        float f[PER];
#pragma unroll
        for (int i = 0; i < PER; i++) f[i] = bad ? NAN : 0.0f;
        const u32x4 v = T::pack(f);
#pragma unroll
        for (int n = 0; n < kFewGroups; n++)
            if (at + n * kChunkBlock < groups) store16_once(out + (int64_t)(at + n * kChunkBlock) * 16, v);
        if (has_loose) T::put(out, j, f[0]);
    } else {
        u32x4 held[kFewGroups];
        load_groups<T, kFewGroups, kChunkBlock, false>(held, row, at, groups);
        const float loose = has_loose ? T::one(row, j) : 0.0f;
        int64_t m = 1;
        if (a.reduction != RLX_LOSS_SUM) {
            const bool all = a.reduction == RLX_LOSS_TOKEN_MEAN;
            int64_t begin, end, unused;
            sequence_at(a.batch, all ? 0 : s, begin, end);
            if (all) sequence_at(a.batch, n_seqs - 1, unused, end);
            m = count_rows(a.batch, targets, wide, begin, end);
        }
        const float advantage = a.advantages[a.per_token ? (int64_t)r : s];
        const float old = a.old_logp ? a.old_logp[r] : 0.0f, ref = a.ref_logp ? a.ref_logp[r] : 0.0f;
        const float zt = target_logits[r];
        Row rv = row_of(join_chunks<true>(partials + (int64_t)r * gridDim.x, (int)gridDim.x), zt, k);
        const bool rare = !ordinary(rv.sum());
        if (rare && c != 0) return;                          // the first chunk's workgroup does a rare row by itself
        if (rare) rv = row_by_maximum<T, kChunkBlock>(row, x.vocab, (int)t, k, shared);
        o = row_terms<DOT>(a, rv, zt, old, ref, advantage, m, k, inv_t);
        const int target = (int)t;
        if (rare) {
            __syncthreads();                                 // every lane has read what is overwritten now
            rare_gradient<T, kChunkBlock, DOT>(o.grad, row, out, 0, x.vocab, k, target);
        } else {
#pragma unroll
            for (int n = 0; n < kFewGroups; n++) {
                const int g = at + n * kChunkBlock;
                const u32x4 v = grad_group<T, DOT>(o.grad, held[n], k, target - g * PER);
                if (g < groups) store16_once(out + (int64_t)g * 16, v);
            }
            if (has_loose) {
                const float d = grad_of<DOT>(o.grad, loose, k);
                T::put(out, j, j == target ? o.grad.hot : d);
            }
        }
    }
    if (c != 0) return;
    if (tid == 0) {
        logp[r] = o.values.logp;
        if (entropy) entropy[r] = o.values.entropy;
    }
    if (!last_with(o.terms, terms, r, gridDim.y, ticket, &last_shared)) return;
    const Terms v = sum_published<kChunkBlock>(terms, gridDim.y, sums, sums_n);
    if (tid == 0) write_stats(v, a.kl_coef, a.entropy_coef, stats);
}

// --- preference loss -------------------------------------------------------------------------------------------------

struct Preference {
    const float* ref_logp;
    Batch batch;
    int64_t n_pairs;
    float beta, smoothing, margin, grad_scale;
    int average;
};

struct PairTerms {
    double loss, correct, diff, chosen, rejected;
};

struct PairValues {
    PairTerms terms;
    float grad[2];               // of each counted token of the chosen and of the rejected sequence
};

// A pair's loss and gradient from its sums of log ratios and counts (chosen, rejected).
__device__ __forceinline__ PairValues pair_values(const Preference& a, const double (&sum)[2], const int64_t (&n)[2]) {
    double per[2], reward[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        per[i] = (double)a.beta * (a.average ? 1.0 / (double)(n[i] > 0 ? n[i] : 1) : 1.0);
        reward[i] = sum[i] * per[i];
    }
    const double diff = reward[0] - reward[1], x = diff - (double)a.margin, ls = (double)a.smoothing;
    // with e = exp(-|x|): log sigmoid(x) = min(x, 0) - log(1 + e), sigmoid(|x|) = 1 / (1 + e), sigmoid(-|x|) = e / (1 + e)
    const double e = exp(-fabs(x)), l = log1p(e), inv = 1.0 / (1.0 + e);
    const double log_s = fmin(x, 0.0) - l, log_n = fmin(-x, 0.0) - l;
    const double s = x >= 0.0 ? inv : e * inv, s_neg = x >= 0.0 ? e * inv : inv;
    const double slope = (ls * s - (1.0 - ls) * s_neg) / (double)a.n_pairs * (double)a.grad_scale;
    // 0 * (-inf) of a label that is not smoothed is 0
    const double loss = -(1.0 - ls) * (ls < 1.0 ? log_s : 0.0) - ls * (ls > 0.0 ? log_n : 0.0);
    return {{loss, diff > 0.0 ? 1.0 : 0.0, diff, reward[0], reward[1]}, {(float)(slope * per[0]), (float)(-slope * per[1])}};
}

// Sum of the log ratios and number of the counted tokens of one sequence, by LANES lanes.
struct RatioSum {
    double sum;
    int64_t n;
};

template <int LANES>
__device__ __forceinline__ RatioSum sum_ratios(const Preference& a, const float* logp, int64_t begin, int64_t end, int lane) {
    RatioSum o = {0.0, 0};
    int64_t t = begin + lane * 4;
    for (; t + 4 <= end; t += LANES * 4) {
        const f32x4_any x = load4(logp + t), y = a.ref_logp ? load4(a.ref_logp + t) : f32x4_any{0.0f, 0.0f, 0.0f, 0.0f};
        const uint32_t in = a.batch.mask ? nonzero_bytes(load_mask4(a.batch.mask + t)) : 0x80808080u;
#pragma unroll
        for (int i = 0; i < 4; i++) o.sum += in >> (8 * i) & 0x80u ? (double)x[i] - (double)y[i] : 0.0;
        o.n += __builtin_popcount(in);
    }
    for (int64_t u = t; u < end && u < t + 4; u++) {
        if (a.batch.mask && a.batch.mask[u] == 0) continue;
        o.sum += (double)logp[u] - (a.ref_logp ? (double)a.ref_logp[u] : 0.0);
        o.n++;
    }
    return o;
}

template <int LANES>
__device__ __forceinline__ void put_gradients(const Preference& a, float* dlogp, int64_t begin, int64_t end, float g, int lane) {
    int64_t t = begin + lane * 4;
    for (; t + 4 <= end; t += LANES * 4) {
        const uint32_t in = a.batch.mask ? nonzero_bytes(load_mask4(a.batch.mask + t)) : 0x80808080u;
        f32x4_any d;
#pragma unroll
        for (int i = 0; i < 4; i++) d[i] = in >> (8 * i) & 0x80u ? g : 0.0f;
        store4(dlogp + t, d);
    }
    for (int64_t u = t; u < end && u < t + 4; u++) dlogp[u] = !a.batch.mask || a.batch.mask[u] ? g : 0.0f;
}

// Zeros for the tokens in front of the first and behind the last sequence; lane `at` of `step`.
__device__ __forceinline__ void clear_outside(const Preference& a, float* dlogp, int64_t at, int64_t step) {
    if (!a.batch.cu) return;
    int64_t lo, hi, unused;
    sequence_at(a.batch, 0, lo, unused);
    sequence_at(a.batch, 2 * a.n_pairs - 1, unused, hi);
    for (int64_t t = at; t < lo; t += step) dlogp[t] = 0.0f;
    for (int64_t t = hi + at; t < a.batch.tokens; t += step) dlogp[t] = 0.0f;
}

constexpr int kPairBlock = 512;

// One workgroup per pair: both sums, the pair's loss, and the gradient of its
// tokens (1,024 sequences, 3.1 M tokens, 40 MB: 12 us, latencies of two phases and 8 us of memory; 19 with a token per
// lane).  Each lane has its first kPairQuads quads of both sequences on the way at once (that covers 4,096 tokens a
// sequence) and keeps which of their tokens count for the gradient; the rest of longer sequences goes in a loop.
constexpr int kPairQuads = 2;

__global__ __launch_bounds__(kPairBlock) void preference_loss_kernel(Preference a, const float* __restrict__ logp,
                                                                     float* __restrict__ dlogp, float* __restrict__ rewards,
                                                                     PairTerms* __restrict__ partials) {
    __shared__ double shared[2 * kPairBlock / 64];
    __shared__ int64_t shared_n[2 * kPairBlock / 64];
    __shared__ float grads[2];
    const int64_t pair = blockIdx.x;
    const float* ref = a.ref_logp ? a.ref_logp : logp;
    int64_t begin[2], end[2], n[2];
    double sum[2];
    f32x4_any x[2][kPairQuads], y[2][kPairQuads];
    uint32_t in[2][kPairQuads];
#pragma unroll
    for (int side = 0; side < 2; side++) sequence_at(a.batch, pair + side * a.n_pairs, begin[side], end[side]);
    const bool quads = a.batch.tokens >= 4;               // below that everything goes in the loop
    const int64_t head = quads ? kPairQuads * kPairBlock * 4 : 0;
    if (quads) {
#pragma unroll
        for (int side = 0; side < 2; side++) {
#pragma unroll
            for (int q = 0; q < kPairQuads; q++) {
                const int64_t own = begin[side] + ((int64_t)q * kPairBlock + threadIdx.x) * 4;
                const int64_t t = own + 4 <= a.batch.tokens ? own : a.batch.tokens - 4;
                x[side][q] = load4(logp + t);
                y[side][q] = load4(ref + t);
                in[side][q] = load_mask4(a.batch.mask ? a.batch.mask + t : (const uint8_t*)(logp + t));
            }
        }
    }
#pragma unroll
    for (int side = 0; side < 2; side++) {
        sum[side] = 0.0;
        n[side] = 0;
#pragma unroll
        for (int q = 0; q < kPairQuads; q++) {
            if (!quads) continue;
            const int64_t own = begin[side] + ((int64_t)q * kPairBlock + threadIdx.x) * 4;
            const int64_t t = own + 4 <= a.batch.tokens ? own : a.batch.tokens - 4;
            in[side][q] = (a.batch.mask ? nonzero_bytes(in[side][q]) : 0x80808080u) & tokens_within(t, own, end[side]);
#pragma unroll
            for (int i = 0; i < 4; i++)
                sum[side] += in[side][q] >> (8 * i) & 0x80u
                                 ? (double)x[side][q][i] - (a.ref_logp ? (double)y[side][q][i] : 0.0) : 0.0;
            n[side] += __builtin_popcount(in[side][q]);
        }
        const RatioSum o = sum_ratios<kPairBlock>(a, logp, begin[side] + head, end[side], threadIdx.x);
        sum[side] += o.sum;
        n[side] += o.n;
    }
    sum_block<kPairBlock, 2>(sum, shared);
    sum_block<kPairBlock, 2>(n, shared_n);
    // by one wavefront: its few hundred FP64 instructions in all eight would hold up the compute unit
    if (threadIdx.x < 64) {
        const PairValues v = pair_values(a, sum, n);
        if (threadIdx.x == 0) {
            grads[0] = v.grad[0];
            grads[1] = v.grad[1];
            if (rewards) {
                rewards[pair] = (float)v.terms.chosen;
                rewards[a.n_pairs + pair] = (float)v.terms.rejected;
            }
            partials[pair] = v.terms;
        }
    }
    __syncthreads();
#pragma unroll
    for (int side = 0; side < 2; side++) {
        const float g = grads[side];
#pragma unroll
        for (int q = 0; q < kPairQuads; q++) {
            if (!quads) continue;
            const int64_t own = begin[side] + ((int64_t)q * kPairBlock + threadIdx.x) * 4;
            const int64_t t = own + 4 <= a.batch.tokens ? own : a.batch.tokens - 4;
            f32x4_any d;
#pragma unroll
            for (int i = 0; i < 4; i++) d[i] = in[side][q] >> (8 * i) & 0x80u ? g : 0.0f;
            if (own + 4 <= end[side]) {
                store4(dlogp + own, d);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (t + i >= own && t + i < end[side]) dlogp[t + i] = d[i];
            }
        }
        put_gradients<kPairBlock>(a, dlogp, begin[side] + head, end[side], g, threadIdx.x);
    }
    clear_outside(a, dlogp, pair * kPairBlock + threadIdx.x, (int64_t)gridDim.x * kPairBlock);
}

__device__ __forceinline__ void write_pair_stats(const double (&v)[5], int64_t n, rlx_preference_stats* stats) {
    const double m = n > 0 ? 1.0 / (double)n : 0.0;
    *stats = {(float)(v[0] * m), (float)(v[1] * m), (float)(v[2] * m), (float)(v[3] * m), (float)(v[4] * m)};
}

// The whole of a small batch in one launch of one workgroup, a wavefront per pair.
constexpr int64_t kSmallPairs = 32, kSmallPairTokens = 16384;

__global__ __launch_bounds__(kPairBlock) void preference_loss_small_kernel(Preference a, const float* __restrict__ logp,
                                                                     float* __restrict__ dlogp, float* __restrict__ rewards,
                                                                     rlx_preference_stats* __restrict__ stats) {
    __shared__ double shared[5 * kPairBlock / 64];
    const int lane = threadIdx.x & 63;
    double terms[5] = {0.0, 0.0, 0.0, 0.0, 0.0};
    for (int64_t pair = threadIdx.x >> 6; pair < a.n_pairs; pair += kPairBlock / 64) {
        int64_t begin[2], end[2], n[2];
        double sum[2];
#pragma unroll
        for (int side = 0; side < 2; side++) {
            sequence_at(a.batch, pair + side * a.n_pairs, begin[side], end[side]);
            const RatioSum o = sum_ratios<64>(a, logp, begin[side], end[side], lane);
            sum[side] = wave_sum8(o.sum);
            n[side] = wave_sum8(o.n);
        }
        const PairValues v = pair_values(a, sum, n);
#pragma unroll
        for (int side = 0; side < 2; side++) put_gradients<64>(a, dlogp, begin[side], end[side], v.grad[side], lane);
        if (lane == 0) {
            if (rewards) {
                rewards[pair] = (float)v.terms.chosen;
                rewards[a.n_pairs + pair] = (float)v.terms.rejected;
            }
            terms[0] += v.terms.loss;
            terms[1] += v.terms.correct;
            terms[2] += v.terms.diff;
            terms[3] += v.terms.chosen;
            terms[4] += v.terms.rejected;
        }
    }
    if (a.n_pairs) clear_outside(a, dlogp, threadIdx.x, kPairBlock);
    sum_block<kPairBlock, 5>(terms, shared);
    if (threadIdx.x == 0) write_pair_stats(terms, a.n_pairs, stats);
}

__global__ __launch_bounds__(kStatsBlock) void preference_stats_kernel(const PairTerms* __restrict__ partials, int64_t n,
                                                                       rlx_preference_stats* __restrict__ stats) {
    __shared__ double shared[5 * kStatsBlock / 64];
    double v[5] = {0.0, 0.0, 0.0, 0.0, 0.0};
    for (int64_t i = threadIdx.x; i < n; i += kStatsBlock) {
        const PairTerms p = partials[i];
        v[0] += p.loss;
        v[1] += p.correct;
        v[2] += p.diff;
        v[3] += p.chosen;
        v[4] += p.rejected;
    }
    sum_block<kStatsBlock, 5>(v, shared);
    if (threadIdx.x == 0) write_pair_stats(v, n, stats);
}

// --- host side -------------------------------------------------------------------------------------------------------

constexpr int64_t kMaxRows = 0x7fffffff;
constexpr int64_t kMaxVocab = 1 << 30;
constexpr int64_t kMaxPairs = 1 << 22;               // a workgroup of 512 lanes each: below the 2^32 lanes of one launch
constexpr uint32_t kRowsPerLaunch = 1u << 21;        // times up to 1,024 lanes: below the 2^32 lanes of one launch

size_t elem_size(int dtype) { return dtype == RLX_DTYPE_F32 ? 4 : 2; }

// Elements from the first to one past the last of a matrix of rows, -1 if its strides are not usable.
int64_t logits_span(const rlx_logits& x) {
    const int64_t inner = x.group_rows > 0 && x.group_rows < x.rows ? x.group_rows : x.rows;
    const int64_t outer = inner ? (x.rows + inner - 1) / inner : 0;
    if (x.rows == 0) return 0;
    if (inner > 1 && x.row_stride < x.vocab) return -1;
    if (outer > 1 && x.group_stride < x.vocab) return -1;
    // strides that could overflow or that overlap: the larger step has to clear everything the smaller one spans
    const int64_t lim = (int64_t)1 << 60;
    if ((inner > 1 && x.row_stride > lim / inner) || (outer > 1 && x.group_stride > lim / outer)) return -1;
    const int64_t in_span = inner > 1 ? (inner - 1) * x.row_stride : 0;
    const int64_t out_span = outer > 1 ? (outer - 1) * x.group_stride : 0;
    if (inner > 1 && outer > 1) {
        const bool rows_inside = x.group_stride >= in_span + x.vocab, groups_inside = x.row_stride >= out_span + x.vocab;
        if (!rows_inside && !groups_inside) return -1;
    }
    return in_span + out_span + x.vocab;
}

int check_logits(const rlx_logits* x) {
    if (!x || x->rows < 0 || x->vocab < 1 || x->group_rows < 0 || x->reserved != 0) return RLX_ERR_INVALID_ARG;
    if (x->dtype != RLX_DTYPE_F16 && x->dtype != RLX_DTYPE_F32 && x->dtype != RLX_DTYPE_BF16) return RLX_ERR_INVALID_ARG;
    if (x->rows > kMaxRows || x->vocab > kMaxVocab) return RLX_ERR_TOO_LARGE;
    if (x->rows == 0) return RLX_OK;
    if (logits_span(*x) < 0 || !x->data) return RLX_ERR_INVALID_ARG;
    if (!rlx_is_aligned(x->data, elem_size(x->dtype))) return RLX_ERR_MISALIGNED;
    return RLX_OK;
}

// dx is x itself or does not touch it.
int check_gradient(const rlx_logits* x, const rlx_logits* dx) {
    const int st = check_logits(dx);
    if (st != RLX_OK) return st;
    if (dx->rows != x->rows || dx->vocab != x->vocab || dx->dtype != x->dtype) return RLX_ERR_INVALID_ARG;
    if (x->rows == 0) return RLX_OK;
    const bool one_group = (x->group_rows == 0 || x->group_rows >= x->rows) && (dx->group_rows == 0 || dx->group_rows >= dx->rows);
    if (x->data == dx->data) {
        const bool same = (x->rows == 1) || (x->row_stride == dx->row_stride &&
                          (one_group || (x->group_rows == dx->group_rows && x->group_stride == dx->group_stride)));
        return same ? RLX_OK : RLX_ERR_INVALID_ARG;
    }
    const char *a = (const char*)x->data, *b = (const char*)dx->data;
    const size_t es = elem_size(x->dtype);
    const bool apart = a + logits_span(*x) * es <= b || b + logits_span(*dx) * es <= a;
    return apart ? RLX_OK : RLX_ERR_INVALID_ARG;
}

Logits view(const rlx_logits& x) {
    Logits v;
    v.data = (char*)x.data;
    v.row_stride = x.row_stride;
    v.group_stride = x.group_stride;
    v.rows = (uint32_t)x.rows;
    v.group_rows = x.group_rows > 0 && x.group_rows < x.rows ? (uint32_t)x.group_rows : (uint32_t)x.rows;
    v.vocab = (int32_t)x.vocab;
    return v;
}

int row_groups(const rlx_logits& x) { return (int)(x.vocab / (x.dtype == RLX_DTYPE_F32 ? F32::PER : F16::PER)); }

// How the statistics of rows are cut: lanes and groups per lane of a workgroup, workgroups per row (a row's few elements
// behind its last whole group go with the first).
struct Cut {
    int block, per_lane, chunks;
};

// Rows up to 4,096 groups (32,768 halves) go whole to a workgroup, which writes their results in the same launch; longer
// ones in 32 KiB chunks that a second launch joins, or in 8 KiB ones where those would not fill the chip.  Recorded and
// replayed, whole / in chunks: 32,000 FP16, 1 row 4.2 / 4.8 us, 256 rows 6.6 / 8.8, 8,192 rows 79 / 89; 16,384 FP32 256 rows
// 6.1 / 8.3; 50,257 FP16 1 row 5.7 / 4.8, 8,192 rows 153 / 147.  (512 x 6 beside 512 x 8: 16,384 rows of 17,000 97 / 106.)  In between, for 97 to 256 rows, a launch less weighs more
// than what the few lanes of a workgroup cost: 129 rows of 50,257 FP16 7.8 / 9.1 us, of 90,000 9.7 / 10.0; 64 rows 7.5 / 7.3
// and 9.2 / 7.7; beyond 12,288 groups chunks do better for any number of rows (129 rows of 151,936 13.9 / 12.3).
// 8 KiB / 32 KiB chunks: 151,936 FP16 1 row 4.7 / 5.6 us, 16 rows 5.8 / 6.2, 51 rows 7.4 / 8.0, 64 rows 8.8 / 8.4, 300 rows
// 21.2 / 18.7; FP32 16 rows 6.3 / 7.0, 40 rows 9.4 / 8.2; 50,257 FP16 64 rows 6.1 / 6.5, 90 rows 6.7 / 7.6.
Cut cut_of(const rlx_logits& x) {
    const int groups = row_groups(x);
    if (groups <= 64 * 8) return {64, 8, 1};
    if (groups <= 128 * 8) return {128, 8, 1};
    if (groups <= 256 * 8) return {256, 8, 1};
    if (groups <= 512 * 6) return {512, 6, 1};
    if (groups <= 512 * 8) return {512, 8, 1};
    if (x.rows > 96 && x.rows <= 256) {
        if (groups <= 512 * 14) return {512, 14, 1};
        if (groups <= 1024 * 12) return {1024, 12, 1};
    }
    Cut c = {256, 8, (groups + 256 * 8 - 1) / (256 * 8)};
    if (x.rows * c.chunks < 512) {
        c.per_lane = 2;
        c.chunks = (groups + 256 * 2 - 1) / (256 * 2);
    }
    return c;
}

// Whether the loss from logits is better off with its rows in chunks, read twice, than with a workgroup per row: long rows,
// too few of them to fill the chip.  Time on the GPU, chunks / workgroup per row: 14 rows of 151,936 FP16 11.0 / 24.3 us,
// 85 rows 24.4 / 25.5, 145 rows 35.7 / 27.5; 85 rows of 151,936 FP32 36.8 / 38.4, 145 rows 55.5 / 48.0; 57 rows of 50,257
// BF16 12.4 / 16.6, 164 rows 20.1 / 18.4; 57 rows of 32,000 10.9 / 12.9, 145 rows 14.4 / 13.3; rows of 16,000 gain nothing.
constexpr int64_t kFewRows = 96;
bool few_rows(const rlx_logits& x) { return x.rows > 0 && x.rows <= kFewRows && row_groups(x) > 256 * 8; }
int64_t few_chunks(const rlx_logits& x) { return (row_groups(x) + kChunkBlock * kFewGroups - 1) / (kChunkBlock * kFewGroups); }

// Whether every row starts on a 16-byte boundary.
bool rows_aligned(const rlx_logits& x) {
    const int64_t es = (int64_t)elem_size(x.dtype);
    const bool grouped = x.group_rows > 0 && x.group_rows < x.rows;
    return rlx_is_aligned(x.data, 16) && (x.rows == 1 || x.row_stride * es % 16 == 0) &&
           (!grouped || x.group_stride * es % 16 == 0);
}

int check_targets(const void* targets, int index_type) {
    if (index_type != RLX_INDEX_I32 && index_type != RLX_INDEX_I64) return RLX_ERR_INVALID_ARG;
    if (!targets) return RLX_ERR_INVALID_ARG;
    return rlx_is_aligned(targets, index_type == RLX_INDEX_I64 ? 8 : 4) ? RLX_OK : RLX_ERR_MISALIGNED;
}

int check_temperature(float t) {
    // its reciprocal has to be a finite number too
    return std::isfinite(t) && t > 0.0f && std::isfinite(kLog2e / t) ? RLX_OK : RLX_ERR_BAD_HYPER;
}

int check_workspace(const void* ws, int64_t have, int64_t need) {
    if (have < need || (need > 0 && !ws)) return RLX_ERR_INVALID_ARG;
    return rlx_is_aligned(ws, 16) ? RLX_OK : RLX_ERR_MISALIGNED;
}

bool floats_aligned(std::initializer_list<const void*> all) {
    for (const void* p : all)
        if (!rlx_is_aligned(p, 4)) return false;
    return true;
}

int check_batch(const Batch& b) {
    if (b.tokens < 0 || b.n_seqs < 0) return RLX_ERR_INVALID_ARG;
    if (b.tokens > kMaxRows || b.n_seqs > kMaxRows) return RLX_ERR_TOO_LARGE;
    if (b.tokens > 0 && b.n_seqs == 0) return RLX_ERR_INVALID_ARG;
    if (!b.cu && b.n_seqs > 0 && b.tokens % b.n_seqs != 0) return RLX_ERR_INVALID_ARG;
    return rlx_is_aligned(b.cu, 4) ? RLX_OK : RLX_ERR_MISALIGNED;
}

int64_t round16(int64_t n) { return (n + 15) & ~(int64_t)15; }
int64_t counts_bytes(int64_t n_seqs) { return round16(4 * (n_seqs > kMostInline ? n_seqs : kMostInline)); }
int64_t token_blocks(int64_t tokens) { return (tokens + kTokensPerBlock - 1) / kTokensPerBlock; }

bool small_pairs(int64_t tokens, int64_t n_pairs) { return tokens <= kSmallPairTokens && n_pairs <= kSmallPairs; }
bool small_batch(int64_t tokens, int64_t n_seqs) { return tokens < 4 || (tokens <= kSmallTokens && n_seqs <= kSmallSeqs); }

int make_policy(const rlx_policy_args* p, int64_t tokens, Policy& a) {
    if (!p) return RLX_ERR_INVALID_ARG;
    a.old_logp = p->old_logp;
    a.ref_logp = p->ref_logp;
    a.advantages = p->advantages;
    a.entropy = p->entropy;
    a.batch = {p->mask, p->cu_seqlens, tokens, p->n_seqs};
    const int st = check_batch(a.batch);
    if (st != RLX_OK) return st;
    if (p->reduction < RLX_LOSS_SEQUENCE_MEAN || p->reduction > RLX_LOSS_SUM) return RLX_ERR_INVALID_ARG;
    const float all[] = {p->clip_low, p->clip_high, p->kl_coef, p->entropy_coef, p->norm, p->grad_scale};
    for (float v : all)
        if (!std::isfinite(v)) return RLX_ERR_BAD_HYPER;
    if (p->clip_low < 0.0f || p->clip_low > 1.0f || p->clip_high < 0.0f) return RLX_ERR_BAD_HYPER;
    if (tokens > 0 && !p->advantages) return RLX_ERR_INVALID_ARG;
    if (!floats_aligned({p->old_logp, p->ref_logp, p->advantages, p->entropy})) return RLX_ERR_MISALIGNED;
    a.log_high = std::log1p((double)p->clip_high);
    a.log_low = std::log1p(-(double)p->clip_low);           // -inf for clip_low = 1: nothing is below it
    a.high = 1.0 + (double)p->clip_high;
    a.low = 1.0 - (double)p->clip_low;
    a.norm = (double)p->norm;
    a.kl_coef = p->kl_coef;
    a.entropy_coef = p->entropy_coef;
    a.grad_scale = p->grad_scale;
    a.reduction = p->reduction;
    a.per_token = p->advantage_per_token ? 1 : 0;
    return RLX_OK;
}

// Counts of the sequences (and per token its sequence, if info); for the mean over all tokens of many sequences their sum.
hipError_t launch_counts(const Policy& a, const void* targets, int wide, int32_t* out, int32_t* info, hipStream_t s) {
    const Batch& b = a.batch;
    const int64_t grid = b.n_seqs < (1 << 20) ? b.n_seqs : (1 << 20);
    sequence_counts_kernel<<<dim3((unsigned)grid), dim3(kTokenBlock), 0, s>>>(b, targets, wide, out, info);
    if (a.reduction == RLX_LOSS_TOKEN_MEAN && b.n_seqs > kMostInline)
        total_count_kernel<<<dim3(1), dim3(1024), 0, s>>>(out, b.n_seqs);
    return hipGetLastError();
}

constexpr uint32_t kMostGridY = 65535;

// Calls f(first row, rows) for every launch of a kernel with a grid of (chunks, rows).
template <typename Fn>
int for_row_launches(uint32_t rows, uint32_t most, Fn f) {
    for (uint32_t first = 0; first < rows; first += most) {
        f(first, rows - first < most ? rows - first : most);
        RLX_HIP(hipGetLastError());
    }
    return RLX_OK;
}

// Calls f(T{}) for the logit type.
template <typename Fn>
void for_type(int dtype, Fn f) {
    if (dtype == RLX_DTYPE_F16) f(F16{});
    else if (dtype == RLX_DTYPE_BF16) f(BF16{});
    else f(F32{});
}

template <bool V>
struct Bool {
    static constexpr bool value = V;
};

// Calls f with the two truth values as compile-time ones.
template <typename Fn>
void for_flags(bool a, bool b, Fn f) {
    if (a) b ? f(Bool<true>{}, Bool<true>{}) : f(Bool<true>{}, Bool<false>{});
    else b ? f(Bool<false>{}, Bool<true>{}) : f(Bool<false>{}, Bool<false>{});
}

template <int N>
struct Int {
    static constexpr int value = N;
};

template <typename Fn>
void for_cut(const Cut& c, Fn f) {
    if (c.block == 64) f(Int<64>{}, Int<8>{});
    else if (c.block == 128) f(Int<128>{}, Int<8>{});
    else if (c.block == 512 && c.per_lane == 6) f(Int<512>{}, Int<6>{});
    else if (c.block == 512 && c.per_lane == 8) f(Int<512>{}, Int<8>{});
    else if (c.block == 512) f(Int<512>{}, Int<14>{});
    else if (c.block == 1024) f(Int<1024>{}, Int<12>{});
    else if (c.per_lane == 8) f(Int<256>{}, Int<8>{});
    else f(Int<256>{}, Int<2>{});
}

// Calls f(lanes, 16-byte groups per lane) for the shape that holds a row of `groups` groups in registers.  Groups that a shape
// has and the row has not are loaded all the same (the last one again), so the steps are small: with 512 x 8, 512 x 14, 1,024 x
// 12 and 1,024 x 19 alone 17,000 FP16 took 255 us for 300 M logits, not 233, 36,000 239 and 225, 64,000 265 and 221, 100,000
// 277 and 252, 128,256 243 and 233; of FP32, 150 M logits, 18,000 232 and 224, 32,000 249 and 221, 50,000 257 and 244, 57,000 257
// and 252.  One wavefront of 4 groups beside 8: 200 M logits of 1,000 FP16 351 and 468 us, 2,000 218 and 247; FP32 600 511 and
// 624, 1,000 430 and 411.  Two workgroups of 512 lanes do better on a compute unit than one of 1,024 (64,000 as
// 1,024 x 8: 230), as long as they have the registers (98,304 as 512 x 24: 246, as 1,024 x 12 236).
template <typename Fn>
void for_row_shape(int groups, Fn f) {
    if (groups <= 64 * 4) f(Int<64>{}, Int<4>{});
    else if (groups <= 64 * 8) f(Int<64>{}, Int<8>{});
    else if (groups <= 128 * 8) f(Int<128>{}, Int<8>{});
    else if (groups <= 256 * 8) f(Int<256>{}, Int<8>{});
    else if (groups <= 512 * 6) f(Int<512>{}, Int<6>{});
    else if (groups <= 512 * 8) f(Int<512>{}, Int<8>{});
    else if (groups <= 512 * 10) f(Int<512>{}, Int<10>{});
    else if (groups <= 512 * 14) f(Int<512>{}, Int<14>{});
    else if (groups <= 512 * 16) f(Int<512>{}, Int<16>{});
    else if (groups <= 1024 * 10) f(Int<1024>{}, Int<10>{});
    else if (groups <= 1024 * 12) f(Int<1024>{}, Int<12>{});
    else if (groups <= 1024 * 14) f(Int<1024>{}, Int<14>{});
    else if (groups <= 1024 * 16) f(Int<1024>{}, Int<16>{});
    else f(Int<1024>{}, Int<19>{});
}

}  // namespace

extern "C" {

int64_t rlx_token_logprob_workspace(const rlx_logits* x) {
    if (check_logits(x) != RLX_OK) return -1;
    const Cut c = cut_of(*x);
    return c.chunks > 1 ? x->rows * c.chunks * (int64_t)sizeof(Stat) : 0;
}

int rlx_token_logprob(const rlx_logits* x, const void* targets, int index_type, float temperature, float* logp,
                      float* lse, float* entropy, void* workspace, int64_t workspace_bytes, void* stream) {
    int st = check_logits(x);
    if (st != RLX_OK) return st;
    if ((st = check_temperature(temperature)) != RLX_OK) return st;
    if (x->rows == 0) return RLX_OK;
    if ((st = check_targets(targets, index_type)) != RLX_OK) return st;
    if (!logp || !lse) return RLX_ERR_INVALID_ARG;
    if (!floats_aligned({logp, lse, entropy})) return RLX_ERR_MISALIGNED;
    if ((st = check_workspace(workspace, workspace_bytes, rlx_token_logprob_workspace(x))) != RLX_OK) return st;
    hipStream_t s = (hipStream_t)stream;
    const Logits v = view(*x);
    const float inv_t = 1.0f / temperature, k = kLog2e / temperature;
    const int wide = index_type == RLX_INDEX_I64;
    const Cut cut = cut_of(*x);
    const RowOutputs o = {logp, lse, entropy}, none = {nullptr, nullptr, nullptr};
    Stat* partials = (Stat*)workspace;
    for_type(x->dtype, [&](auto type) {
        typedef decltype(type) T;
        for_flags(entropy != nullptr, rows_aligned(*x), [&](auto dot, auto once) {
            for_cut(cut, [&](auto block, auto ng) {
                constexpr int BLOCK = decltype(block)::value, NG = decltype(ng)::value;
                st = for_row_launches(v.rows, kMostGridY, [&](uint32_t first, uint32_t here) {
                    chunk_statistics_kernel<T, BLOCK, NG, decltype(dot)::value, decltype(once)::value>
                        <<<dim3(cut.chunks, here), dim3(BLOCK), 0, s>>>(v, targets, wide, nullptr, k, inv_t,
                                                                        cut.chunks == 1 ? o : none, partials, nullptr, nullptr,
                                                                        first);
                });
            });
        });
        if (st != RLX_OK || cut.chunks == 1) return;
        st = for_row_launches(v.rows, kRowsPerLaunch, [&](uint32_t first, uint32_t here) {
            const dim3 grid((here + kJoinRows - 1) / kJoinRows), block(kJoinBlock);
            if (entropy)
                token_logprob_join_kernel<T, true><<<grid, block, 0, s>>>(v, targets, wide, k, inv_t, partials, cut.chunks, o, first,
                                                                          here);
            else
                token_logprob_join_kernel<T, false><<<grid, block, 0, s>>>(v, targets, wide, k, inv_t, partials, cut.chunks, o, first,
                                                                           here);
        });
    });
    return st;
}

int rlx_token_logprob_backward_logp(const rlx_logits* x, const void* targets, int index_type, float temperature,
                                    const float* lse, const float* entropy, const float* logp, const float* dlogp,
                                    const float* dentropy, const rlx_logits* dx, void* stream) {
    int st = check_logits(x);
    if (st != RLX_OK) return st;
    if ((st = check_gradient(x, dx)) != RLX_OK) return st;
    if ((st = check_temperature(temperature)) != RLX_OK) return st;
    if (x->rows == 0) return RLX_OK;
    if ((st = check_targets(targets, index_type)) != RLX_OK) return st;
    if (!lse || !dlogp || !entropy != !dentropy) return RLX_ERR_INVALID_ARG;
    if (!floats_aligned({lse, entropy, logp, dlogp, dentropy})) return RLX_ERR_MISALIGNED;
    const Logits v = view(*x), dv = view(*dx);
    const float inv_t = 1.0f / temperature, k = kLog2e / temperature;
    const int wide = index_type == RLX_INDEX_I64, groups = row_groups(*x);
    const unsigned chunks = groups ? (groups + 255) / 256 : 1;          // 4 KiB of a row per workgroup
    for_type(x->dtype, [&](auto type) {
        typedef decltype(type) T;
        for_flags(dentropy != nullptr, rows_aligned(*x), [&](auto dot, auto once) {
            st = for_row_launches(v.rows, kMostGridY, [&](uint32_t first, uint32_t here) {
                constexpr bool ONCE = decltype(once)::value;
                token_logprob_backward_kernel<T, ONCE ? 256 : 128, ONCE ? 1 : 2, decltype(dot)::value, ONCE>
                    <<<dim3(chunks, here), dim3(ONCE ? 256 : 128), 0, (hipStream_t)stream>>>(
                        v, dv, targets, wide, k, inv_t, lse, entropy, logp, dlogp, dentropy, first);
            });
        });
    });
    return st;
}

int rlx_token_logprob_backward(const rlx_logits* x, const void* targets, int index_type, float temperature,
                               const float* lse, const float* entropy, const float* dlogp, const float* dentropy,
                               const rlx_logits* dx, void* stream) {
    return rlx_token_logprob_backward_logp(x, targets, index_type, temperature, lse, entropy, nullptr, dlogp, dentropy, dx, stream);
}

int64_t rlx_policy_loss_workspace(int64_t tokens, int64_t n_seqs) {
    if (tokens < 0 || n_seqs < 0 || tokens > kMaxRows || n_seqs > kMaxRows) return -1;
    if (small_batch(tokens, n_seqs)) return 0;
    return counts_bytes(n_seqs) + token_blocks(tokens) * (int64_t)sizeof(Terms);
}

int rlx_policy_loss(const float* logp, int64_t tokens, const rlx_policy_args* args, float* dlogp, float* dentropy,
                    rlx_policy_stats* stats, void* workspace, int64_t workspace_bytes, void* stream) {
    Policy a;
    int st = make_policy(args, tokens, a);
    if (st != RLX_OK) return st;
    if (!stats || (tokens > 0 && (!logp || !dlogp))) return RLX_ERR_INVALID_ARG;
    if (tokens > 0 && a.entropy_coef != 0.0f && (!a.entropy || !dentropy)) return RLX_ERR_INVALID_ARG;
    if (!floats_aligned({logp, dlogp, dentropy}) || !rlx_is_aligned(stats, 8)) return RLX_ERR_MISALIGNED;
    if ((st = check_workspace(workspace, workspace_bytes, rlx_policy_loss_workspace(tokens, a.batch.n_seqs))) != RLX_OK)
        return st;
    hipStream_t s = (hipStream_t)stream;
    if (small_batch(tokens, a.batch.n_seqs)) {
        if (tokens <= 128 * kSmallPerLane)
            policy_loss_small_kernel<128><<<dim3(1), dim3(128), 0, s>>>(a, logp, dlogp, dentropy, stats);
        else if (tokens <= 256 * kSmallPerLane)
            policy_loss_small_kernel<256><<<dim3(1), dim3(256), 0, s>>>(a, logp, dlogp, dentropy, stats);
        else
            policy_loss_small_kernel<512><<<dim3(1), dim3(512), 0, s>>>(a, logp, dlogp, dentropy, stats);
        RLX_HIP(hipGetLastError());
        return RLX_OK;
    }
    const int64_t blocks = token_blocks(tokens);
    int32_t* seq_counts = (int32_t*)workspace;
    Terms* partials = (Terms*)((char*)workspace + counts_bytes(a.batch.n_seqs));
    if (a.reduction != RLX_LOSS_SUM) RLX_HIP(launch_counts(a, nullptr, 0, seq_counts, nullptr, s));
    policy_loss_kernel<<<dim3((unsigned)blocks), dim3(kTokenBlock), 0, s>>>(a, logp, seq_counts, dlogp, dentropy, partials);
    RLX_HIP(hipGetLastError());
    policy_stats_kernel<<<dim3(1), dim3(kStatsBlock), 0, s>>>(partials, blocks, a.kl_coef, a.entropy_coef, stats);
    RLX_HIP(hipGetLastError());
    return RLX_OK;
}

int64_t rlx_policy_loss_logits_workspace(const rlx_logits* x, int64_t n_seqs) {
    if (check_logits(x) != RLX_OK || n_seqs < 0 || n_seqs > kMaxRows) return -1;
    if (few_rows(*x))
        return round16(x->rows * few_chunks(*x) * (int64_t)sizeof(Stat)) + round16(4 * x->rows) +
               x->rows * (int64_t)sizeof(Terms) + 16;
    return counts_bytes(n_seqs) + round16(4 * x->rows) + x->rows * (int64_t)sizeof(Terms);
}

int rlx_policy_loss_logits(const rlx_logits* x, const void* targets, int index_type, float temperature,
                           const rlx_policy_args* args, float* logp, float* entropy, const rlx_logits* dx,
                           rlx_policy_stats* stats, void* workspace, int64_t workspace_bytes, void* stream) {
    int st = check_logits(x);
    if (st != RLX_OK) return st;
    if ((st = check_gradient(x, dx)) != RLX_OK) return st;
    if ((st = check_temperature(temperature)) != RLX_OK) return st;
    Policy a;
    if ((st = make_policy(args, x->rows, a)) != RLX_OK) return st;
    if (!stats || a.entropy || (x->rows > 0 && !logp)) return RLX_ERR_INVALID_ARG;
    if (x->rows > 0 && (st = check_targets(targets, index_type)) != RLX_OK) return st;
    if (!floats_aligned({logp, entropy}) || !rlx_is_aligned(stats, 8)) return RLX_ERR_MISALIGNED;
    if ((st = check_workspace(workspace, workspace_bytes, rlx_policy_loss_logits_workspace(x, a.batch.n_seqs))) != RLX_OK)
        return st;
    hipStream_t s = (hipStream_t)stream;
    const Logits v = view(*x), dv = view(*dx);
    const float inv_t = 1.0f / temperature, k = kLog2e / temperature;
    const int wide = index_type == RLX_INDEX_I64;
    if (few_rows(*x)) {
        const unsigned chunks = (unsigned)few_chunks(*x);
        Stat* partials = (Stat*)workspace;
        float* target_logits = (float*)((char*)workspace + round16(x->rows * chunks * (int64_t)sizeof(Stat)));
        Terms* terms = (Terms*)((char*)target_logits + round16(4 * x->rows));
        uint32_t* ticket = (uint32_t*)(terms + x->rows);
        const RowOutputs none = {nullptr, nullptr, nullptr};
        for_type(x->dtype, [&](auto type) {
            typedef decltype(type) T;
            const dim3 grid(chunks, v.rows);
            chunk_statistics_kernel<T, kChunkBlock, kFewGroups, true, false><<<grid, dim3(kChunkBlock), 0, s>>>(
                v, targets, wide, a.batch.mask, k, inv_t, none, partials, target_logits, ticket, 0);
            if (a.entropy_coef != 0.0f)
                policy_loss_few_kernel<T, true><<<grid, dim3(kChunkBlock), 0, s>>>(
                    v, dv, targets, wide, k, inv_t, a, partials, target_logits, logp, entropy, terms, ticket, stats);
            else
                policy_loss_few_kernel<T, false><<<grid, dim3(kChunkBlock), 0, s>>>(
                    v, dv, targets, wide, k, inv_t, a, partials, target_logits, logp, entropy, terms, ticket, stats);
        });
        RLX_HIP(hipGetLastError());
        return RLX_OK;
    }
    int32_t* seq_counts = (int32_t*)workspace;
    int32_t* info = (int32_t*)((char*)workspace + counts_bytes(a.batch.n_seqs));
    Terms* partials = (Terms*)((char*)info + round16(4 * x->rows));
    if (v.rows) RLX_HIP(launch_counts(a, targets, wide, seq_counts, info, s));
    for_type(x->dtype, [&](auto type) {
        typedef decltype(type) T;
        for_row_shape(v.vocab / T::PER, [&](auto block, auto ng) {
            constexpr int BLOCK = decltype(block)::value, NG = decltype(ng)::value;
            for_flags(a.entropy_coef != 0.0f, rows_aligned(*x), [&](auto dot, auto once) {
                st = for_row_launches(v.rows, kRowsPerLaunch, [&](uint32_t first, uint32_t here) {
                    policy_loss_row_kernel<T, BLOCK, NG, decltype(dot)::value, decltype(once)::value>
                        <<<dim3(here), dim3(BLOCK), 0, s>>>(v, dv, targets, wide, k, inv_t, a, seq_counts, info, logp, entropy,
                                                            partials, first);
                });
            });
        });
    });
    if (st != RLX_OK) return st;
    policy_stats_kernel<<<dim3(1), dim3(kStatsBlock), 0, s>>>(partials, v.rows, a.kl_coef, a.entropy_coef, stats);
    RLX_HIP(hipGetLastError());
    return RLX_OK;
}

int64_t rlx_preference_loss_workspace(int64_t tokens, int64_t n_pairs) {
    if (tokens < 0 || n_pairs < 0 || tokens > kMaxRows || n_pairs > kMaxPairs) return -1;
    return small_pairs(tokens, n_pairs) ? 0 : n_pairs * (int64_t)sizeof(PairTerms);
}

int rlx_preference_loss(const float* logp, int64_t tokens, const rlx_preference_args* args, float* dlogp,
                        float* rewards, rlx_preference_stats* stats, void* workspace, int64_t workspace_bytes,
                        void* stream) {
    if (!args || !stats || args->reserved != 0 || args->n_pairs < 0) return RLX_ERR_INVALID_ARG;
    if (args->n_pairs > kMaxPairs) return RLX_ERR_TOO_LARGE;
    Preference a;
    a.ref_logp = args->ref_logp;
    a.batch = {args->mask, args->cu_seqlens, tokens, 2 * args->n_pairs};
    int st = check_batch(a.batch);
    if (st != RLX_OK) return st;
    const float all[] = {args->beta, args->label_smoothing, args->margin, args->grad_scale};
    for (float v : all)
        if (!std::isfinite(v)) return RLX_ERR_BAD_HYPER;
    if (args->label_smoothing < 0.0f || args->label_smoothing > 1.0f) return RLX_ERR_BAD_HYPER;
    if (tokens > 0 && (!logp || !dlogp)) return RLX_ERR_INVALID_ARG;
    if (!floats_aligned({logp, args->ref_logp, dlogp, rewards, stats})) return RLX_ERR_MISALIGNED;
    if ((st = check_workspace(workspace, workspace_bytes, rlx_preference_loss_workspace(tokens, args->n_pairs))) != RLX_OK)
        return st;
    a.n_pairs = args->n_pairs;
    a.beta = args->beta;
    a.smoothing = args->label_smoothing;
    a.margin = args->margin;
    a.grad_scale = args->grad_scale;
    a.average = args->average ? 1 : 0;
    hipStream_t s = (hipStream_t)stream;
    if (small_pairs(tokens, a.n_pairs)) {
        preference_loss_small_kernel<<<dim3(1), dim3(kPairBlock), 0, s>>>(a, logp, dlogp, rewards, stats);
        RLX_HIP(hipGetLastError());
        return RLX_OK;
    }
    PairTerms* partials = (PairTerms*)workspace;
    if (a.n_pairs) {
        preference_loss_kernel<<<dim3((unsigned)a.n_pairs), dim3(kPairBlock), 0, s>>>(a, logp, dlogp, rewards, partials);
        RLX_HIP(hipGetLastError());
    }
    preference_stats_kernel<<<dim3(1), dim3(kStatsBlock), 0, s>>>(partials, a.n_pairs, stats);
    RLX_HIP(hipGetLastError());
    return RLX_OK;
}

}  // extern "C"
