// The AdamW step over many tensors in one launch, its moments held in 32 bits or in 8, and the global gradient norm that clips it.
//
//   g' = c g,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,  p = (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Pure streaming: with f32 parameters 28 bytes per element (7 accesses of 4) with 32-bit moments and 16 with 8-bit ones, against 18 and 72 vector instructions (at 6.5 TB/s the
// card issues about 97 in the time of 16 bytes).  The file is compiled without contraction of a * b + c, so that the moments round like the written formulas and the codes of the 8-bit
// moments can be predicted bit for bit.
//
// 8-BIT MOMENTS.  Two bytes per element and two per block of 128 consecutive elements of a tensor.  A code c > 0 with the block's base exponent b stands for
// (1 + (c & 7) / 8) * 2^((c >> 3) + b - 127) — as f32 bits simply (c << 20) + (b << 23) —, c = 0 for zero.  First moment: sign and 7 bits (16 exponents),
// second: 8 bits (32 exponents); the base is the exponent of the block's largest finite value less 14 or 30 (at least 1), so the largest always has a code, with
// room for one carry.  Why a floating code with a shared POWER OF TWO: Adam divides by sqrt(v), so what counts is the relative error of small values too, and
// the block's scale costs no multiplication and no division.  Why STOCHASTIC rounding: with b2 = 0.999 one step moves v by a thousandth of itself, and codes are
// 6 to 12 % apart — rounded to nearest, v would never move unless the gradient jumped eightfold; rounded up with the probability of the distance to the code
// below, its expectation is exact.  Second moments above zero never round to zero (the smallest code instead): the denominator must not vanish; first moments below the
// smallest code keep their expectation (that code with probability |m| / code, else zero).  The floors fit each other: in units of the
// bases, the element with the largest first moment has m >= 2^14 and v <= 2^31, so its step is 2^-1.5 at least, and an element at both floors has 1.125 / sqrt(1.125); below a floor an
// element so moves by at most three times the block's largest step (eps and the end of the exponents aside).  Values that are not finite stay so in their own element: magnitude 127 is NaN,
// second-moment code 255 is infinity.
// The random bits are a function of (seed, step, place of the tensor in the list, element): one hashed word per 8 elements, times an odd constant per element — its
// high and low half are the 16 bits of v and m (each uniform, because an odd multiplier permutes the words).
// Published constants: the mixer's shifts and factors (C. Wellons, "Prospecting for Hash Functions", 2018), the golden ratio (0x9E3779B1), an odd factor of A. Appleby's hashes
// (0x85EBCA6B), the initial words of SHA-256.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <vector>

#include <hip/hip_runtime.h>

#include "../../include/gsicp_hip.h"
#include "raster_common.hpp"

namespace gsicp {
extern thread_local std::string g_last_error;

namespace {

constexpr int TABLE = 64;             // tensors per launch: the table travels in the kernel arguments (< 4 KB), nothing is copied or kept
constexpr int DEV_TABLE = 56;         // with what the device form adds
constexpr int NORM_TABLE = 240;
constexpr int NORM_ROWS_TABLE = 120;  // with rows that are left out
constexpr uint32_t LAST = 0x7FFFFFFF; // a tile number that no launch reaches
constexpr long long MAX_NUMEL = 1ll << 33;   // 2^25 workgroups of the step for one tensor; a launch has less than 2^32 lanes
constexpr unsigned long long STEP_TILES = (1u << 26) - 1, DECODE_TILES = (1u << 24) - 1;
constexpr int TILE_ELEMS = 256;       // elements of a workgroup of the step and of the gathering: ONE wave, four consecutive elements a lane, no loop
constexpr int NORM_GRID = 2048;       // partial sums of one norm launch
constexpr int NORM_SMALL_TILES = 64;  // 4 KB tiles that one workgroup of 16 waves takes by itself: 64 of them 7.4 us against 10.9 in two launches, 128 12.3 against 10.8 (they are
                                      // even somewhere between: 64 is on the safe side, not the crossing itself)
constexpr int QBLOCK = 128;           // elements per base exponent: 32 lanes x 4

enum Dtype { F32 = 0, BF16 = 1, F16 = 2 };

// vector types without an alignment demand beyond the element's: views of a flat buffer begin anywhere
typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2), aligned(2)));

struct StepEntry {
    void* p;
    const void* g;
    void* s0;              // exp_avg, or the packed 8-bit moments
    void* s1;              // exp_avg_sq, or the base exponents
    float* master;
    uint64_t word;         // 35 bits numel, 3 bits Dtype | 4 with a master, 1 bit: frozen rows are left alone, 24 bits from 40: place in the list (random bits)
    union {
        float scale[2];    // lr / (1 - b1^t) and 1 - lr wd    (host form)
        double wd;         // the device form takes lr from memory
    };
    __host__ __device__ long long numel() const { return (long long)(word & ((1ull << 35) - 1)); }
    __host__ __device__ uint32_t kind() const { return (uint32_t)(word >> 35) & 7u; }
    __host__ __device__ bool frozen() const { return (word >> 38 & 1u) != 0; }
    __host__ __device__ uint32_t place() const { return (uint32_t)(word >> 40); }
};
template <bool DEV> struct StepTable;
template <> struct StepTable<false> {
    uint32_t first[64];    // first tile of each tensor (an empty one has its successor's); LAST behind them
    StepEntry e[TABLE];
};
template <> struct StepTable<true> {
    uint32_t first[64];
    StepEntry e[DEV_TABLE];
    uint32_t row_width[DEV_TABLE], row_magic[DEV_TABLE];   // elements per map row (live rows, masks), 0: whole tensor; the division's multiplier
};
struct StepHyper {
    float b1, omb1, b2, omb2, eps;
    float inv_bc2_sqrt;    // 1 / sqrt(1 - b2^t)            (host step count)
    double ln_b1, ln_b2;   // for the same on the device     (device step count)
    const float* clip;     // device: the factor of every gradient (NULL: 1)
    const double* lr_dev;
    const int* step_dev;
    int step;              // host: the step count; device: what to add to *step_dev
    uint32_t seed;
    const uint32_t* guard_count;
    uint32_t guard_limit;
    const int *live_rows, *row_freeze, *grad_rows;
    int src;               // index of the table's first tensor in lr_dev
};
static_assert(sizeof(StepTable<false>) + sizeof(StepHyper) <= 4096 && sizeof(StepTable<true>) + sizeof(StepHyper) <= 4096, "kernel arguments of a launch");

__device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x7FEB352Du;
    x = (x ^ (x >> 15)) * 0x846CA68Bu;
    return x ^ (x >> 16);
}
__device__ __forceinline__ uint32_t lane_word(int e) {
    constexpr uint32_t w[8] = {0x6A09E667u, 0xBB67AE85u, 0x3C6EF373u, 0xA54FF53Bu, 0x510E527Fu, 0x9B05688Du, 0x1F83D9ABu, 0x5BE0CD19u};
    return w[e];
}

// The tensor a tile belongs to: the number of first tiles at or before it, less one.  `first` lies in the kernel arguments and `tile` is the same for the wave, so all of this is
// scalar: sixteen entries a load, and the scalar cache answers while the vector path is full of the other waves' streams.
// Tile numbers are below 2^31: the sign of first - tile - 1 is the comparison (a boolean sum would go through vector registers).
template <int ENTRIES>
__device__ __forceinline__ uint32_t find_tensor(const uint32_t (&first)[ENTRIES], uint32_t tile) {
    uint32_t k = 0;
#pragma unroll
    for (int i = 1; i < 16; ++i) k += (first[i] + ~tile) >> 31;
    if (tile >= first[16]) {
        k = 16;
#pragma unroll
        for (int i = 32; i < ENTRIES; i += 16) k += (first[i] + ~tile) >> 31 << 4;
        const uint32_t* f = first + k;
#pragma unroll
        for (int i = 1; i < 16; ++i) k += (f[i] + ~tile) >> 31;
    }
    return k;
}
// Demands a wave-uniform value here, in scalar registers: without it the compiler moves each load of a table entry to its first use, and the wave waits for them one by one.
template <class T> __device__ __forceinline__ void at_hand(T x) { asm volatile("" : : "s"(x)); }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float from16(uint32_t h, int dtype) {
    return dtype == BF16 ? __uint_as_float(h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
// two values, the first in the low half; round to nearest, ties to even
__device__ __forceinline__ uint32_t to16x2(float x, float y, int dtype) {
    const f32x2 f = {x, y};
    if (dtype == F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, f16x2));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
}

// one overload per vector type: a deduced type would lose the element's alignment
#define GSICP_ACCESS(V)                                                                                                          \
    template <bool NT> __device__ __forceinline__ V get(const V* p) { return NT ? __builtin_nontemporal_load(p) : *p; }           \
    template <bool NT> __device__ __forceinline__ void put(V* p, V v) { if (NT) __builtin_nontemporal_store(v, p); else *p = v; }
GSICP_ACCESS(f32x4)
GSICP_ACCESS(u32x4)
GSICP_ACCESS(u32x2)
#undef GSICP_ACCESS

// four consecutive elements; FULL: all of them exist, else only the first nv
template <int DT, bool FULL, bool NT>
__device__ __forceinline__ void load4(const void* base, long long at, int nv, float out[4]) {
    if (DT == F32) {
        const float* p = (const float*)base + at;
        if (FULL) {
            const f32x4 a = get<NT>((const f32x4*)p);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = a[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = j < nv ? p[j] : 0.f;
        }
    } else {
        const uint16_t* p = (const uint16_t*)base + at;
        if (FULL) {
            const u32x2 a = get<NT>((const u32x2*)p);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = from16((a[j >> 1] >> (16 * (j & 1))) & 0xFFFFu, DT);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = j < nv ? from16(p[j], DT) : 0.f;
        }
    }
}
template <int DT, bool FULL, bool NT>
__device__ __forceinline__ void store4(void* base, long long at, int nv, const float x[4]) {
    if (DT == F32) {
        float* p = (float*)base + at;
        if (FULL) {
            f32x4 a;
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] = x[j];
            put<NT>((f32x4*)p, a);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) if (j < nv) p[j] = x[j];
        }
    } else {
        uint16_t* p = (uint16_t*)base + at;
        if (FULL) {
            u32x2 a;
#pragma unroll
            for (int j = 0; j < 2; ++j) a[j] = to16x2(x[2 * j], x[2 * j + 1], DT);
            put<NT>((u32x2*)p, a);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) if (j < nv) p[j] = (uint16_t)to16x2(x[j], 0.f, DT);
        }
    }
}
template <bool FULL, bool NT>
__device__ __forceinline__ void load_codes(const void* base, long long at, int nv, uint32_t c[2]) {
    const uint16_t* p = (const uint16_t*)base + at;
    if (FULL) {
        const u32x2 a = get<NT>((const u32x2*)p);
        c[0] = a[0]; c[1] = a[1];
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) c[j] = (2 * j < nv ? (uint32_t)p[2 * j] : 0u) | (2 * j + 1 < nv ? (uint32_t)p[2 * j + 1] << 16 : 0u);
    }
}
template <bool FULL, bool NT>
__device__ __forceinline__ void store_codes(void* base, long long at, int nv, const uint32_t c[2]) {
    uint16_t* p = (uint16_t*)base + at;
    if (FULL) {
        u32x2 a;
        a[0] = c[0]; a[1] = c[1];
        put<NT>((u32x2*)p, a);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) if (j < nv) p[j] = (uint16_t)(c[j >> 1] >> (16 * (j & 1)));
    }
}

__device__ __forceinline__ float decode_m(uint32_t c16, uint32_t bm23) {
    const uint32_t mag = c16 & 0x7Fu;
    uint32_t bits = (c16 << 24 & 0x80000000u) | ((mag << 20) + bm23);
    bits = mag == 127u ? 0x7FC00000u : bits;
    return __uint_as_float(mag == 0u ? 0u : bits);
}
__device__ __forceinline__ float decode_v(uint32_t c16, uint32_t bv23) {
    const uint32_t c = c16 >> 8 & 0xFFu;
    uint32_t bits = (c << 20) + bv23;
    bits = c == 255u ? 0x7F800000u : bits;
    return __uint_as_float(c == 0u ? 0u : bits);
}
// largest value of each half of the wave, in every lane of it: four rotations within rows of 16, one exchange of neighbouring rows
__device__ __forceinline__ uint32_t half_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xF, 0xF, true));   // row_ror:8
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xF, 0xF, true));   // row_ror:4
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xF, 0xF, true));   // row_ror:2
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xF, 0xF, true));   // row_ror:1
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return max((uint32_t)r[0], (uint32_t)r[1]);
}
__device__ __forceinline__ uint32_t base_exponent(uint32_t top, int below) {
    const int b = (int)(top >> 23) - below;
    return (uint32_t)(b < 1 ? 1 : b);
}

// what one step needs to know of a tensor, after the hyper-parameters are folded
struct Fold { float b1, omb1, b2, omb2, eps, ibc2, decay, step_size, clip; };

// Four elements.  The moments round operation by operation; the parameter takes the hardware's root and reciprocal (measured over all exponents: off by less than 1.6 * 2^-24 of the
// result each, where the correctly rounded sequences cost 25 instructions an element) and fused sums.  The hardware's root takes a subnormal for zero: a wave that holds a
// subnormal second moment goes the long way.
__device__ __forceinline__ void adamw4(float p[4], float m[4], float v[4], const float g[4], const Fold& f) {
    bool subnormal = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        m[j] = m[j] * f.b1 + g[j] * f.omb1;
        v[j] = v[j] * f.b2 + g[j] * f.omb2 * g[j];
        subnormal |= __builtin_amdgcn_classf(v[j], 0x80);
    }
    float root[4];
    if (__ballot(subnormal) == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) root[j] = __builtin_amdgcn_sqrtf(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) root[j] = sqrtf(v[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        p[j] = __builtin_fmaf(-f.step_size, m[j] * __builtin_amdgcn_rcpf(__builtin_fmaf(root[j], f.ibc2, f.eps)), p[j] * f.decay);
}

constexpr uint32_t TOP_CODE = 0x7F700000u;      // 1.875 * 2^127: the last finite code of any base
// New moments -> codes.  SPECIAL: some value of the wave is not finite, or so large that it could round up to what is not.
template <bool SPECIAL>
__device__ __forceinline__ void encode4(const float m[4], const float v[4], uint32_t bm, uint32_t bv, uint32_t word, uint32_t o[2]) {
    const float low = __uint_as_float((bm << 23) + (1u << 20)), low16 = low * 0x1p-16f, low17 = low16 * 0.5f;
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t r = word * ((threadIdx.x & 1) ? lane_word(j + 4) : lane_word(j));
        uint32_t mb = __float_as_uint(m[j]) & 0x7FFFFFFFu, vb = SPECIAL ? __float_as_uint(v[j]) & 0x7FFFFFFFu : __float_as_uint(v[j]);
        const bool m_out = SPECIAL && mb >= 0x7F800000u, v_out = SPECIAL && vb >= 0x7F800000u;
        if (SPECIAL) { mb = min(mb, TOP_CODE); vb = min(vb, TOP_CODE); }
        const float a = __uint_as_float(mb);
        uint32_t mc = ((mb + ((r << 4 & 0xFFFF0u) | 8u)) >> 20) - (bm << 3);
        // fma: low16 * (u + 1/2), rounded once
        mc = a < low ? (a > __builtin_fmaf(low16, (float)(r & 0xFFFFu), low17) ? 1u : 0u) : mc;
        mc = (__float_as_uint(m[j]) >> 24 & 0x80u) | mc;
        const int vs = (int)((vb + ((r >> 12 & 0xFFFF0u) | 8u)) >> 20) - (int)(bv << 3);
        uint32_t vc = vb == 0u ? 0u : (uint32_t)max(vs, 1);
        if (m_out) mc = 127u;
        if (v_out) vc = 255u;
        h[j] = vc << 8 | mc;
    }
    o[0] = h[1] << 16 | h[0];
    o[1] = h[3] << 16 | h[2];
}

// Rows of a map tensor and what is said of them.  Division by the width: the host's multiplier (floor(2^32 (2^s - w) / w) + 1 with s = ceil(log2 w)) makes
// (t + ((n - t) >> 1)) >> (s - 1), t = high word of multiplier * n, exact for every 32-bit n (w > 1).
struct Rows {
    uint32_t width, magic, shift;      // width 0: no rows
    const int *grad, *freeze;
    __device__ __forceinline__ uint32_t of(uint32_t n) const {
        const uint32_t t = __umulhi(magic, n);
        return width == 1u ? n : (t + ((n - t) >> 1)) >> shift;
    }
    // rows of the elements at ... at + nv - 1, those behind them as the first: at most two rows when a row has three elements or more
    __device__ __forceinline__ void of4(uint32_t at, int nv, uint32_t row[4]) const {
        const uint32_t w = width, first = of(at), col = at - first * w, last = of(at + (uint32_t)max(nv, 1) - 1u);
#pragma unroll
        for (int j = 0; j < 4; ++j) row[j] = w >= 3u ? (col + j < w ? first : last) : (w == 2u ? (at + j) >> 1 : at + j);
#pragma unroll
        for (int j = 1; j < 4; ++j) row[j] = j < nv ? row[j] : row[0];
    }
};
__device__ __forceinline__ uint32_t row_shift(uint32_t w) { return w > 1u ? 31u - __builtin_clz(w - 1u) : 0u; }
// one bit per element: word > 0 (kind 0) or word == 0 (kind 1)
__device__ __forceinline__ uint32_t row_flag(int word, int kind) { return kind == 0 ? (word > 0 ? 1u : 0u) : (word == 0 ? 1u : 0u); }
__device__ __forceinline__ uint32_t flags4(const int* words, const uint32_t row[4], int kind) {
    uint32_t f = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) f |= row_flag(words[row[j]], kind) << j;
    return f;
}
__device__ __forceinline__ uint32_t flags2(const int* words, const uint32_t row[4], int kind) {        // row[0], and row[3] or an earlier one equal to it
    const uint32_t a = row_flag(words[row[0]], kind), b = row_flag(words[max(max(row[1], row[2]), row[3])], kind);
    uint32_t f = a;
#pragma unroll
    for (int j = 1; j < 4; ++j) f |= (row[j] == row[0] ? a : b) << j;
    return f;
}

template <bool Q8, int DT, bool MASTER, bool FULL, bool MASKED, bool NT>
__device__ __forceinline__ void step_tile(const StepEntry& e, const Fold& f, const Rows& rows, uint32_t key, uint32_t tile, long long numel) {
    const long long at = (long long)tile * TILE_ELEMS + 4 * threadIdx.x;
    const int nv = FULL ? 4 : (int)max(0ll, min(4ll, numel - at));
    float p[4], g[4], m[4], v[4];
    uint32_t c[2], exps = 0;
    if (MASTER) load4<F32, FULL, NT>(e.master, at, nv, p); else load4<DT, FULL, NT>(e.p, at, nv, p);
    const long long block = (long long)tile * (TILE_ELEMS / QBLOCK) + (threadIdx.x >> 5);
    if (Q8) {
        load_codes<FULL, NT>(e.s0, at, nv, c);
        if (FULL || nv > 0) exps = ((const uint16_t*)e.s1)[block];
    } else {
        load4<F32, FULL, NT>(e.s0, at, nv, m);
        load4<F32, FULL, NT>(e.s1, at, nv, v);
    }
    uint32_t keep = 0;                          // elements of frozen rows
    if (!MASKED || rows.width == 0) {
        load4<DT, FULL, NT>(e.g, at, nv, g);
    } else {
        // Two words to read where the four elements are of two rows, not four.  With the division by multiplication and the gradient
        // not read where all four are culled, 23.0 -> 20.8 us for 4.2 M elements of 300 k rows.
        const uint32_t w = rows.width;
        uint32_t row[4];
        rows.of4((uint32_t)at, nv, row);
        uint32_t live = 0xFu;
        if (FULL || nv > 0) {
            if (rows.grad) live = w >= 3u ? flags2(rows.grad, row, 0) : flags4(rows.grad, row, 0);
            if (e.frozen()) keep = w >= 3u ? ~flags2(rows.freeze, row, 1) : ~flags4(rows.freeze, row, 1);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) g[j] = 0.f;
        if (live) load4<DT, FULL, NT>(e.g, at, nv, g);          // culled rows: zero, whatever the gradient's memory holds there
#pragma unroll
        for (int j = 0; j < 4; ++j) g[j] = live >> j & 1u ? g[j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] *= f.clip;
    if (Q8) {
        const uint32_t bm23 = (exps & 0xFFu) << 23, bv23 = (exps >> 8) << 23;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t c16 = c[j >> 1] >> (16 * (j & 1));
            m[j] = decode_m(c16, bm23);
            v[j] = decode_v(c16, bv23);
        }
    }
    float p0[4], m0[4], v0[4];
    if (MASKED && !Q8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) { p0[j] = p[j]; m0[j] = m[j]; v0[j] = v[j]; }
    }
    adamw4(p, m, v, g, f);
    if (MASKED && !Q8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) if (keep >> j & 1u) { p[j] = p0[j]; m[j] = m0[j]; v[j] = v0[j]; }
    }
    if (MASTER) store4<F32, FULL, NT>(e.master, at, nv, p);
    store4<DT, FULL, NT>(e.p, at, nv, p);
    if (!Q8) {
        store4<F32, FULL, NT>(e.s0, at, nv, m);
        store4<F32, FULL, NT>(e.s1, at, nv, v);
        return;
    }
    uint32_t tm = 0, tv = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (FULL || j < nv) {
            tm = max(tm, __float_as_uint(m[j]) & 0x7FFFFFFFu);
            tv = max(tv, __float_as_uint(v[j]));
        }
    const uint32_t word = mix32(((uint32_t)tile * (TILE_ELEMS / 8) + (threadIdx.x >> 1)) ^ key);
    uint32_t bm, bv, o[2];
    if (__ballot(max(tm, tv) > TOP_CODE) == 0) {
        bm = base_exponent(half_max(tm), 14);
        bv = base_exponent(half_max(tv), 30);
        encode4<false>(m, v, bm, bv, word, o);
    } else {                                    // the largest FINITE values say the base
        tm = tv = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t mb = __float_as_uint(m[j]) & 0x7FFFFFFFu, vb = __float_as_uint(v[j]) & 0x7FFFFFFFu;
            if ((FULL || j < nv) && mb < 0x7F800000u) tm = max(tm, mb);
            if ((FULL || j < nv) && vb < 0x7F800000u) tv = max(tv, vb);
        }
        bm = base_exponent(half_max(tm), 14);
        bv = base_exponent(half_max(tv), 30);
        encode4<true>(m, v, bm, bv, word, o);
    }
    store_codes<FULL, NT>(e.s0, at, nv, o);
    if ((threadIdx.x & 31) == 0 && (FULL || nv > 0)) ((uint16_t*)e.s1)[block] = (uint16_t)(bm | bv << 8);
}

// 1 - b^t on the device, in f32, within 8 units of 2^-24 of itself: y = t ln(b) rounded once, then -(e^y - 1) by its series where that would cancel (|y| <= 0.35: the first
// term left out is y^8 / 9! of the first), else by the hardware's 2^x.  In f32, not by pow in double, because every wave evaluates it.
__device__ __forceinline__ float one_minus_power(double ln_b, int t) {
    const float y = (float)fmax((double)t * ln_b, -100.0);
    constexpr float c[8] = {1.f, 1.f / 2, 1.f / 6, 1.f / 24, 1.f / 120, 1.f / 720, 1.f / 5040, 1.f / 40320};
    float s = c[7];
#pragma unroll
    for (int k = 6; k >= 0; --k) s = __builtin_fmaf(s, y, c[k]);
    return y > -0.35f ? -y * s : 1.f - __builtin_amdgcn_exp2f(y * 1.44269504088896341f);
}

// One workgroup, one wave, 256 elements, no loop: the launch hands the tiles out in order and the streams stay local in DRAM.  DEV: step count and learning rates come from
// device memory (a captured graph replays them).
// Measured: 236 M f32 parameters, 32-bit moments 1.08 ms = 6.1 TB/s (a copy written the same way 6.5; a grid-stride loop of 2 048 workgroups of 256 lanes 1.34 ms, one tile of
// 2 048 elements a workgroup 1.26, of 1 024 1.10 - 1.14); 140 M with 8-bit moments 0.345 ms = 6.5 TB/s (with the correctly rounded root and quotient and 108 instructions an
// element 0.382: bound by them); 560 k parameters 4.1 us, 608 in 64 tensors 3.5 us: a launch.  The device form on 4.2 M parameters of 300 k rows: 19.2 us,
// with a radii mask 20.3; 8-bit 13.8 and 15.5.
template <bool Q8, bool DEV, bool MASKED, bool NT>
__global__ __launch_bounds__(64) void adamw_step_kernel(StepTable<DEV> t, StepHyper h) {
    const uint32_t tile = blockIdx.x, k = find_tensor(t.first, tile), mine = tile - t.first[k];
    const StepEntry e = t.e[k];
    float clip = 1.f;
    if (h.clip) clip = *h.clip;
    int step = h.step;
    Fold f = {h.b1, h.omb1, h.b2, h.omb2, h.eps, h.inv_bc2_sqrt, e.scale[1], e.scale[0], clip};
    at_hand(e.p); at_hand(e.g); at_hand(e.s0); at_hand(e.s1); at_hand(e.master); at_hand(e.word); at_hand(mine); at_hand(f.decay); at_hand(f.step_size);
    at_hand(f.b1); at_hand(f.omb1); at_hand(f.b2); at_hand(f.omb2); at_hand(f.eps); at_hand(f.ibc2); at_hand(clip);
    long long numel = e.numel();
    Rows rows = {0, 0, 0, h.grad_rows, h.row_freeze};
    if constexpr (DEV) {
        if (h.guard_count && *h.guard_count > h.guard_limit) return;      // the iteration that made these gradients is void: nothing moves
        rows.width = t.row_width[k];
        if (MASKED) { rows.magic = t.row_magic[k]; rows.shift = row_shift(rows.width); }
        if (h.live_rows && rows.width > 0) numel = min(numel, (long long)*h.live_rows * rows.width);     // rows behind the live count are not parameters
        step += *h.step_dev;
        const double lr = h.lr_dev[h.src + k];
        const float bc = one_minus_power(threadIdx.x & 1 ? h.ln_b2 : h.ln_b1, step);      // both powers in one evaluation
        const float bc1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, bc), 0));
        const float bc2 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, bc), 1));
        f.ibc2 = __builtin_amdgcn_rsqf(bc2);
        f.decay = (float)(1.0 - lr * e.wd);
        f.step_size = (float)lr * __builtin_amdgcn_rcpf(bc1);
    }
    const long long left = numel - (long long)mine * TILE_ELEMS;
    if (left <= 0) return;
    const uint32_t key = Q8 ? mix32(h.seed + (uint32_t)step * 0x9E3779B1u + e.place() * 0x85EBCA6Bu) : 0u;
    const bool full = left >= TILE_ELEMS;
    const uint32_t kind = e.kind();
#define GSICP_STEP(DT, MASTER)                                                                                                                \
    (full ? step_tile<Q8, DT, MASTER, true, MASKED, NT>(e, f, rows, key, mine, numel)                          \
          : step_tile<Q8, DT, MASTER, false, MASKED, NT>(e, f, rows, key, mine, numel))
    if (MASKED || kind == F32) GSICP_STEP(F32, false);
    else if (kind == BF16) GSICP_STEP(BF16, false);
    else if (kind == F16) GSICP_STEP(F16, false);
    else if (kind == (BF16 | 4)) GSICP_STEP(BF16, true);
    else GSICP_STEP(F16, true);
#undef GSICP_STEP
}

__global__ void adamw_bump_kernel(int* step_dev, const uint32_t* guard_count, uint32_t guard_limit, uint32_t* skipped) {
    if (guard_count && *guard_count > guard_limit) {
        if (skipped) *skipped += 1u;
        return;
    }
    *step_dev += 1;
}

// ------------------------------------------------------------------------------------------------ values of the codes
struct DecodeEntry { const void* codes; const void* exps; void* m; void* v; long long numel; };
struct DecodeTable { uint32_t first[64]; DecodeEntry e[64]; };

// 256 lanes x 8: with 6 or 10 bytes an element, tiles of one wave are bound by the rate at which workgroups start (140 M elements to bf16: 203 us, so 136 = 6.2 TB/s)
constexpr int DECODE_ELEMS = 2048;

template <int DT, bool FULL, bool NT>
__device__ __forceinline__ void decode_tile(const DecodeEntry& e, uint32_t tile) {
    const long long at = (long long)tile * DECODE_ELEMS + 4 * threadIdx.x;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const long long i = at + 1024 * h;
        const int nv = FULL ? 4 : (int)max(0ll, min(4ll, e.numel - i));
        if (nv == 0) return;
        uint32_t c[2];
        load_codes<FULL, NT>(e.codes, i, nv, c);
        const uint32_t exps = ((const uint16_t*)e.exps)[i / QBLOCK];
        float m[4], v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t c16 = c[j >> 1] >> (16 * (j & 1));
            m[j] = decode_m(c16, (exps & 0xFFu) << 23);
            v[j] = decode_v(c16, (exps >> 8) << 23);
        }
        store4<DT, FULL, NT>(e.m, i, nv, m);
        store4<DT, FULL, NT>(e.v, i, nv, v);
    }
}
// bf16 holds every code's value exactly (four significant bits, f32's exponents)
template <int DT, bool NT>
__global__ __launch_bounds__(256) void adamw_decode_kernel(DecodeTable t) {
    const uint32_t k = find_tensor(t.first, blockIdx.x);
    const DecodeEntry& e = t.e[k];
    const uint32_t mine = blockIdx.x - t.first[k];
    if (e.numel - (long long)mine * DECODE_ELEMS >= DECODE_ELEMS) decode_tile<DT, true, NT>(e, mine);
    else decode_tile<DT, false, NT>(e, mine);
}

// ------------------------------------------------------------------------------------------------ rows of 8-bit moments
// Row r of the result is row index[r] of the source, re-blocked.  As bases are powers of two, a code moves to another base by adding eight times the difference of the bases: exact,
// but for codes that fall below the new block's smallest (first moments become zero, second the smallest code).  Rows that the source does not have come out zero.
// Measured: nine tenths of 300 k rows of 59 elements 38 us.  Two-byte loads through the index bound it; a map is pruned once in hundreds of steps.
struct GatherEntry { const uint16_t* codes; const uint16_t* exps; uint16_t* out_codes; uint16_t* out_exps; uint32_t width, magic; };
struct GatherTable { uint32_t first[64]; GatherEntry e[TABLE]; };
static_assert(sizeof(GatherTable) + 64 <= 4096, "kernel arguments of a launch");

__global__ __launch_bounds__(64) void adamw_gather_kernel(GatherTable t, const long long* __restrict__ index, uint32_t n_rows, long long src_rows) {
    const uint32_t k = find_tensor(t.first, blockIdx.x), mine = blockIdx.x - t.first[k];
    const GatherEntry e = t.e[k];
    const Rows rows = {e.width, e.magic, row_shift(e.width), nullptr, nullptr};
    const uint32_t numel = n_rows * e.width, at = mine * TILE_ELEMS + 4 * threadIdx.x;       // below 2^32 (checked on the host)
    uint32_t am[4], av[4], sign[4], tm = 0, tv = 0;      // code + 8 base; 0: zero, ~0: not finite
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t c = 0, x = 0;
        if (at + j < numel && at + j >= at) {
            const uint32_t row = rows.of(at + j), col = at + j - row * e.width;
            const long long from = index[row];
            if (from >= 0 && from < src_rows) {
                const long long i = from * e.width + col;
                c = e.codes[i];
                x = e.exps[i / QBLOCK];
            }
        }
        const uint32_t mag = c & 0x7Fu, vc = c >> 8;
        sign[j] = c & 0x80u;
        am[j] = mag == 0u ? 0u : mag == 127u ? ~0u : mag + 8u * (x & 0xFFu);
        av[j] = vc == 0u ? 0u : vc == 255u ? ~0u : vc + 8u * (x >> 8);
        tm = max(tm, am[j] == ~0u ? 0u : am[j]);
        tv = max(tv, av[j] == ~0u ? 0u : av[j]);
    }
    const int bm = max((int)(half_max(tm) >> 3) - 14, 1), bv = max((int)(half_max(tv) >> 3) - 30, 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int mc = am[j] == ~0u ? 127 : am[j] == 0u ? 0 : max((int)am[j] - 8 * bm, 0), vc = av[j] == ~0u ? 255 : av[j] == 0u ? 0 : max((int)av[j] - 8 * bv, 1);
        if (at + j < numel && at + j >= at) e.out_codes[at + j] = (uint16_t)(vc << 8 | sign[j] | mc);
    }
    if ((threadIdx.x & 31) == 0 && at < numel) e.out_exps[at / QBLOCK] = (uint16_t)(bm | bv << 8);
}

// ------------------------------------------------------------------------------------------------ global norm
// Squares and sums in 64 bits: 133 M f16 gradients summed in 32 would lose what the clip factor needs to be the same from run to run and split to split, and the squares of large
// or small f32 gradients would leave its range.  The sums are split over the workgroups by position alone and joined in a fixed order.
// Measured: 133 M f16 gradients 42 us = 6.4 TB/s and 4.7 us for the join of 2 048 sums, 45 as calls follow each other (with 1 024 workgroups 53); 4.2 M f32 ones 4.8 + 2.2 us.
struct NormEntry { const void* g; long long numel; int dtype; bool frozen; };
struct NormPacked {      // 58 bits address, 2 bits Dtype, the rest of numel (2 bits), 1 bit: rows may be frozen
    uint32_t at_low, at_high, numel_low;
    __host__ void set(const void* g, long long numel, int dtype, bool frozen) {
        const uint64_t at = (uint64_t)(uintptr_t)g | (uint64_t)dtype << 58 | (uint64_t)numel >> 32 << 60 | (uint64_t)frozen << 62;
        *this = {(uint32_t)at, (uint32_t)(at >> 32), (uint32_t)numel};
    }
    __device__ __forceinline__ NormEntry entry() const {
        const uint64_t at = (uint64_t)at_high << 32 | at_low;
        return {(const void*)(at & ((1ull << 58) - 1)), (long long)((at >> 60 & 3u) << 32 | numel_low), (int)(at >> 58 & 3u), (at >> 62 & 1u) != 0};
    }
};
template <bool ROWS> struct NormTable;
template <> struct NormTable<false> {      // 16 bytes a tensor: 240 of them in one launch (128 in entries of 28: 200 tensors of 7 and 12 elements 17.3 us, so 14.3; 400 of them 26.9 and 18.0)
    uint32_t first[NORM_TABLE];
    NormPacked e[NORM_TABLE];
};
template <> struct NormTable<true> {       // rows behind a live count and frozen rows are no parameters: their gradients do not count, whatever they hold
    uint32_t first[128];
    NormPacked e[NORM_ROWS_TABLE];
    uint32_t row_width[NORM_ROWS_TABLE], row_magic[NORM_ROWS_TABLE];   // as in StepTable<true>
    const int *live_rows, *row_freeze;
};
static_assert(sizeof(NormTable<false>) + 64 <= 4096 && sizeof(NormTable<true>) + 64 <= 4096, "kernel arguments of a launch");

__host__ __device__ constexpr int norm_tile_elems(int dtype, int bytes) { return bytes / (dtype == F32 ? 4 : 2); }

template <int DT>
__device__ __forceinline__ double square_sum16(const u32x4& r) {      // of one 16-byte load
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (DT == F32) { const double x = __uint_as_float(r[j]); s = __builtin_fma(x, x, s); }
        else {
            const double x = from16(r[j] & 0xFFFFu, DT), y = from16(r[j] >> 16, DT);
            s = __builtin_fma(x, x, s);
            s = __builtin_fma(y, y, s);
        }
    }
    return s;
}
// `lanes` lanes, four 16-byte loads of each in flight; lane l of load k takes unit k * lanes + l
template <int DT, bool NT>
__device__ __forceinline__ double norm_tile(const NormEntry& e, uint32_t tile, int lanes, int lane) {
    constexpr int V = DT == F32 ? 4 : 8;
    const long long at = (long long)tile * (4 * V * lanes), left = e.numel - at;
    const char* p = (const char*)e.g + at * (16 / V);
    double s = 0.0;
    if (left >= 4 * V * lanes) {
        u32x4 r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = get<NT>((const u32x4*)(p + 16 * (size_t)(k * lanes + lane)));
#pragma unroll
        for (int k = 0; k < 4; ++k) s += square_sum16<DT>(r[k]);
    } else {
        const int whole = (int)(left / V), rest = (int)(left - (long long)whole * V);
        for (int u = lane; u < whole; u += lanes) s += square_sum16<DT>(*(const u32x4*)(p + 16 * (size_t)u));
        if (lane < rest) {
            const size_t i = (size_t)whole * V + lane;
            const double x = DT == F32 ? ((const float*)p)[i] : from16(((const uint16_t*)p)[i], DT);
            s = __builtin_fma(x, x, s);
        }
    }
    return s;
}
// The same of an f32 tensor of less than 2^32 elements without its frozen rows; FULL: the whole tile exists.  4.2 M elements of 300 k rows: 8.9 us with half of the rows frozen, 5.8
// with a live count only, 5.0 as they are.
template <bool FULL>
__device__ __forceinline__ double norm_frozen_tile(const NormEntry& e, const Rows& rows, uint32_t tile, int lanes, int lane) {
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const long long at = (long long)tile * (16 * lanes) + 4 * (k * lanes + lane);
        const int nv = FULL ? 4 : (int)max(0ll, min(4ll, e.numel - at));
        if (!FULL && nv == 0) break;
        float x[4];
        uint32_t row[4];
        load4<F32, FULL, false>(e.g, at, nv, x);
        rows.of4((uint32_t)at, nv, row);
        const uint32_t moves = rows.width >= 3u ? flags2(rows.freeze, row, 1) : flags4(rows.freeze, row, 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double y = moves >> j & 1u ? x[j] : 0.f;
            s = __builtin_fma(y, y, s);
        }
    }
    return s;
}
template <bool NT, bool ROWS>
__device__ __forceinline__ double norm_any_tile(const NormTable<ROWS>& t, uint32_t tile, int lanes, int lane) {
    const uint32_t k = find_tensor(t.first, tile);
    NormEntry e = t.e[k].entry();
    const uint32_t mine = tile - t.first[k];
    if constexpr (ROWS) {
        const uint32_t w = t.row_width[k];
        if (t.live_rows && w > 0) e.numel = min(e.numel, (long long)*t.live_rows * w);
        if ((long long)mine * norm_tile_elems(e.dtype, 64 * lanes) >= e.numel) return 0.0;
        if (e.frozen) {
            const Rows rows = {w, t.row_magic[k], row_shift(w), nullptr, t.row_freeze};
            return ((long long)mine + 1) * (16 * lanes) <= e.numel ? norm_frozen_tile<true>(e, rows, mine, lanes, lane) : norm_frozen_tile<false>(e, rows, mine, lanes, lane);
        }
    }
    return e.dtype == F32 ? norm_tile<F32, NT>(e, mine, lanes, lane) : e.dtype == BF16 ? norm_tile<BF16, NT>(e, mine, lanes, lane) : norm_tile<F16, NT>(e, mine, lanes, lane);
}
template <int WAVES>
__device__ __forceinline__ double block_sum(double s) {      // complete in thread 0
    __shared__ double part[WAVES];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_down(s, off, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = part[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += part[w];
    }
    return s;
}
// the norm, and min(1, max_norm / (norm + 1e-6)): NaN when the norm is, as torch.nn.utils.clip_grad_norm_ has it
__device__ __forceinline__ void norm_results(double sum, double max_norm, float* norm_out, float* clip_out) {
    const float norm = (float)sqrt(sum);
    const double c = max_norm / ((double)norm + 1e-6);
    *norm_out = norm;
    if (clip_out) *clip_out = max_norm > 0.0 ? (float)(c > 1.0 ? 1.0 : c) : 1.f;
}
template <bool NT, bool ROWS>
__global__ __launch_bounds__(256, 8) void grad_norm_kernel(NormTable<ROWS> t, uint32_t tiles, double* partial) {
    double s = 0.0;
    for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) s += norm_any_tile<NT, ROWS>(t, tile, 256, threadIdx.x);
    s = block_sum<4>(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}
__global__ __launch_bounds__(1024) void grad_norm_finish_kernel(const double* __restrict__ partial, int n, double max_norm, float* norm_out, float* clip_out) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 4096) {      // four loads in flight
        double x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = partial[min(i + 1024 * j, n - 1)];
#pragma unroll
        for (int j = 1; j < 4; ++j) x[j] = i + 1024 * j < n ? x[j] : 0.0;
        s += (x[0] + x[1]) + (x[2] + x[3]);
    }
    s = block_sum<16>(s);
    if (threadIdx.x == 0) norm_results(s, max_norm, norm_out, clip_out);
}
// few small tensors: one workgroup, a tile per WAVE, no second launch
template <bool ROWS>
__global__ __launch_bounds__(1024) void grad_norm_small_kernel(NormTable<ROWS> t, uint32_t tiles, double max_norm, float* norm_out, float* clip_out) {
    double s = 0.0;
    for (uint32_t tile = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); tile < tiles; tile += 16) s += norm_any_tile<false, ROWS>(t, tile, 64, threadIdx.x & 63);
    s = block_sum<16>(s);
    if (threadIdx.x == 0) norm_results(s, max_norm, norm_out, clip_out);
}

// ------------------------------------------------------------------------------------------------ host
int fail(const char* what) { g_last_error = what; return -2; }

size_t dtype_bytes(int dt) { return dt == F32 ? 4 : 2; }

// Non-temporal loads and stores for a call that touches more than half of the 256 MB memory-side cache: by the next step, the program has touched as much again, and lines that only
// pass through it cost write-backs of others.  A step over a map of f32 rows of 59, plain / non-temporal, with two other sets of its size stepped in between: 72 MiB 20.6 / 23.0 us,
// 108 MiB 34.0 / 33.0, 144 MiB 50.2 / 43.4, 270 MiB 90.5 / 80.4, 900 MiB 293 / 265; stepped alone again and again: 108 MiB 29.8 / 30.9, 270 MiB 72.0 / 79.4, 360 MiB 112 / 104.
// Values of codes to bf16: 17.7 M 20.9 / 27.1, 140 M 212 / 203 (in the one-wave form of the time).
bool stream_past_cache(unsigned long long bytes) { return bytes > 128ull << 20; }

// What a call writes must not overlap anything else it touches: a tensor given twice would be updated by two workgroups at once.  Gradients may overlap each other.
struct Range { uintptr_t begin, end; bool written; bool operator<(const Range& o) const { return begin < o.begin; } };
bool disjoint(std::vector<Range>& r) {
    if (!std::is_sorted(r.begin(), r.end())) std::sort(r.begin(), r.end());
    uintptr_t any = 0, written = 0;      // where what came before ends
    for (const Range& x : r) {
        if (x.begin < (x.written ? any : written)) return false;
        any = std::max(any, x.end);
        if (x.written) written = std::max(written, x.end);
    }
    return true;
}

// the multiplier of Rows::of for a width above 1
uint32_t row_magic(uint32_t w) { return (uint32_t)(((1ull << 32) * ((2ull << (31 - __builtin_clz(w - 1))) - w)) / w + 1); }

uint32_t tiles_of(long long numel) { return (uint32_t)((numel + TILE_ELEMS - 1) / TILE_ELEMS); }

struct StepCall {
    int n; void* const* params; const void* const* grads; float* const* masters; void* const* s0; void* const* s1;
    const long long* numel; const int* dtype; const double* lr; const double* wd; const int* place;
};

// fills one table from tensor k on and launches it; -> the next tensor
template <bool Q8, bool DEV>
int launch_step(const StepCall& c, int k, StepHyper& h, double inv_bc1, const gsicp_adamw_device* dev, bool masked, bool nt, hipStream_t stream) {
    StepTable<DEV> t = {};
    int n = 0;
    unsigned long long tiles = 0;
    h.src = k;
    for (; k < c.n && n < (DEV ? DEV_TABLE : TABLE) && tiles + tiles_of(c.numel[k]) <= STEP_TILES; ++k, ++n) {
        StepEntry& e = t.e[n];
        e.p = c.params[k]; e.g = c.grads[k]; e.s0 = c.s0[k]; e.s1 = c.s1[k]; e.master = c.masters ? c.masters[k] : nullptr;
        const uint64_t kind = (uint64_t)c.dtype[k] | (e.master ? 4u : 0u), place = (uint64_t)(c.place ? c.place[k] : k);
        e.word = (uint64_t)c.numel[k] | kind << 35 | place << 40;
        if constexpr (DEV) {
            e.wd = c.wd[k];
            const uint32_t w = dev->row_width && dev->row_width[k] > 0 ? (uint32_t)dev->row_width[k] : 0u;
            t.row_width[n] = w;
            if (w > 1) t.row_magic[n] = row_magic(w);
            if (dev->row_freeze && dev->group_frozen[k] && t.row_width[n] > 0) e.word |= 1ull << 38;
        } else {
            e.scale[0] = (float)(c.lr[k] * inv_bc1);
            e.scale[1] = (float)(1.0 - c.lr[k] * c.wd[k]);
        }
        t.first[n] = (uint32_t)tiles;
        tiles += tiles_of(c.numel[k]);
    }
    for (int i = n; i < 64; ++i) t.first[i] = LAST;
    if (tiles == 0) return k;
    const dim3 grid((unsigned)tiles);
    if constexpr (!DEV) {
        if (nt) hipLaunchKernelGGL((adamw_step_kernel<Q8, false, false, true>), grid, dim3(64), 0, stream, t, h);
        else hipLaunchKernelGGL((adamw_step_kernel<Q8, false, false, false>), grid, dim3(64), 0, stream, t, h);
    } else if (masked) {
        if (nt) hipLaunchKernelGGL((adamw_step_kernel<Q8, true, true, true>), grid, dim3(64), 0, stream, t, h);
        else hipLaunchKernelGGL((adamw_step_kernel<Q8, true, true, false>), grid, dim3(64), 0, stream, t, h);
    } else {
        if (nt) hipLaunchKernelGGL((adamw_step_kernel<Q8, true, false, true>), grid, dim3(64), 0, stream, t, h);
        else hipLaunchKernelGGL((adamw_step_kernel<Q8, true, false, false>), grid, dim3(64), 0, stream, t, h);
    }
    return k;
}

template <bool Q8>
int adamw_call(const StepCall& c, double b1, double b2, double eps, int step, uint32_t seed, const float* clip, const gsicp_adamw_device* dev, hipStream_t stream) {
    if (c.n < 0 || (c.n > 0 && (!c.params || !c.grads || !c.s0 || !c.s1 || !c.numel || !c.dtype || !c.wd))) return fail("gsicp_adamw_step: missing arrays");
    if (!(b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0 && eps >= 0.0)) return fail("gsicp_adamw_step: betas are in [0, 1), eps is not negative");
    // the hardware's reciprocal takes a subnormal for zero: an element that has never had a gradient would become 0 * inf
    if ((float)eps > 0.f && (float)eps < 0x1p-126f) return fail("gsicp_adamw_step: eps is 0 or at least 2^-126");
    if (dev) {
        if (!dev->lr_dev || !dev->step_dev || dev->bump_step < 0 || dev->bump_step > 2)
            return fail("gsicp_adamw_step: the device form needs learning rates, a step counter and bump_step 0, 1 or 2");
        if ((dev->live_rows || dev->row_freeze || dev->grad_rows) && !dev->row_width) return fail("gsicp_adamw_step: live rows and row masks need row_width");
        if (dev->row_freeze && !dev->group_frozen) return fail("gsicp_adamw_step: row_freeze needs group_frozen");
        if (Q8 && dev->row_freeze) return fail("gsicp_adamw_step_8bit: frozen rows would share block exponents with rows that move");
    } else if (step < 1 || (c.n > 0 && !c.lr)) {
        return fail("gsicp_adamw_step: the host form needs learning rates and a step count of at least 1");
    }
    const bool masked = dev && (dev->row_freeze || dev->grad_rows);
    static thread_local std::vector<Range> ranges;
    ranges.clear();
    unsigned long long bytes = 0;
    for (int k = 0; k < c.n; ++k) {
        const long long n = c.numel[k];
        if (n < 0 || n > MAX_NUMEL) return fail("gsicp_adamw_step: a tensor has 0 to 2^33 elements");
        const int dt = c.dtype[k], place = c.place ? c.place[k] : k;
        if (place < 0 || place >= (1 << 24)) return fail("gsicp_adamw_step: a place in the list is 0 to 2^24 - 1");
        if (n == 0) continue;
        if (dt < F32 || dt > F16) return fail("gsicp_adamw_step: dtype is 0 (f32), 1 (bf16) or 2 (f16)");
        float* master = c.masters ? c.masters[k] : nullptr;
        if (!c.params[k] || !c.grads[k] || !c.s0[k] || !c.s1[k]) return fail("gsicp_adamw_step: null pointer of a tensor that is not empty");
        if (master && dt == F32) return fail("gsicp_adamw_step: an f32 parameter has no master");
        if (masked && (dt != F32 || n >= (1ll << 32))) return fail("gsicp_adamw_step: row masks go with f32 parameters of less than 2^32 elements");
        auto add = [&](const void* q, size_t bytes, bool written = true) { ranges.push_back({(uintptr_t)q, (uintptr_t)q + bytes, written}); };
        add(c.grads[k], (size_t)n * dtype_bytes(dt), false);
        add(c.params[k], (size_t)n * dtype_bytes(dt));
        if (master) add(master, (size_t)n * 4);
        if (Q8) { add(c.s0[k], (size_t)n * 2); add(c.s1[k], (size_t)((n + QBLOCK - 1) / QBLOCK) * 2); }
        else { add(c.s0[k], (size_t)n * 4); add(c.s1[k], (size_t)n * 4); }
    }
    for (const Range& r : ranges) bytes += r.end - r.begin;
    if (!disjoint(ranges)) return fail("gsicp_adamw_step: a tensor that the step writes overlaps another one (the same given twice?)");

    StepHyper h = {};
    double inv_bc1 = 1.0;
    h.b1 = (float)b1; h.omb1 = (float)(1.0 - b1); h.b2 = (float)b2; h.omb2 = (float)(1.0 - b2); h.eps = (float)eps;
    h.ln_b1 = b1 > 0.0 ? std::log(b1) : -1e9; h.ln_b2 = b2 > 0.0 ? std::log(b2) : -1e9; h.clip = clip; h.seed = seed;
    if (dev) {
        h.lr_dev = dev->lr_dev; h.step_dev = dev->step_dev; h.step = dev->bump_step == 2 ? 0 : 1;
        h.guard_count = dev->guard_count; h.guard_limit = dev->guard_limit;
        h.live_rows = dev->live_rows; h.row_freeze = dev->row_freeze; h.grad_rows = dev->grad_rows;
    } else {
        h.step = step;
        inv_bc1 = 1.0 / (1.0 - std::pow(b1, step));
        h.inv_bc2_sqrt = (float)(1.0 / std::sqrt(1.0 - std::pow(b2, step)));
    }
    {
        ProfileScope ps(ST_ADAM, stream);
        const bool nt = stream_past_cache(bytes);
        for (int k = 0; k < c.n;)
            k = dev ? launch_step<Q8, true>(c, k, h, inv_bc1, dev, masked, nt, stream) : launch_step<Q8, false>(c, k, h, inv_bc1, dev, masked, nt, stream);
        if (dev && dev->bump_step == 1)
            hipLaunchKernelGGL(adamw_bump_kernel, dim3(1), dim3(1), 0, stream, dev->step_dev, dev->guard_count, dev->guard_limit, dev->skipped);
    }
    if (hipGetLastError() != hipSuccess) { g_last_error = "gsicp_adamw_step: kernel launch failed"; return -1; }
    return 0;
}

}  // namespace
}  // namespace gsicp

using namespace gsicp;

extern "C" {

int gsicp_adamw_step(int n, void* const* params, const void* const* grads, float* const* masters, float* const* exp_avg, float* const* exp_avg_sq,
                     const long long* numel, const int* dtype, const double* lr, const double* weight_decay, double beta1, double beta2, double eps, int step,
                     const float* clip, const gsicp_adamw_device* dev, void* stream) {
    try {
        return adamw_call<false>({n, params, grads, masters, (void* const*)exp_avg, (void* const*)exp_avg_sq, numel, dtype, lr, weight_decay, nullptr}, beta1, beta2, eps, step, 0u,
                                 clip, dev, (hipStream_t)stream);
    } catch (const std::exception& ex) { g_last_error = ex.what(); return -1; }
}

int gsicp_adamw_step_8bit(int n, void* const* params, const void* const* grads, float* const* masters, uint16_t* const* moments, uint16_t* const* block_exps,
                          const long long* numel, const int* dtype, const double* lr, const double* weight_decay, double beta1, double beta2, double eps, int step,
                          uint32_t seed, const int* place, const float* clip, const gsicp_adamw_device* dev, void* stream) {
    try {
        return adamw_call<true>({n, params, grads, masters, (void* const*)moments, (void* const*)block_exps, numel, dtype, lr, weight_decay, place}, beta1, beta2, eps, step, seed,
                                clip, dev, (hipStream_t)stream);
    } catch (const std::exception& ex) { g_last_error = ex.what(); return -1; }
}

int gsicp_adamw_decode(int n, const uint16_t* const* moments, const uint16_t* const* block_exps, void* const* exp_avg, void* const* exp_avg_sq, const long long* numel,
                       int dtype, void* stream_v) {
    hipStream_t stream = (hipStream_t)stream_v;
    if (n < 0 || (n > 0 && (!moments || !block_exps || !exp_avg || !exp_avg_sq || !numel))) return fail("gsicp_adamw_decode: missing arrays");
    if (dtype != F32 && dtype != BF16) return fail("gsicp_adamw_decode: dtype is 0 (f32) or 1 (bf16)");
    unsigned long long bytes = 0;
    for (int k = 0; k < n; ++k) {
        if (numel[k] < 0 || numel[k] > MAX_NUMEL) return fail("gsicp_adamw_decode: a tensor has 0 to 2^33 elements");
        if (numel[k] > 0 && (!moments[k] || !block_exps[k] || !exp_avg[k] || !exp_avg_sq[k])) return fail("gsicp_adamw_decode: null pointer of a tensor that is not empty");
        bytes += (unsigned long long)numel[k] * (dtype == F32 ? 10 : 6);
    }
    for (int k = 0; k < n;) {
        DecodeTable t = {};
        int m = 0;
        unsigned long long tiles = 0;
        for (; k < n && m < 64; ++k) {
            const unsigned long long more = (unsigned long long)((numel[k] + DECODE_ELEMS - 1) / DECODE_ELEMS);
            if (more == 0) continue;
            if (tiles + more > DECODE_TILES) break;
            t.e[m] = {moments[k], block_exps[k], exp_avg[k], exp_avg_sq[k], numel[k]};
            t.first[m++] = (uint32_t)tiles;
            tiles += more;
        }
        for (int i = m; i < 64; ++i) t.first[i] = LAST;
        if (m == 0) break;
        const dim3 grid((unsigned)tiles);
        const bool nt = stream_past_cache(bytes);
        if (dtype == F32 && nt) hipLaunchKernelGGL((adamw_decode_kernel<F32, true>), grid, dim3(256), 0, stream, t);
        else if (dtype == F32) hipLaunchKernelGGL((adamw_decode_kernel<F32, false>), grid, dim3(256), 0, stream, t);
        else if (nt) hipLaunchKernelGGL((adamw_decode_kernel<BF16, true>), grid, dim3(256), 0, stream, t);
        else hipLaunchKernelGGL((adamw_decode_kernel<BF16, false>), grid, dim3(256), 0, stream, t);
    }
    if (hipGetLastError() != hipSuccess) { g_last_error = "gsicp_adamw_decode: kernel launch failed"; return -1; }
    return 0;
}

int gsicp_adamw_gather_rows(int n, const uint16_t* const* moments, const uint16_t* const* block_exps, uint16_t* const* out_moments, uint16_t* const* out_exps,
                            const long long* row_width, const long long* index, long long n_rows, long long src_rows, void* stream_v) {
    hipStream_t stream = (hipStream_t)stream_v;
    if (n < 0 || n_rows < 0 || src_rows < 0 || (n > 0 && (!moments || !block_exps || !out_moments || !out_exps || !row_width))) return fail("gsicp_adamw_gather_rows: missing arrays");
    if (n > 0 && n_rows > 0 && !index) return fail("gsicp_adamw_gather_rows: missing index");
    try {
        std::vector<Range> ranges;
        for (int k = 0; k < n; ++k) {
            const long long w = row_width[k];
            if (w <= 0 || n_rows == 0 || src_rows == 0 || n_rows > 0xFFFFFFFFll / w || src_rows > MAX_NUMEL / w) continue;       // empty, or refused below
            auto add = [&](const void* q, long long numel, bool written) { ranges.push_back({(uintptr_t)q, (uintptr_t)q + 2 * (size_t)numel, written}); };
            add(moments[k], src_rows * w, false); add(block_exps[k], (src_rows * w + QBLOCK - 1) / QBLOCK, false);
            add(out_moments[k], n_rows * w, true); add(out_exps[k], (n_rows * w + QBLOCK - 1) / QBLOCK, true);
        }
        if (!disjoint(ranges)) return fail("gsicp_adamw_gather_rows: the result overlaps its source or itself");
    } catch (const std::exception& ex) { g_last_error = ex.what(); return -1; }
    for (int k = 0; k < n; ++k) {
        const long long w = row_width[k];
        if (w < 0 || (w > 0 && (n_rows > 0xFFFFFFFFll / w || src_rows > MAX_NUMEL / w))) return fail("gsicp_adamw_gather_rows: a tensor has less than 2^32 elements");
        if (w == 0 || n_rows == 0) continue;
        if (!moments[k] || !block_exps[k] || !out_moments[k] || !out_exps[k]) return fail("gsicp_adamw_gather_rows: null pointer of a tensor that is not empty");
    }
    for (int k = 0; k < n;) {
        GatherTable t = {};
        int m = 0;
        unsigned long long tiles = 0;
        for (; k < n && m < TABLE; ++k) {
            const long long numel = n_rows * row_width[k];
            if (numel == 0) continue;
            if (tiles + tiles_of(numel) > STEP_TILES) break;
            const uint32_t w = (uint32_t)row_width[k];
            t.e[m] = {moments[k], block_exps[k], out_moments[k], out_exps[k], w, w > 1 ? row_magic(w) : 0u};
            t.first[m++] = (uint32_t)tiles;
            tiles += tiles_of(numel);
        }
        for (int i = m; i < 64; ++i) t.first[i] = LAST;
        if (m == 0) break;
        hipLaunchKernelGGL(adamw_gather_kernel, dim3((unsigned)tiles), dim3(64), 0, stream, t, index, (uint32_t)n_rows, src_rows);
    }
    if (hipGetLastError() != hipSuccess) { g_last_error = "gsicp_adamw_gather_rows: kernel launch failed"; return -1; }
    return 0;
}

// few small tensors, which one workgroup adds up in one launch
static bool norm_is_small(int n, const long long* numel, const int* dtype) {
    unsigned long long tiles = 0;
    int used = 0;
    for (int k = 0; k < n && used <= NORM_TABLE && tiles <= NORM_SMALL_TILES; ++k) {
        if (numel[k] <= 0) continue;
        ++used;
        const int te = norm_tile_elems(dtype[k], 64 * 64);
        tiles += (unsigned long long)((numel[k] + te - 1) / te);
    }
    return used <= NORM_TABLE && tiles <= NORM_SMALL_TILES;
}

size_t gsicp_grad_norm_scratch_bytes(int n, const long long* numel, const int* dtype) {
    return n <= 0 || !numel || !dtype || norm_is_small(n, numel, dtype) ? 0 : (size_t)((n + NORM_ROWS_TABLE - 1) / NORM_ROWS_TABLE) * NORM_GRID * sizeof(double);
}

}  // extern "C"

// ROWS: live_rows, row_width, row_freeze and group_frozen of *rows apply
template <bool ROWS>
static int grad_norm_call(int n, const void* const* grads, const long long* numel, const int* dtype, const gsicp_adamw_device* rows, double max_norm, float* norm_out,
                          float* clip_out, void* scratch, hipStream_t stream) {
    constexpr int ENTRIES = ROWS ? NORM_ROWS_TABLE : NORM_TABLE;
    if (n < 0 || (n > 0 && (!grads || !numel || !dtype)) || !norm_out) return fail("gsicp_grad_norm: missing arrays");
    if (ROWS && n > 0 && !rows->row_width) return fail("gsicp_grad_norm: live rows and frozen rows need row_width");
    if (ROWS && rows->row_freeze && !rows->group_frozen) return fail("gsicp_grad_norm: row_freeze needs group_frozen");
    for (int k = 0; k < n; ++k) {
        if (numel[k] < 0 || numel[k] > MAX_NUMEL) return fail("gsicp_grad_norm: a tensor has 0 to 2^33 elements");
        if (numel[k] == 0) continue;
        if (!grads[k] || dtype[k] < F32 || dtype[k] > F16) return fail("gsicp_grad_norm: null pointer, or a dtype that is not 0 (f32), 1 (bf16) or 2 (f16)");
        if ((uint64_t)(uintptr_t)grads[k] >> 58) return fail("gsicp_grad_norm: an address has less than 2^58");
        if (ROWS && rows->row_freeze && rows->group_frozen[k] && (dtype[k] != F32 || numel[k] >= (1ll << 32)))
            return fail("gsicp_grad_norm: frozen rows go with f32 gradients of less than 2^32 elements");
    }
    const bool one = norm_is_small(n, numel, dtype);      // at most NORM_SMALL_TILES tensors then: one table of either kind
    if (!one && !scratch) return fail("gsicp_grad_norm: missing scratch");
    const int tile_bytes = one ? 64 * 64 : 256 * 64;
    double* partial = (double*)scratch;
    int used = 0;
    for (int k = 0; k < n || one;) {
        NormTable<ROWS> t = {};
        int m = 0;
        unsigned long long tiles = 0;
        for (; k < n && m < ENTRIES; ++k) {
            if (numel[k] == 0) continue;
            bool frozen = false;
            if constexpr (ROWS) {
                const uint32_t w = rows->row_width[k] > 0 ? (uint32_t)rows->row_width[k] : 0u;
                t.row_width[m] = w;
                t.row_magic[m] = w > 1 ? row_magic(w) : 0u;
                frozen = rows->row_freeze && rows->group_frozen[k] && w > 0;
            }
            t.e[m].set(grads[k], numel[k], dtype[k], frozen);
            t.first[m++] = (uint32_t)tiles;
            const int te = norm_tile_elems(dtype[k], tile_bytes);
            tiles += (unsigned long long)((numel[k] + te - 1) / te);       // at most 2^21 of one tensor
        }
        for (int i = m; i < (int)(sizeof(t.first) / sizeof(t.first[0])); ++i) t.first[i] = LAST;
        if constexpr (ROWS) { t.live_rows = rows->live_rows; t.row_freeze = rows->row_freeze; }
        if (one) {
            hipLaunchKernelGGL((grad_norm_small_kernel<ROWS>), dim3(1), dim3(1024), 0, stream, t, (uint32_t)tiles, max_norm, norm_out, clip_out);
            break;
        }
        if (m == 0) break;
        const unsigned grid = (unsigned)std::min<unsigned long long>(tiles, NORM_GRID);
        // Before a clipped step the gradients had better stay in the memory-side cache for it (its own streams pass by): norm and step of 225 MiB of gradients 278 us, with
        // non-temporal loads here 302, of 45 MiB 61 and 66.  The norm alone is better off without: 43 and 39 us, 12.4 and 12.3.
        if (ROWS || max_norm > 0.0) hipLaunchKernelGGL((grad_norm_kernel<false, ROWS>), dim3(grid), dim3(256), 0, stream, t, (uint32_t)tiles, partial + used);
        else hipLaunchKernelGGL((grad_norm_kernel<!ROWS, ROWS>), dim3(grid), dim3(256), 0, stream, t, (uint32_t)tiles, partial + used);
        used += (int)grid;
    }
    if (!one) hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(1024), 0, stream, (const double*)partial, used, max_norm, norm_out, clip_out);
    if (hipGetLastError() != hipSuccess) { g_last_error = "gsicp_grad_norm: kernel launch failed"; return -1; }
    return 0;
}

extern "C" {

int gsicp_grad_norm(int n, const void* const* grads, const long long* numel, const int* dtype, double max_norm, float* norm_out, float* clip_out, void* scratch,
                    void* stream) {
    return grad_norm_call<false>(n, grads, numel, dtype, nullptr, max_norm, norm_out, clip_out, scratch, (hipStream_t)stream);
}

int gsicp_grad_norm_rows(int n, const void* const* grads, const long long* numel, const int* dtype, const gsicp_adamw_device* rows, double max_norm, float* norm_out,
                         float* clip_out, void* scratch, void* stream) {
    if (!rows || rows->grad_rows) return fail("gsicp_grad_norm_rows: rows is missing, or has gradients of which some rows were not written");
    return grad_norm_call<true>(n, grads, numel, dtype, rows, max_norm, norm_out, clip_out, scratch, (hipStream_t)stream);
}

}  // extern "C"
