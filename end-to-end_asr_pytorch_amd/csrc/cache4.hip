// K / V cache held in 4 bits: quantising put, reading back, attention over it, re-gathering by parent hypothesis (asr_hip.h: asr_cache4_*).
//
// A row of 64 values (one head of one token) is 32 bytes of signed codes - byte j: value 2j in the low nibble, 2j + 1 in the high one - and
// one 32-bit word, the bf16 pair (scale low, mid high): value = mid + scale * code.  scale = bf16((max - min) * (1/15)) and mid = bf16(min
// + 8 scale) put min at code -8 and max at 7 with half a step of room on either side, which is what the two bf16 roundings may use up (mid's is
// half a step only where |mid| > 256 scale: rows whose level is 17 times their spread).
#include <type_traits>

#include "asr_common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(2))) int i32x2;

constexpr int CACHE4_MAX_T = 1 << 24;      // slots of a row: 32-bit offsets inside a row (32 bytes a slot), 64-bit ones in front of it

__device__ __forceinline__ uint32_t bf16_bits(float x) { return (uint32_t)__builtin_bit_cast(uint16_t, (bf16_t)x); }
__device__ __forceinline__ float meta_scale(uint32_t m) { return __builtin_bit_cast(float, m << 16); }
__device__ __forceinline__ float meta_mid(uint32_t m) { return __builtin_bit_cast(float, m & 0xffff0000u); }
__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// ---- 16 consecutive values of a row ---------------------------------------------------------------------------------------------------
template <typename T> struct Row16;
template <> struct Row16<bf16_t> {
    u32x4 w[2];
    __device__ __forceinline__ void load(const bf16_t* p) { w[0] = reinterpret_cast<const u32x4*>(p)[0]; w[1] = reinterpret_cast<const u32x4*>(p)[1]; }
    __device__ __forceinline__ void widen(float (&v)[16]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) { v[2 * i] = meta_scale(w[i >> 2][i & 3]); v[2 * i + 1] = meta_mid(w[i >> 2][i & 3]); }
    }
};
template <> struct Row16<float> {
    f32x4 w[4];
    __device__ __forceinline__ void load(const float* p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const f32x4*>(p)[i];
    }
    __device__ __forceinline__ void widen(float (&v)[16]) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = w[i >> 2][i & 3];
    }
};
__device__ __forceinline__ void store8(bf16_t* p, const float (&v)[8]) {
    bf16x8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (bf16_t)v[i];
    *reinterpret_cast<bf16x8*>(p) = o;
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
}

template <int CTRL> __device__ __forceinline__ float dpp_f(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// d / s with one correction: the quotient rounded to nearest (where it has few bits - on a border k + 1/2 - exactly that), rs = 1 / s to an ulp or two
__device__ __forceinline__ float quotient(float d, float s, float rs) {
    const float y = d * rs;
    return __builtin_fmaf(__builtin_fmaf(-y, s, d), rs, y);
}

// Quantising reads 128 (bf16) or 256 bytes a row and writes 36: HBM, with the VALU next to it (11 instructions a value, 27 us of issue at 2.4 GHz
// for the 1.15 M rows below).  4 lanes a row share the row's own arithmetic (8 lanes: 3 instructions a value more); the next row's loads are
// in flight while this one is worked on.  Measured: 12 x 32 x 4 rows of 1000 tokens in bf16 54.5 us = 4.6 TB/s (a copy of 1 GiB moves 5.15 here);
// rows of 500 to 1000 tokens 60 us = 3.2 TB/s behind a launch whose 197 MB of results are still on their way to memory (51 at best).
//
// The codes of 16 values of a row whose 64 values lie in 4 neighbouring lanes: -> the two 32-bit words of nibbles, and the row's (scale, mid).
// Every decision is that of (x - mid) / scale computed exactly.  The corrected quotient settles it unless the subtraction was rounded and
// the quotient is next to a border:
//   bf16  x and mid have 8 bits, so d = x - mid is exact unless one of them is 2^-16 of the other.  |mid| is 0 or at least 2^-6 scale and |x|
//         at most 17 scale; a tiny x leaves d = -mid, which can only matter if mid itself lies on a border.  Elsewhere a quotient that is
//         not on a border is 2^-20 away from it or more, and its error below 8 is under 2^-22.
//   f32   any value may be within the error of a border: those closer than 2^-19 are looked at again.
// (Exact for all of them, with the rounding error of the subtraction carried along, is 12 instructions a value more: VALU-bound.)
template <typename T> __device__ __forceinline__ u32x2 quantise16(const float (&x)[16], uint32_t& meta) {
#pragma clang fp contract(off)
    float lo = x[0], hi = x[0];      // (v_minimum3 / v_maximum3: a NaN stays, an infinity is an extreme - span is finite only if every value is)
#pragma unroll
    for (int i = 1; i < 16; ++i) {
        lo = __builtin_elementwise_minimum(lo, x[i]);
        hi = __builtin_elementwise_maximum(hi, x[i]);
    }
    lo = __builtin_elementwise_minimum(lo, dpp_f<0xB1>(lo));      // quad_perm: lane xor 1, lane xor 2
    hi = __builtin_elementwise_maximum(hi, dpp_f<0xB1>(hi));
    lo = __builtin_elementwise_minimum(lo, dpp_f<0x4E>(lo));
    hi = __builtin_elementwise_maximum(hi, dpp_f<0x4E>(hi));
    const float span = hi - lo;
    const bool finite = span < INFINITY;
    const float sc = span < 0x1p-100f || !finite ? 0.f : (float)(bf16_t)(span * (1.f / 15.f));      // (the format: a product, not a quotient)
    const float mid = (float)(bf16_t)(lo + 8.f * sc);
    const bool fine = finite && fabsf(mid) < INFINITY;      // (a middle that rounds past bf16's largest is no middle)
    meta = fine ? bf16_bits(sc) | (bf16_bits(mid) << 16) : 0x7fc07fc0u;
    if (sc == 0.f || !fine) return u32x2{0u, 0u};
    const float rs = __builtin_amdgcn_rcpf(sc);
    constexpr float MAGIC = 12582912.f + 8.f;      // 1.5 * 2^23: adding it rounds to the nearest integer, ties to even, and leaves code + 8 in the low bits
    float y[16], near = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        y[i] = quotient(x[i] - mid, sc, rs);
        if (sizeof(T) == 4) near = fmaxf(near, fabsf(y[i] - __builtin_rintf(y[i])));
        y[i] = __builtin_amdgcn_fmed3f(y[i], -8.f, 7.f);
    }
    bool again = near > 0.5f - 0x1p-19f;
    if (sizeof(T) == 2) {
        const float ym = 2.f * quotient(mid, sc, rs);
        again = __builtin_rintf(ym) == ym && __builtin_rintf(0.5f * ym) != 0.5f * ym;
    }
    if (__builtin_expect(again, 0)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float d = x[i] - mid, bb = d - x[i], e = (x[i] - (d - bb)) + (-mid - bb);      // d + e = x - mid exactly
            const float k = __builtin_rintf(y[i]), r = __builtin_fmaf(-k, sc, d);                // exact next to a border: k sc has 12 bits
            const float g = (fabsf(r) - 0.5f * sc) + (r > 0.f ? e : -e);                         // > 0: the neighbour is nearer
            const bool move = (g > 0.f) | ((g == 0.f) & (((int)k & 1) != 0));
            y[i] = __builtin_amdgcn_fmed3f(move ? k + __builtin_copysignf(1.f, r) : k, -8.f, 7.f);
        }
    }
    u32x2 w;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        uint32_t p[4];      // the low byte: two codes
#pragma unroll
        for (int i = 0; i < 4; ++i)
            p[i] = __builtin_bit_cast(uint32_t, y[8 * j + 2 * i] + MAGIC) | (__builtin_bit_cast(uint32_t, y[8 * j + 2 * i + 1] + MAGIC) << 4);
        w[j] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(p[3], p[2], 0x0c0c0400u), __builtin_amdgcn_perm(p[1], p[0], 0x0c0c0400u), 0x05040100u);
    }
    return w ^ 0x88888888u;      // offset code -> two's complement nibble
}

// Slots of one call: which rows a block works on.  A block is 256 / LANES groups of LANES lanes, one row of 64 values each; 2^tb_log2 tokens
// of as many rows as fill the block side by side, so that a single token per row fills it as well as a long chunk does.  A long chunk's
// block belongs to one row (ONE_ROW: its addresses are scalar) and walks `iter` times its width.
struct slots_t {
    const int32_t* pos; const int32_t* n_tok;
    int pos_stride, N, h, L, Tmax, tb_log2, rb_log2, iter, chunks, rows;
};
struct strides_t { int64_t kv, n, head, tok; };
struct range_t { int64_t x0, c0; int i, end, step, lo, hi; };      // tokens i, i + step, .. < end; those of [lo, hi) have a slot: c0 + token

template <int LANES, bool ONE_ROW> __device__ __forceinline__ bool range_of(const slots_t& s, const strides_t& st, range_t& r) {
    const int chunk = s.chunks == 1 ? 0 : blockIdx.x % s.chunks, rows = s.chunks == 1 ? blockIdx.x : blockIdx.x / s.chunks, group = threadIdx.x / LANES;
    const int row = ONE_ROW ? rows : (rows << s.rb_log2) + (group >> s.tb_log2);
    if (row >= s.rows) return false;
    const int head = row % s.h, kn = row / s.h, n = kn % s.N, kv = kn / s.N;
    const int64_t first = s.pos ? s.pos[(int64_t)n * s.pos_stride] : 0, room = (int64_t)s.Tmax - first;
    const int count = s.n_tok ? clampi(s.n_tok[n], 0, s.L) : s.L;
    r.lo = first < 0 ? (int)(-first < s.L ? -first : s.L) : 0;
    r.hi = (int)(room < count ? (room > 0 ? room : 0) : count);
    r.x0 = kv * st.kv + n * st.n + head * st.head;
    r.c0 = (int64_t)row * s.Tmax + first;
    r.step = 1 << s.tb_log2;
    const int t0 = chunk * (s.iter << s.tb_log2);
    r.i = t0 + (group & (r.step - 1));
    r.end = min(t0 + (s.iter << s.tb_log2), s.L);
    return true;
}

template <typename T, bool ONE_ROW>
__global__ __launch_bounds__(256) void cache4_put_kernel(const T* __restrict__ x, strides_t st, uint32_t* __restrict__ codes,
                                                         uint32_t* __restrict__ meta, slots_t s) {
    range_t r;
    if (!range_of<4, ONE_ROW>(s, st, r)) return;
    const int l4 = threadIdx.x & 3, end = min(r.end, r.hi);
    const T* px = x + r.x0 + l4 * 16;
    uint32_t* pc = codes + r.c0 * 8 + l4 * 2;
    uint32_t* pm = meta + r.c0;
    int i = r.i;
    if (i < r.lo) i += (r.lo - i + r.step - 1) & ~(r.step - 1);
    if (i >= end) return;      // (one token's 4 lanes agree, here and below)
    Row16<T> w;
    w.load(px + (int64_t)i * st.tok);
    for (; i < end; i += r.step) {
        float v[16];
        w.widen(v);
        if (i + r.step < end) w.load(px + (int64_t)(i + r.step) * st.tok);      // the next row's while this one is worked on
        uint32_t m;
        const u32x2 c = quantise16<T>(v, m);
        *reinterpret_cast<u32x2*>(pc + (unsigned)i * 8u) = c;
        if (l4 == 0) pm[(unsigned)i] = m;
    }
}

// Reading back: 36 bytes in, 128 or 256 out.  8 lanes a row, 16 bytes (bf16) of output each: whole cache lines per store.  Measured: 12 x 32 x 4
// rows of 1000 tokens to bf16 42.8 us = 5.9 TB/s.
template <typename T, bool ONE_ROW>
__global__ __launch_bounds__(256) void cache4_get_kernel(T* __restrict__ out, strides_t st, const uint32_t* __restrict__ codes,
                                                         const uint32_t* __restrict__ meta, slots_t s) {
    range_t r;
    if (!range_of<8, ONE_ROW>(s, st, r)) return;
    const int l8 = threadIdx.x & 7;
    T* po = out + r.x0 + l8 * 8;
    const uint32_t* pc = codes + r.c0 * 8 + l8;
    const uint32_t* pm = meta + r.c0;
#pragma unroll 2
    for (int i = r.i; i < r.end; i += r.step) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (i >= r.lo && i < r.hi) {
            const uint32_t w = pc[(unsigned)i * 8u], m = pm[(unsigned)i];
            const float sc = meta_scale(m), mid = meta_mid(m);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __builtin_fmaf(sc, (float)((int)(w << (28 - 4 * j)) >> 28), mid);      // one rounding: sc * code is exact
        }
        store8(po + (int64_t)i * st.tok, v);
    }
}

// ---- re-gathering by parent ------------------------------------------------------------------------------------------------------------
// A group is one (kv, utterance, head).  A block takes 256 pieces of its positions - 16-byte halves of the codes, or meta words - and a thread
// its piece for all the beam's rows: it reads every source row's before it writes any, so source and destination may be the same cache.  The
// parents are the same for a whole block: lane r of a wave reads row r's, row addresses are scalar (with them in vector registers: 236 VGPRs, 70 us).
// Measured: 12 x 8 utterances x 8 beams x 4 heads x 777 positions into another cache 44 us = 3.9 TB/s (40 at best), 29.6 where the Infinity Cache
// holds both, 26.5 there in place; a step of 32 x 5 beams, 51 positions 8.2 us, in place 7.4.
template <typename V, int BEAM> __device__ __forceinline__ void regather(const V* src, V* dst, unsigned parents, int64_t row, int beam, unsigned u,
                                                                         bool in_place) {
    V v[BEAM];
    int from[BEAM];
#pragma unroll
    for (int r = 0; r < BEAM; ++r) {
        from[r] = (parents >> (4 * r)) & 15;
        if (r < beam && !(in_place && from[r] == r)) v[r] = (src + (int64_t)from[r] * row)[u];
    }
#pragma unroll
    for (int r = 0; r < BEAM; ++r)
        if (r < beam && !(in_place && from[r] == r)) (dst + (int64_t)r * row)[u] = v[r];
}

template <int BEAM>
__global__ __launch_bounds__(256) void cache4_reorder_kernel(const u32x4* codes, const uint32_t* meta, u32x4* out_codes, uint32_t* out_meta,
                                                             const int64_t* __restrict__ parent, const int32_t* __restrict__ state, int B,
                                                             int beam, int h, int Tmax, int chunks_codes, int chunks_meta, int in_place) {
    const int chunks = chunks_codes + chunks_meta, grp = blockIdx.x / chunks;
    int chunk = blockIdx.x % chunks;
    const int hd = grp % h, kb = grp / h, b = kb % B;
    const int64_t row0 = ((int64_t)kb * beam * h + hd) * Tmax;      // slots in front of the group's first row
    const int n = clampi(state[0], -1, Tmax - 1) + 1;
    const bool is_meta = chunk >= chunks_codes;
    if (is_meta) chunk -= chunks_codes;
    const unsigned u = chunk * 256u + threadIdx.x;
    const unsigned live = is_meta ? n : 2 * n;
    if ((u & ~63u) >= live) return;      // (whole waves: in the others all lanes are there for the parents)
    // lane r: the source row of row r within the utterance.  Compared as 64 bits: an id far outside must not come back modulo 2^32
    const int64_t first = (int64_t)b * beam, id = parent[first + min((int)threadIdx.x & 63, beam - 1)];
    const int mine = id < first ? 0 : id < first + beam ? (int)(id - first) : beam - 1;
    unsigned parents = 0;      // four bits a row.  (Read in front of the return: behind it lane r may be gone)
#pragma unroll
    for (int r = 0; r < BEAM; ++r) parents |= (unsigned)__builtin_amdgcn_readlane(mine, r) << (4 * r);
    if (u >= live) return;
    if (is_meta) regather<uint32_t, BEAM>(meta + row0, out_meta + row0, parents, (int64_t)h * Tmax, beam, u, in_place);
    else regather<u32x4, BEAM>(codes + row0 * 2, out_codes + row0 * 2, parents, (int64_t)h * Tmax * 2, beam, u, in_place);
}

// ---- attention ---------------------------------------------------------------------------------------------------------------------------
// With k_j = mid_j + scale_j c_j and v_j = mid'_j + scale'_j c'_j:
//     s_j = scale_j (q . c_j) + mid_j sum(q)           p_j = 2^(s_j - m)
//     o   = (sum_j p_j mid'_j + sum_j (p_j scale'_j) c'_j) / sum_j p_j
// Both products run over the codes themselves, on the int8 matrix instruction: a nibble masked in place is the byte 16 c, three VALU
// operations for eight codes, and no value of the cache is ever widened.  The other operand is cut into int8 digits of base 256: the query
// once per launch (relative to its largest element), the weights w_j = p_j scale'_j once per tile of 64 tokens (relative to the tile's
// largest, so a tile of small weights keeps its precision).  ND = 2 digits for bf16 queries (half a step is 2^-16 of the largest, below the
// 2^-9 that a bf16 weight is rounded by), 3 for f32 (2^-24).  The products are exact int32; softmax statistics and the output are f32.
//
// A wave owns 64 tokens at a time, token = lane.  A 16-byte load of K is half a token's channels, so the four lane groups of a QK instruction
// hold the halves of two tokens: the query operand is zero in the rows whose results land with the other token, and an accumulator of 32
// tokens holds (2 queries x 2 digits, or 1 x 3) a lane.
// The weights go through LDS (16 bytes per token: all digits of all queries) into the A operand of the PV product - ds_read_b64_tr_b8 turns
// them into rows (query, digit) - whose B operand, 16 tokens of one channel per lane, is what ds_read_b64_tr_b4 makes of the tile's
// row-major codes.
// The running reference m of a query is renewed only when a score passes it by LAG (weights are f32 and scaled per tile: nothing needs them
// below 1), so a tile costs one reduction across the wave per query, the largest weight's, and four queries share its steps.  Sums of weights
// times values grow to 2^LAG times what the values themselves add up to, and have to stay below f32's 2^128: with LAG 8 that leaves 2^119
// for the values of a row (|mid| + 8 scale) and a bit to spare.  LAG 32 takes 24 bits of that range and is no faster where the (base-2)
// scores have a standard deviation of 1.4 (18 sizes and types within 1 %); at 5.8 it gains up to 2 % with 256 queries, nothing with few.
// The next tile's loads are issued before the present one is worked on, the first tile's before the query is.
//
// What bounds it: HBM for long rows (72 bytes a token and head; 4 rows x 4 heads of up to 100003 slots, 16 splits: 20.5 us = 4.6 TB/s, + 3.9 us for
// the join), launch and one chain of loads for a decoding step (32 x 4 rows of 1000 slots: 5.3 us a replayed call with one query, 6.5 with
// five), the VALU and the chain of a tile for many queries (the dense kernel below).
template <int ND> struct Digits {
    static constexpr float UNIT = ND == 2 ? 127.f * 256.f : 127.f * 65536.f;      // the integer that the largest element becomes
    static constexpr int BIAS = ND == 2 ? 0x80 : 0x8080;                          // u + BIAS, its lower bytes' sign bits inverted: the digits, lowest first
    static constexpr int QPP = ND == 2 ? 2 : 1;                                   // queries per accumulator
    static __device__ __forceinline__ float join(int d0, int d1, int d2) {
        const float low = (float)((d1 << 8) + d0);
        return ND == 2 ? low : __builtin_fmaf((float)d2, 65536.f, low);
    }
};

struct attn4_t {
    const void* q; int64_t q_n, q_head, q_tok;
    const u32x4* kc; const uint32_t* km; const u32x4* vc; const uint32_t* vm;
    void* ctx; float* lse; float* part;
    const int32_t* k_len;
    int h, h_kv, Lq, T, splits, qtiles, per_tile, rows, waves;
};
constexpr int PART = 66;      // floats of a partial result: 64 outputs (not divided), reference, sum
constexpr int MAX_NQ = 4, MAX_WAVES = 8, DENSE_ROW = 68;
constexpr int TILE_V = 64 * 32, WAVE_LDS = TILE_V + 64 * 16;      // LDS bytes of a wave: a tile's codes of V; 16 bytes a token behind them
constexpr float NO_REF = -3.4028234663852886e38f;
constexpr float LAG = 8.f;      // log2

// position of element k of 16 in the byte order that unpacking leaves: low nibbles of the first word, its high ones, then the second word's
__device__ __forceinline__ int unpack_pos(int k) { return (k & 8) + (k & 1) * 4 + ((k >> 1) & 3); }
__device__ __forceinline__ i32x4 unpack16(uint32_t w0, uint32_t w1) {
    return i32x4{(int)((w0 << 4) & 0xf0f0f0f0u), (int)(w0 & 0xf0f0f0f0u), (int)((w1 << 4) & 0xf0f0f0f0u), (int)(w1 & 0xf0f0f0f0u)};
}

// ---- reductions over the wave: v_permlane32_swap / v_permlane16_swap exchange halves / rows of two registers, the 16 lanes of a row by DPP ----
struct MaxPos {      // non-negative floats as their bit patterns (a NaN stays the largest)
    static __device__ __forceinline__ uint32_t f(uint32_t a, uint32_t b) { return max(a, b); }
};
struct MaxF {
    static __device__ __forceinline__ uint32_t f(uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_maximum(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));      // (a NaN stays)
    }
};
struct SumF {
    static __device__ __forceinline__ uint32_t f(uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
    }
};
template <typename OP, int CTRL> __device__ __forceinline__ uint32_t dpp_step(uint32_t x) {
    return OP::f(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false));
}
template <typename OP> __device__ __forceinline__ uint32_t row16(uint32_t x) {      // row_ror 8, 4, 2, 1
    x = dpp_step<OP, 0x128>(x);
    x = dpp_step<OP, 0x124>(x);
    x = dpp_step<OP, 0x122>(x);
    return dpp_step<OP, 0x121>(x);
}
template <typename OP> __device__ __forceinline__ uint32_t swap32(uint32_t a, uint32_t b) {      // lanes 0..31: a's both halves, 32..63: b's
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    return OP::f(r[0], r[1]);
}
template <typename OP> __device__ __forceinline__ uint32_t swap16(uint32_t a, uint32_t b) {      // even rows: a's row pair, odd rows: b's
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    return OP::f(r[0], r[1]);
}
template <typename OP> __device__ __forceinline__ float wave_all(float v) {      // the same for all lanes
    uint32_t x = __builtin_bit_cast(uint32_t, v);
    x = swap32<OP>(x, x);
    x = swap16<OP>(x, x);
    return __builtin_bit_cast(float, row16<OP>(x));
}
// over the four rows of 16 lanes: lanes of the same place in their rows
template <typename OP> __device__ __forceinline__ float over_c(float v) {
    const uint32_t x = swap32<OP>(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v));
    return __builtin_bit_cast(float, swap16<OP>(x, x));
}
// four values at once: row c of the result holds value c's, 9 steps instead of 24
template <typename OP> __device__ __forceinline__ float wave_four(float v0, float v1, float v2, float v3) {
    const uint32_t a = swap32<OP>(__builtin_bit_cast(uint32_t, v0), __builtin_bit_cast(uint32_t, v2));
    const uint32_t b = swap32<OP>(__builtin_bit_cast(uint32_t, v1), __builtin_bit_cast(uint32_t, v3));
    return __builtin_bit_cast(float, row16<OP>(swap16<OP>(a, b)));
}

__device__ __forceinline__ void wave_lds_fence() {      // LDS written by other lanes of this wave
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

struct tile4_t { u32x4 kw[2], vw[2]; uint32_t km, vm; };
// a tile's 64 tokens, cut to `last` (what is behind the row's last token is masked where it is used)
__device__ __forceinline__ void load_tile(tile4_t& t, const u32x4* kc, const u32x4* vc, const uint32_t* km, const uint32_t* vm, int t0, int last, int lane) {
    const int n16 = lane & 15, c = lane >> 4;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        t.kw[j] = kc[(unsigned)min(t0 + 32 * j + 16 * (c >> 1) + n16, last) * 2u + (c & 1)];
        t.vw[j] = vc[(unsigned)min(t0 + 32 * j + (lane >> 1), last) * 2u + (lane & 1)];
    }
    const unsigned tok = min(t0 + lane, last);
    t.km = km[tok];
    t.vm = vm[tok];
}

// ---- what the two attention kernels share -----------------------------------------------------------------------------------------------
struct work4_t { int row, split, n, hk, group, q0, nq; int64_t base; };
// block -> (row, query tile, split): the query tiles of one stream of keys follow each other at a distance of 8 blocks (one XCD's L2)
__device__ __forceinline__ bool work_of(const attn4_t& a, work4_t& b) {
    int stream = blockIdx.x, qt = 0;
    if (a.qtiles > 1) {
        const int per8 = 8 * a.qtiles, oct = stream / per8, rest = stream - oct * per8;
        stream = oct * 8 + (rest & 7);
        qt = rest >> 3;
    }
    if (stream >= a.rows * a.splits) return false;
    b.row = a.splits == 1 ? stream : stream / a.splits;
    b.split = stream - b.row * a.splits;
    b.n = a.h_kv == 1 ? b.row : b.row / a.h_kv;
    b.hk = b.row - b.n * a.h_kv;
    b.base = (int64_t)b.row * a.T;
    b.group = a.h / a.h_kv;
    b.q0 = qt * a.per_tile;
    b.nq = min(a.per_tile, b.group * a.Lq - b.q0);
    return true;
}
// the digits of a block's queries, [width][ND][64] in the unpacked operands' order, and behind them [width][2]: the unit of the digits (with the
// codes' 16), the sum in that unit.  Queries that are not there become zeros.
template <typename T, int ND> __device__ __forceinline__ float* query_digits(const attn4_t& a, const work4_t& b, int width, unsigned char* sm_q, int wave, int W, int lane) {
    using D = Digits<ND>;
    float* sm_qs = reinterpret_cast<float*>(sm_q + width * ND * 64);
    for (int j = wave; j < width; j += W) {
        float v = 0.f;
        if (j < b.nq) {
            const int qi = b.q0 + j, g = a.Lq == 1 ? qi : qi / a.Lq, i = qi - g * a.Lq;
            v = to_f32(static_cast<const T*>(a.q)[b.n * a.q_n + (b.hk * b.group + g) * a.q_head + i * a.q_tok + lane]);
        }
        const float top = wave_all<MaxPos>(fabsf(v)), sum = wave_all<SumF>(v);
        const bool some = !(top < 0x1p-100f);      // (below: a query of zeros)
        const uint32_t u = some ? (uint32_t)((int)__builtin_rintf(v * (D::UNIT / top)) + D::BIAS) ^ D::BIAS : 0u;
#pragma unroll
        for (int d = 0; d < ND; ++d) sm_q[(j * ND + d) * 64 + (lane & 48) + unpack_pos(lane & 15)] = (unsigned char)(u >> (8 * d));
        const float unit = some ? top * (1.f / (16.f * D::UNIT)) : 1.f;
        if (lane == 0) { sm_qs[2 * j] = unit; sm_qs[2 * j + 1] = some ? sum / unit : 0.f; }
    }
    return sm_qs;
}
// query q of the block from its waves' parts: sm_o [W][width][pitch] outputs (mid part added), sm_m [W][width][2] references and sums
template <typename T>
__device__ __forceinline__ void write_query(const attn4_t& a, const work4_t& b, int q, int width, int pitch, const float* sm_o, const float* sm_m, int W, int lane) {
    float M = sm_m[q * 2], L = 0.f, o = 0.f;
    for (int w = 1; w < W; ++w) M = fmaxf(M, sm_m[(w * width + q) * 2]);
    for (int w = 0; w < W; ++w) {
        const float f = __builtin_amdgcn_exp2f(sm_m[(w * width + q) * 2] - M);
        L = __builtin_fmaf(sm_m[(w * width + q) * 2 + 1], f, L);
        o = __builtin_fmaf(sm_o[(w * width + q) * pitch + lane], f, o);
    }
    const int qi = b.q0 + q, g = a.Lq == 1 ? qi : qi / a.Lq, i = qi - g * a.Lq, head = b.hk * b.group + g;
    if (a.splits == 1) {
        static_cast<T*>(a.ctx)[(((int64_t)b.n * a.Lq + i) * a.h + head) * 64 + lane] = from_f32<T>(L == 0.f ? 0.f : o / L);
        if (a.lse && lane == 0) a.lse[((int64_t)b.n * a.h + head) * a.Lq + i] = L == 0.f ? -INFINITY : M + __log2f(L);
    } else {
        float* p = a.part + (((int64_t)b.row * b.group * a.Lq + qi) * a.splits + b.split) * PART;
        p[lane] = o;
        if (lane == 0) { p[64] = M; p[65] = L; }
    }
}

template <typename T, int ND, int NQ, bool CAUSAL>
__global__ __launch_bounds__(MAX_WAVES * 64) void cache4_attn_kernel(attn4_t a) {
    using D = Digits<ND>;
    constexpr int PASSES = (NQ + D::QPP - 1) / D::QPP;
    static_assert(NQ <= MAX_NQ, "the rows of lane group c are query c's digits");
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = a.waves, n16 = lane & 15, c = lane >> 4;
    work4_t b;
    if (!work_of(a, b)) return;
    const u32x4* kc = a.kc + b.base * 2;
    const u32x4* vc = a.vc + b.base * 2;
    const uint32_t* km = a.km + b.base;
    const uint32_t* vm = a.vm + b.base;
    int tile = b.split * W + wave;
    tile4_t cur;
    if (tile * 64 < a.T) load_tile(cur, kc, vc, km, vm, tile * 64, a.T - 1, lane);      // (before the row's length is there: inside the cache either way)
    const int klen = a.k_len ? clampi(a.k_len[b.n], 0, a.T) : a.T, tiles = (klen + 63) >> 6;
    if (b.split > 0 && b.split * W >= tiles) return;      // (the joining launch knows which splits have a tile)

    unsigned char* sm_v = lds + wave * WAVE_LDS;              // 64 rows of 32 bytes, the halves of rows 8 .. 15 of 16 exchanged
    unsigned char* sm_p = sm_v + TILE_V;                    // 64 tokens x 16 bytes: the digits of the weights
    unsigned char* sm_q = lds + W * WAVE_LDS;                 // [NQ][ND][64] digits of the queries
    float* sm_qs = query_digits<T, ND>(a, b, NQ, sm_q, wave, W, lane);
    __syncthreads();
    i32x4 qa[PASSES][2];      // [half]: the first or second 16 of a lane's 32 channels
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int r = n16 & 3, q = D::QPP == 2 ? 2 * p + (r >> 1) : p, d = D::QPP == 2 ? r & 1 : r;
        const bool on = ((n16 >> 2) & 1) == (c >> 1) && q < NQ && d < ND;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const i32x4 v = *reinterpret_cast<const i32x4*>(sm_q + (min(q, NQ - 1) * ND + min(d, ND - 1)) * 64 + (2 * (c & 1) + half) * 16);
            qa[p][half] = on ? v : i32x4{0, 0, 0, 0};
        }
    }
    float unit[NQ], qsum[NQ], m[NQ], l[NQ], mv[NQ], acc[4];
    int lim[NQ];      // first token that the query does not see
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        unit[q] = sm_qs[2 * q]; qsum[q] = sm_qs[2 * q + 1];
        m[q] = NO_REF; l[q] = 0.f; mv[q] = 0.f;
        lim[q] = CAUSAL ? klen - (a.Lq - 1) + (b.q0 + q) % a.Lq : klen;
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) acc[d] = 0.f;

    const int step = a.splits * W;
    for (; tile < tiles; tile += step) {
        const int tok = tile * 64 + lane;
        i32x4 ku[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            ku[j][0] = unpack16(cur.kw[j][0], cur.kw[j][1]);
            ku[j][1] = unpack16(cur.kw[j][2], cur.kw[j][3]);
            const int r = 32 * j + (lane >> 1);
            *reinterpret_cast<u32x4*>(sm_v + r * 32 + (((lane & 1) ^ ((r >> 3) & 1)) << 4)) = cur.vw[j];
        }
        const bool live = tok < klen;      // (what is behind the last token may be anything)
        const uint32_t kmeta = live ? cur.km : 0u, vmeta = live ? cur.vm : 0u;
        const float hide = live ? 0.f : -INFINITY;
        if (tile + step < tiles) load_tile(cur, kc, vc, km, vm, (tile + step) * 64, klen - 1, lane);
        const float ksc = meta_scale(kmeta), kmid = meta_mid(kmeta), vsc = meta_scale(vmeta), vmid = meta_mid(vmeta);
        float s[NQ], e[NQ], top = -INFINITY;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            i32x4 dot[2];      // [j]: rows of the lanes 32 j .. 32 j + 31
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                dot[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[p][0], ku[j][0], i32x4{0, 0, 0, 0}, 0, 0, 0);
                dot[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[p][1], ku[j][1], dot[j], 0, 0, 0);
            }
            const i32x4 d = {lane < 32 ? dot[0][0] : dot[1][0], lane < 32 ? dot[0][1] : dot[1][1], lane < 32 ? dot[0][2] : dot[1][2], lane < 32 ? dot[0][3] : dot[1][3]};
#pragma unroll
            for (int i = 0; i < D::QPP; ++i)
                if (D::QPP * p + i < NQ) s[D::QPP * p + i] = D::QPP == 2 ? D::join(d[2 * i], d[2 * i + 1], 0) : D::join(d[0], d[1], d[2]);
        }
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            s[q] = __builtin_fmaf(s[q], ksc, __builtin_fmaf(kmid, qsum[q], hide));      // in units of unit[q]
            if (CAUSAL) s[q] = tok < lim[q] ? s[q] : -INFINITY;
            e[q] = __builtin_fmaf(s[q], unit[q], -m[q]);
            top = fmaxf(top, e[q]);
        }
        if (__builtin_amdgcn_ballot_w64(top > LAG)) {
            const float big = NQ == 1 ? wave_all<MaxF>(s[0]) : wave_four<MaxF>(s[0], s[NQ > 1 ? 1 : 0], s[NQ > 2 ? 2 : 0], s[NQ > 3 ? 3 : 0]);      // of query c
            float f = 1.f;
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const float mn = __builtin_elementwise_maximum(m[q], __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, big), 16 * q)) * unit[q]);
                const float al = __builtin_amdgcn_exp2f(m[q] - mn);
                m[q] = mn; l[q] *= al; mv[q] *= al;
                e[q] = __builtin_fmaf(s[q], unit[q], -mn);
                f = c == q ? al : f;
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[d] *= f;
        }
        // weights -> digits
        float w[MAX_NQ];
        uint32_t u[MAX_NQ];
#pragma unroll
        for (int q = 0; q < MAX_NQ; ++q) {
            w[q] = 0.f;
            u[q] = 0u;
            if (q >= NQ) continue;
            const float p = __builtin_amdgcn_exp2f(e[q]);
            const bool seen = !CAUSAL || tok < lim[q];      // (0 * NaN of a token that another query sees must not enter the sums)
            l[q] += p;
            mv[q] = __builtin_fmaf(p, seen ? vmid : 0.f, mv[q]);
            w[q] = p * (seen ? vsc : 0.f);
        }
        const float most = NQ == 1 ? wave_all<MaxPos>(w[0]) : wave_four<MaxPos>(w[0], w[1], w[2], w[3]);      // of query c
        // (UNIT / most has to be finite: weights below 1e-30 of a reference that is within 2^LAG of the largest probability count as 0)
        const float inv = most > 1e-30f ? D::UNIT * __builtin_amdgcn_rcpf(most) : 0.f, wunit = most * (1.f / (16.f * D::UNIT));
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const float iq = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, inv), 16 * q));
            if (ND == 2) u[q] = __builtin_bit_cast(uint32_t, __builtin_fmaf(w[q], iq, 12582912.f + D::BIAS));      // round to nearest: the integer in the low bits
            else u[q] = (uint32_t)__builtin_fmaf(w[q], iq, D::BIAS + 0.5f);
            u[q] ^= D::BIAS;
        }
        unsigned char* to = sm_p + ((lane & 48) + unpack_pos(n16)) * 16;
        if (NQ == 1) *reinterpret_cast<uint32_t*>(to) = u[0];
        else if (NQ == 2) *reinterpret_cast<u32x2*>(to) = u32x2{u[0], u[1]};
        else *reinterpret_cast<u32x4*>(to) = u32x4{u[0], u[1], u[2], u[3]};
        wave_lds_fence();
        lds_i32x2* from = (lds_i32x2*)((__attribute__((address_space(3))) unsigned char*)sm_p + c * 256 + n16 * 8);
        const i32x2 p0 = __builtin_amdgcn_ds_read_tr8_b64_v2i32(from), p1 = __builtin_amdgcn_ds_read_tr8_b64_v2i32(from + 16);
        const i32x4 pa = {p0[0], p0[1], p1[0], p1[1]};
#pragma unroll
        for (int d = 0; d < 4; ++d) {      // 16 channels: group c of 16 lanes reads rows 16 c .. 16 c + 15, 8 bytes each, transposed on the way
            const i32x2 vt = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2*)((__attribute__((address_space(3))) unsigned char*)sm_v + lane * 32 +
                                                                                  (((d >> 1) ^ ((lane >> 3) & 1)) << 4) + (d & 1) * 8));
            const i32x4 o = __builtin_amdgcn_mfma_i32_16x16x64_i8(pa, unpack16((uint32_t)vt[0], (uint32_t)vt[1]), i32x4{0, 0, 0, 0}, 0, 0, 0);
            acc[d] = __builtin_fmaf(D::join(o[0], o[1], o[2]), wunit, acc[d]);
        }
        wave_lds_fence();
    }

    // join the waves: [W][NQ] references, sums, and outputs (with the mid part added)
    __syncthreads();
    float* sm_o = reinterpret_cast<float*>(lds);      // [W][NQ][64]
    float* sm_m = sm_o + W * NQ * 64;                 // [W][NQ][2]
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const float lw = wave_all<SumF>(l[q]), mw = wave_all<SumF>(mv[q]);
        if (lane == 0) { sm_m[(wave * NQ + q) * 2] = m[q]; sm_m[(wave * NQ + q) * 2 + 1] = lw; }
        if (c == q)
#pragma unroll
            for (int d = 0; d < 4; ++d) sm_o[(wave * NQ + q) * 64 + d * 16 + n16] = acc[d] + mw;
    }
    __syncthreads();
    for (int q = wave; q < b.nq; q += W) write_query<T>(a, b, q, NQ, 64, sm_o, sm_m, W, lane);
}

// Many queries: the same products turned round.  K is the A operand (16 tokens a row, 8 bytes of codes a lane), 16 queries the columns, so a lane
// holds the scores of ONE query for 16 of the tile's 64 tokens - statistics, masks and scales are per lane - and those 16 weights are, as they
// stand, the lane's share of the PV product's B operand: no LDS between the two products.  V is the A operand (ds_read_b64_tr_b4, its rows read
// in the order in which the lane holds the tokens), the output [channel, query].  430 VALU instructions a tile for 16 queries (counted over rows of 313
// tiles) where the kernel above takes 205 for four; the tokens' scales reach the lanes through LDS.  64 rows x 33 causal queries x up to 2011
// slots: 12.7 us; VALU issue fills 6 us of it on the 192 CUs that have a block, the rest is the chain of a tile (QK, maximum, digits, PV).
constexpr int DENSE_NQ = 16;
template <typename T, int ND, bool CAUSAL>
__global__ __launch_bounds__(MAX_WAVES * 64) void cache4_attn_dense_kernel(attn4_t a) {
    using D = Digits<ND>;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = a.waves, n16 = lane & 15, c = lane >> 4;
    work4_t b;
    if (!work_of(a, b)) return;
    const u32x2* kc = reinterpret_cast<const u32x2*>(a.kc + b.base * 2);
    const u32x4* vc = a.vc + b.base * 2;
    const uint32_t* km = a.km + b.base;
    const uint32_t* vm = a.vm + b.base;
    u32x2 kw[4];
    u32x4 vw[2];
    uint32_t kmeta, vmeta;
    const auto load = [&](int t0, int last) {
#pragma unroll
        for (int i = 0; i < 4; ++i) kw[i] = kc[(unsigned)min(t0 + 16 * i + n16, last) * 4u + c];
#pragma unroll
        for (int j = 0; j < 2; ++j) vw[j] = vc[(unsigned)min(t0 + 32 * j + (lane >> 1), last) * 2u + (lane & 1)];
        const unsigned tok = min(t0 + lane, last);
        kmeta = km[tok];
        vmeta = vm[tok];
    };
    int tile = b.split * W + wave;
    if (tile * 64 < a.T) load(tile * 64, a.T - 1);
    const int klen = a.k_len ? clampi(a.k_len[b.n], 0, a.T) : a.T, tiles = (klen + 63) >> 6;
    if (b.split > 0 && b.split * W >= tiles) return;

    unsigned char* sm_v = lds + wave * WAVE_LDS;                            // 64 rows of 32 bytes, the halves of rows 8 .. 15 of 16 exchanged
    f32x2* sm_k2 = reinterpret_cast<f32x2*>(sm_v + TILE_V);               // (scale, mid) of K and of V by token
    f32x2* sm_v2 = sm_k2 + 64;
    unsigned char* sm_q = lds + W * WAVE_LDS;
    float* sm_qs = query_digits<T, ND>(a, b, DENSE_NQ, sm_q, wave, W, lane);
    __syncthreads();
    i32x4 qb[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) qb[d] = *reinterpret_cast<const i32x4*>(sm_q + (n16 * ND + d) * 64 + c * 16);
    const float unit = sm_qs[2 * n16], qsum = sm_qs[2 * n16 + 1];
    const int lim = CAUSAL ? klen - (a.Lq - 1) + (b.q0 + n16) % a.Lq : klen, all_see = CAUSAL ? klen - (a.Lq - 1) : klen;
    float m = NO_REF, l = 0.f, mv = 0.f;
    f32x4 acc[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int step = a.splits * W;
    for (; tile < tiles; tile += step) {
        const int t0 = tile * 64;
        i32x4 ku[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) ku[i] = unpack16(kw[i][0], kw[i][1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = 32 * j + (lane >> 1);
            *reinterpret_cast<u32x4*>(sm_v + r * 32 + (((lane & 1) ^ ((r >> 3) & 1)) << 4)) = vw[j];
        }
        const bool live = t0 + lane < klen;      // (what is behind the last token may be anything)
        if (!live) kmeta = vmeta = 0u;
        sm_k2[lane] = f32x2{meta_scale(kmeta), meta_mid(kmeta)};
        sm_v2[lane] = f32x2{meta_scale(vmeta), meta_mid(vmeta)};
        if (tile + step < tiles) load((tile + step) * 64, klen - 1);
        wave_lds_fence();
        const auto work = [&](auto masked) {
            float s[4][4], e[4][4], top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                i32x4 dot[ND];
#pragma unroll
                for (int d = 0; d < ND; ++d) dot[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(ku[i], qb[d], i32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; r += 2) {      // tokens 16 i + 4 c + r, + 1
                    const f32x4 k2 = *reinterpret_cast<const f32x4*>(sm_k2 + 16 * i + 4 * c + r);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float v = __builtin_fmaf(D::join(dot[0][r + h], dot[1][r + h], dot[ND - 1][r + h]), k2[2 * h], k2[2 * h + 1] * qsum);
                        if (decltype(masked)::value) v = t0 + 16 * i + 4 * c + r + h < lim ? v : -INFINITY;
                        s[i][r + h] = v;
                        e[i][r + h] = __builtin_fmaf(v, unit, -m);
                        top = fmaxf(top, e[i][r + h]);
                    }
                }
            }
            if (__builtin_amdgcn_ballot_w64(top > LAG)) {
                float big = s[0][0];
#pragma unroll
                for (int x = 1; x < 16; ++x) big = __builtin_elementwise_maximum(big, s[x >> 2][x & 3]);
                const float mn = __builtin_elementwise_maximum(m, over_c<MaxF>(big) * unit), al = __builtin_amdgcn_exp2f(m - mn);
                m = mn; l *= al; mv *= al;
#pragma unroll
                for (int d = 0; d < 4; ++d) acc[d] *= al;
#pragma unroll
                for (int x = 0; x < 16; ++x) e[x >> 2][x & 3] = __builtin_fmaf(s[x >> 2][x & 3], unit, -m);
            }
            uint32_t most = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    const f32x4 v2 = *reinterpret_cast<const f32x4*>(sm_v2 + 16 * i + 4 * c + r);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float p = __builtin_amdgcn_exp2f(e[i][r + h]);
                        const bool seen = !decltype(masked)::value || t0 + 16 * i + 4 * c + r + h < lim;      // (0 * NaN of a token that another query sees)
                        l += p;
                        mv = __builtin_fmaf(p, seen ? v2[2 * h + 1] : 0.f, mv);
                        s[i][r + h] = p * (seen ? v2[2 * h] : 0.f);
                        most = max(most, __builtin_bit_cast(uint32_t, s[i][r + h]));
                    }
                }
            const float mo = over_c<MaxPos>(__builtin_bit_cast(float, most));
            const float inv = mo > 1e-30f ? D::UNIT * __builtin_amdgcn_rcpf(mo) : 0.f, wunit = mo * (1.f / (16.f * D::UNIT));
            i32x4 pb[ND];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t u[4];
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    u[r] = ND == 2 ? __builtin_bit_cast(uint32_t, __builtin_fmaf(s[i][r], inv, 12582912.f + D::BIAS)) : (uint32_t)__builtin_fmaf(s[i][r], inv, D::BIAS + 0.5f);
                const uint32_t t01 = __builtin_amdgcn_perm(u[1], u[0], 0x05010400u), t23 = __builtin_amdgcn_perm(u[3], u[2], 0x05010400u);
                pb[0][i] = (int)(__builtin_amdgcn_perm(t23, t01, 0x05040100u) ^ 0x80808080u);
                pb[1][i] = (int)(__builtin_amdgcn_perm(t23, t01, 0x07060302u) ^ (ND == 3 ? 0x80808080u : 0u));
                if (ND == 3) pb[ND - 1][i] = (int)(__builtin_amdgcn_perm(u[1], u[0], 0x0c0c0602u) | __builtin_amdgcn_perm(u[3], u[2], 0x06020c0cu));
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                // lane k of group c reads the row of the token that is element k of the unpacked operand: byte r of word i = token 16 i + 4 c + r
                const int row = 16 * ((n16 & 1) + 2 * (n16 >> 3)) + 4 * c + ((n16 >> 1) & 3);
                const i32x2 vt = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2*)((__attribute__((address_space(3))) unsigned char*)sm_v + row * 32 +
                                                                                      (((d >> 1) ^ ((row >> 3) & 1)) << 4) + (d & 1) * 8));
                const i32x4 va = unpack16((uint32_t)vt[0], (uint32_t)vt[1]);
                i32x4 o[ND];
#pragma unroll
                for (int x = 0; x < ND; ++x) o[x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(va, pb[x], i32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[d][r] = __builtin_fmaf(D::join(o[0][r], o[1][r], o[ND - 1][r]), wunit, acc[d][r]);
            }
        };
        if (t0 + 64 <= all_see) work(std::false_type{});
        else work(std::true_type{});
        wave_lds_fence();
    }

    __syncthreads();
    float* sm_o = reinterpret_cast<float*>(lds);                      // [W][16][DENSE_ROW], 68 floats a row: 16 lanes' 16-byte stores meet no bank twice
    float* sm_m = sm_o + W * DENSE_NQ * DENSE_ROW;                    // [W][16][2]
    l = over_c<SumF>(l);
    mv = over_c<SumF>(mv);
#pragma unroll
    for (int d = 0; d < 4; ++d) *reinterpret_cast<f32x4*>(sm_o + (wave * DENSE_NQ + n16) * DENSE_ROW + 16 * d + 4 * c) = acc[d] + mv;
    if (c == 0) { sm_m[(wave * DENSE_NQ + n16) * 2] = m; sm_m[(wave * DENSE_NQ + n16) * 2 + 1] = l; }
    __syncthreads();
    for (int q = wave; q < b.nq; q += W) write_query<T>(a, b, q, DENSE_NQ, DENSE_ROW, sm_o, sm_m, W, lane);
}

// joins the splits of one query: 8 waves of up to MAX_SPLITS / 8 partial results each, all loads in front
constexpr int MAX_SPLITS = 32, JOIN_WAVES = 8;
template <typename T>
__global__ __launch_bounds__(JOIN_WAVES * 64) void cache4_join_kernel(attn4_t a) {
    __shared__ float sm[JOIN_WAVES][PART];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = a.h / a.h_kv, Q = group * a.Lq;
    const int row = blockIdx.x / Q, qi = blockIdx.x - row * Q, n = row / a.h_kv, hk = row - n * a.h_kv;
    const float* part = a.part + ((int64_t)row * Q + qi) * a.splits * PART;
    constexpr int MINE = MAX_SPLITS / JOIN_WAVES;
    float v[MINE], ms[MINE], ls[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {      // (inside the workspace also where a split had no tile and left nothing: not used below)
        const float* p = part + (int64_t)min(wave + i * JOIN_WAVES, a.splits - 1) * PART;
        v[i] = p[lane]; ms[i] = p[64]; ls[i] = p[65];
    }
    const int klen = a.k_len ? clampi(a.k_len[n], 0, a.T) : a.T, live = clampi(((klen + 63) / 64 + a.waves - 1) / a.waves, 1, a.splits);
    float M = NO_REF, L = 0.f, o = 0.f;
#pragma unroll
    for (int i = 0; i < MINE; ++i) M = wave + i * JOIN_WAVES < live ? fmaxf(M, ms[i]) : M;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        if (wave + i * JOIN_WAVES >= live) continue;
        const float f = __builtin_amdgcn_exp2f(ms[i] - M);
        L = __builtin_fmaf(ls[i], f, L);
        o = __builtin_fmaf(v[i], f, o);
    }
    sm[wave][lane] = o;
    if (lane == 0) { sm[wave][64] = M; sm[wave][65] = L; }
    __syncthreads();
    if (wave) return;
    L = 0.f; o = 0.f;
#pragma unroll
    for (int w = 0; w < JOIN_WAVES; ++w) M = fmaxf(M, sm[w][64]);
#pragma unroll
    for (int w = 0; w < JOIN_WAVES; ++w) {
        const float f = __builtin_amdgcn_exp2f(sm[w][64] - M);
        L = __builtin_fmaf(sm[w][65], f, L);
        o = __builtin_fmaf(sm[w][lane], f, o);
    }
    const int g = qi / a.Lq, head = hk * group + g, i = qi - g * a.Lq;
    static_cast<T*>(a.ctx)[(((int64_t)n * a.Lq + i) * a.h + head) * 64 + lane] = from_f32<T>(L == 0.f ? 0.f : o / L);
    if (a.lse && lane == 0) a.lse[((int64_t)n * a.h + head) * a.Lq + i] = L == 0.f ? -INFINITY : M + __log2f(L);
}

// How a call is cut.  Times in us, bf16, graph replays, keys cold where they do not fit the caches.
//   kernel            the dense one does half the work a query and has the longer chain a tile: from 9 queries a key head up, where there is work
//                     for many waves - 12 tiles of four queries a SIMD, or four blocks a CU.  64 rows x 2011 slots: 33 queries 12.3 against 16.5, 128
//                     queries 20.3 against 33.1, but 16 queries 12.3 against 8.7; 640 rows x 101 slots: 16 queries 10.9 against 12.8, 8 queries 8.9
//                     against 8.1; 8 rows x 20000 slots: 64 queries 18.3 against 26.4, 16 queries 12.4 either way
//   queries a block   up to 4 (16 in the dense kernel), evenly: eight in the first kernel need 184 VGPRs instead of 106 and lose at every size (5
//                     queries x 128 rows x 1000 slots 8.4 against 7.1; three a block 6.9, two 7.8)
//   waves             one per tile of 64 slots up to 8; 4 where more blocks than CUs make a CU take two anyway (300 rows x 2000 slots 12.9 with 8,
//                     11.8 with 4; 230 rows 9.3 and 9.3; 128 rows x 1000 slots 6.0 with 8, 6.1 with 4, 7.8 with 2).  The dense kernel's waves also
//                     share the queries' digits: never fewer for few tiles (640 rows x 101 slots: 11.1 with 4, 12.7 with 2)
//   splits            where a wave would walk more than 4 tiles and there are no more than 128 blocks: as many as fill 256 CUs with a block each,
//                     two tiles a wave at least (16 rows x 100003 slots: 1 split 143, 16 splits 26.0, 32 splits 26.6; 4 rows: 32 splits 11.7, 20
//                     13.5).  Below that the second launch costs more than it gives (20 rows x 777 slots 4.9 against 6.8; 130 rows x 6000 15.1
//                     against 19.6).
struct plan_t { int nq, qtiles, splits, waves; bool dense; };
plan_t attn_plan(int rows, int Q, int T) {
    plan_t p;
    const int tiles = (T + 63) / 64;
    const int64_t fours = (int64_t)rows * ((Q + MAX_NQ - 1) / MAX_NQ);
    p.dense = Q > 8 && (fours * tiles >= 12 * 1024 || fours > 1024);
    const int width = p.dense ? DENSE_NQ : MAX_NQ;
    p.qtiles = (Q + width - 1) / width;
    p.nq = (Q + p.qtiles - 1) / p.qtiles;
    const int64_t blocks = (int64_t)rows * p.qtiles;
    const int most = blocks > 256 ? 4 : MAX_WAVES;
    p.waves = p.dense ? most : 1;
    while (p.waves < most && p.waves < tiles) p.waves *= 2;
    p.splits = 1;
    if (tiles > 32 && blocks <= 128) {
        const int64_t room = 256 / blocks, work = (tiles + 15) / 16, cap = MAX_SPLITS;
        p.splits = (int)(room < work ? (room < cap ? room : cap) : (work < cap ? work : cap));
    }
    return p;
}

template <typename T, int ND> int attn_launch(hipStream_t s, const attn4_t& a, const plan_t& p, bool causal) {
    const int width = p.dense ? DENSE_NQ : p.nq, pitch = p.dense ? DENSE_ROW : 64;
    const size_t work = (size_t)p.waves * WAVE_LDS + width * (ND * 64 + 8), join = (size_t)p.waves * width * (pitch + 2) * 4;
    const size_t lds = work > join ? work : join;
    static_assert(MAX_WAVES * DENSE_NQ * (DENSE_ROW + 2) * 4 <= 40 * 1024 && MAX_WAVES * WAVE_LDS + DENSE_NQ * (ND * 64 + 8) <= 40 * 1024, "a quarter of a CU's 160 KiB");
    const int64_t streams = (int64_t)a.rows * a.splits;
    const dim3 grid((unsigned)(a.qtiles == 1 ? streams : (streams + 7) / 8 * 8 * a.qtiles)), block(p.waves * 64);
#define ASR_C4(...)                                                                                     \
    do {                                                                                                \
        if (causal) hipLaunchKernelGGL((__VA_ARGS__, true>), grid, block, lds, s, a);                   \
        else hipLaunchKernelGGL((__VA_ARGS__, false>), grid, block, lds, s, a);                         \
    } while (0)
    if (p.dense) ASR_C4(cache4_attn_dense_kernel<T, ND);
    else if (p.nq == 1) ASR_C4(cache4_attn_kernel<T, ND, 1);
    else if (p.nq == 2) ASR_C4(cache4_attn_kernel<T, ND, 2);
    else if (p.nq == 3) ASR_C4(cache4_attn_kernel<T, ND, 3);
    else ASR_C4(cache4_attn_kernel<T, ND, 4);
#undef ASR_C4
    ASR_LAUNCH_CHECK("cache4_attention");
    if (a.splits > 1) {
        hipLaunchKernelGGL((cache4_join_kernel<T>), dim3((unsigned)((int64_t)a.rows * (a.h / a.h_kv) * a.Lq)), dim3(JOIN_WAVES * 64), 0, s, a);
        ASR_LAUNCH_CHECK("cache4_attention (join)");
    }
    return 0;
}

// a * b * c <= most, for sizes whose product may pass 64 bits
bool fits(int64_t a, int64_t b, int64_t c, int64_t most) { return a <= most && b <= most / a && c <= most / (a * b); }
constexpr int64_t MAX_BLOCKS = (1 << 24) - 1;      // of 256 threads: a launch holds fewer than 2^32
constexpr int64_t MAX_QUERIES = (1 << 24) - 1;     // (a block each of up to 256 threads, or more queries a block)

int slots_plan(const char* name, int lanes, slots_t& s, int64_t& blocks, int n_kv, int N, int h, int L, int Tmax, const int32_t* pos, int pos_stride,
               const int32_t* n_tok) {
    ASR_REQUIRE(n_kv > 0 && N > 0 && h > 0 && L > 0 && Tmax > 0, ASR_ERR_ARG, "%s: bad sizes (n_kv=%d N=%d h=%d L=%d Tmax=%d)", name, n_kv, N, h, L, Tmax);
    ASR_REQUIRE(Tmax <= CACHE4_MAX_T && L <= CACHE4_MAX_T, ASR_ERR_UNSUPPORTED, "%s: more than 2^24 slots", name);
    ASR_REQUIRE(pos_stride == 0 || pos_stride == 1, ASR_ERR_ARG, "%s: pos_stride is 0 (one position for all rows) or 1", name);
    ASR_REQUIRE(fits(n_kv, N, h, INT32_MAX - 64), ASR_ERR_UNSUPPORTED, "%s: too many rows", name);
    const int64_t rows = (int64_t)n_kv * N * h;
    const int groups_log2 = lanes == 4 ? 6 : 5;      // rows of 64 values side by side in a block of 256 threads
    int lg = 0;
    while (lg < groups_log2 && (1 << lg) < L) ++lg;
    // a group of lanes walks 4 rows: reading back 12 x 32 x 4 x 1000 rows 42.8 us (49.8 with 2, 43.9 with 8), put 54.6 (53.8, 55.7).  It costs the calls
    // of few blocks a chain of loads: 2 x 7 x 4 x 333 f32 rows put 5.4 and read back 4.5 (3.9 and 3.9 with one row each)
    const int rb_log2 = groups_log2 - lg, iter = 4, chunks = (int)((L + ((int64_t)iter << lg) - 1) / ((int64_t)iter << lg));
    blocks = (rows + (1 << rb_log2) - 1) / (1 << rb_log2) * chunks;
    ASR_REQUIRE(blocks <= MAX_BLOCKS, ASR_ERR_UNSUPPORTED, "%s: too many rows", name);
    s = slots_t{pos, n_tok, pos_stride, N, h, L, Tmax, lg, rb_log2, iter, chunks, (int)rows};
    return 0;
}
bool strides_ok(const strides_t& st, int per16) { return st.kv % per16 == 0 && st.n % per16 == 0 && st.head % per16 == 0 && st.tok % per16 == 0; }

}  // namespace

extern "C" int asr_cache4_put(void* stream, const void* x, int x_dtype, int64_t s_kv, int64_t s_n, int64_t s_head, int64_t s_tok, void* codes,
                              void* meta, const int32_t* pos, int pos_stride, const int32_t* n_new, int n_kv, int N, int h, int L, int Tmax) {
    ASR_REQUIRE(x && codes && meta, ASR_ERR_ARG, "cache4_put: null pointer");
    ASR_REQUIRE(x_dtype == ASR_F32 || x_dtype == ASR_BF16, ASR_ERR_ARG, "cache4_put: dtype %d (ASR_F32 or ASR_BF16)", x_dtype);
    slots_t s; int64_t blocks;
    if (const int rc = slots_plan("cache4_put", 4, s, blocks, n_kv, N, h, L, Tmax, pos, pos_stride, n_new)) return rc;
    const strides_t st{s_kv, s_n, s_head, s_tok};
    ASR_REQUIRE(asr_aligned(x, 16) && asr_aligned(codes, 16) && asr_aligned(meta, 4) && strides_ok(st, x_dtype == ASR_F32 ? 4 : 8), ASR_ERR_ALIGN,
                "cache4_put: rows of x start on 16 bytes, codes on 16, meta on 4");
    hipStream_t hs = static_cast<hipStream_t>(stream);
    if (x_dtype == ASR_F32) {
        if (s.rb_log2 == 0) hipLaunchKernelGGL((cache4_put_kernel<float, true>), dim3((unsigned)blocks), dim3(256), 0, hs, static_cast<const float*>(x), st, static_cast<uint32_t*>(codes), static_cast<uint32_t*>(meta), s);
        else hipLaunchKernelGGL((cache4_put_kernel<float, false>), dim3((unsigned)blocks), dim3(256), 0, hs, static_cast<const float*>(x), st, static_cast<uint32_t*>(codes), static_cast<uint32_t*>(meta), s);
    } else {
        if (s.rb_log2 == 0) hipLaunchKernelGGL((cache4_put_kernel<bf16_t, true>), dim3((unsigned)blocks), dim3(256), 0, hs, static_cast<const bf16_t*>(x), st, static_cast<uint32_t*>(codes), static_cast<uint32_t*>(meta), s);
        else hipLaunchKernelGGL((cache4_put_kernel<bf16_t, false>), dim3((unsigned)blocks), dim3(256), 0, hs, static_cast<const bf16_t*>(x), st, static_cast<uint32_t*>(codes), static_cast<uint32_t*>(meta), s);
    }
    ASR_LAUNCH_CHECK("cache4_put");
    return 0;
}

extern "C" int asr_cache4_get(void* stream, const void* codes, const void* meta, void* out, int out_dtype, int64_t s_kv, int64_t s_n, int64_t s_head,
                              int64_t s_tok, const int32_t* pos, int pos_stride, const int32_t* n_tok, int n_kv, int N, int h, int L, int Tmax) {
    ASR_REQUIRE(out && codes && meta, ASR_ERR_ARG, "cache4_get: null pointer");
    ASR_REQUIRE(out_dtype == ASR_F32 || out_dtype == ASR_BF16, ASR_ERR_ARG, "cache4_get: dtype %d (ASR_F32 or ASR_BF16)", out_dtype);
    slots_t s; int64_t blocks;
    if (const int rc = slots_plan("cache4_get", 8, s, blocks, n_kv, N, h, L, Tmax, pos, pos_stride, n_tok)) return rc;
    const strides_t st{s_kv, s_n, s_head, s_tok};
    ASR_REQUIRE(asr_aligned(out, 16) && asr_aligned(codes, 16) && asr_aligned(meta, 4) && strides_ok(st, out_dtype == ASR_F32 ? 4 : 8), ASR_ERR_ALIGN,
                "cache4_get: rows of out start on 16 bytes, codes on 16, meta on 4");
    hipStream_t hs = static_cast<hipStream_t>(stream);
    if (out_dtype == ASR_F32) {
        if (s.rb_log2 == 0) hipLaunchKernelGGL((cache4_get_kernel<float, true>), dim3((unsigned)blocks), dim3(256), 0, hs, static_cast<float*>(out), st, static_cast<const uint32_t*>(codes), static_cast<const uint32_t*>(meta), s);
        else hipLaunchKernelGGL((cache4_get_kernel<float, false>), dim3((unsigned)blocks), dim3(256), 0, hs, static_cast<float*>(out), st, static_cast<const uint32_t*>(codes), static_cast<const uint32_t*>(meta), s);
    } else {
        if (s.rb_log2 == 0) hipLaunchKernelGGL((cache4_get_kernel<bf16_t, true>), dim3((unsigned)blocks), dim3(256), 0, hs, static_cast<bf16_t*>(out), st, static_cast<const uint32_t*>(codes), static_cast<const uint32_t*>(meta), s);
        else hipLaunchKernelGGL((cache4_get_kernel<bf16_t, false>), dim3((unsigned)blocks), dim3(256), 0, hs, static_cast<bf16_t*>(out), st, static_cast<const uint32_t*>(codes), static_cast<const uint32_t*>(meta), s);
    }
    ASR_LAUNCH_CHECK("cache4_get");
    return 0;
}

extern "C" int asr_cache4_reorder(void* stream, const void* codes, const void* meta, void* out_codes, void* out_meta, const int64_t* parent,
                                  const int32_t* state, int n_kv, int B, int beam, int h, int Tmax) {
    ASR_REQUIRE(codes && meta && out_codes && out_meta && parent && state && n_kv > 0 && B > 0 && h > 0 && Tmax > 0, ASR_ERR_ARG, "cache4_reorder: bad args");
    ASR_REQUIRE(beam >= 1 && beam <= 8, ASR_ERR_UNSUPPORTED, "cache4_reorder: beam_size %d (at most 8)", beam);
    ASR_REQUIRE(Tmax <= CACHE4_MAX_T, ASR_ERR_UNSUPPORTED, "cache4_reorder: more than 2^24 slots");
    ASR_REQUIRE((codes == out_codes) == (meta == out_meta), ASR_ERR_ARG, "cache4_reorder: in place means codes and meta both");
    ASR_REQUIRE(asr_aligned(codes, 16) && asr_aligned(out_codes, 16) && asr_aligned(meta, 4) && asr_aligned(out_meta, 4), ASR_ERR_ALIGN, "cache4_reorder: alignment");
    const int chunks_codes = (2 * Tmax + 255) / 256, chunks_meta = (Tmax + 255) / 256;
    ASR_REQUIRE(fits(n_kv, B, h, MAX_BLOCKS / (chunks_codes + chunks_meta)), ASR_ERR_UNSUPPORTED, "cache4_reorder: too many rows");
    const int blocks = n_kv * B * h * (chunks_codes + chunks_meta);
    hipStream_t hs = static_cast<hipStream_t>(stream);
#define ASR_C4(BEAM)                                                                                                                                     \
    hipLaunchKernelGGL((cache4_reorder_kernel<BEAM>), dim3((unsigned)blocks), dim3(256), 0, hs, static_cast<const u32x4*>(codes), static_cast<const uint32_t*>(meta), \
                       static_cast<u32x4*>(out_codes), static_cast<uint32_t*>(out_meta), parent, state, B, beam, h, Tmax, chunks_codes, chunks_meta, codes == out_codes)
    if (beam <= 2) ASR_C4(2);
    else if (beam <= 4) ASR_C4(4);
    else ASR_C4(8);
#undef ASR_C4
    ASR_LAUNCH_CHECK("cache4_reorder");
    return 0;
}

extern "C" int64_t asr_cache4_attention_workspace_bytes(int N, int h, int h_kv, int Lq, int T) {
    if (N <= 0 || h_kv <= 0 || h <= 0 || h % h_kv || Lq <= 0 || T <= 0 || T > CACHE4_MAX_T || !fits(N, h, Lq, MAX_QUERIES)) return 0;      // (no call that is taken)
    const plan_t p = attn_plan(N * h_kv, h / h_kv * Lq, T);
    return p.splits == 1 ? 0 : (int64_t)N * h * Lq * p.splits * PART * 4;
}

extern "C" int asr_cache4_attention(void* stream, const void* q, int dtype, int64_t s_n, int64_t s_head, int64_t s_tok, const void* k_codes,
                                    const void* k_meta, const void* v_codes, const void* v_meta, void* ctx, float* lse, int N, int h, int h_kv, int Lq,
                                    int T, const int32_t* k_len, int causal, void* workspace, int64_t workspace_bytes) {
    ASR_REQUIRE(q && k_codes && k_meta && v_codes && v_meta && ctx, ASR_ERR_ARG, "cache4_attention: null pointer");
    ASR_REQUIRE(dtype == ASR_F32 || dtype == ASR_BF16, ASR_ERR_ARG, "cache4_attention: dtype %d (ASR_F32 or ASR_BF16)", dtype);
    ASR_REQUIRE(N > 0 && h > 0 && h_kv > 0 && Lq > 0 && T > 0 && h % h_kv == 0, ASR_ERR_ARG, "cache4_attention: bad sizes (N=%d h=%d h_kv=%d Lq=%d T=%d)", N, h, h_kv, Lq, T);
    ASR_REQUIRE(T <= CACHE4_MAX_T, ASR_ERR_UNSUPPORTED, "cache4_attention: more than 2^24 slots");
    ASR_REQUIRE(fits(N, h, Lq, MAX_QUERIES), ASR_ERR_UNSUPPORTED, "cache4_attention: more than 2^24 queries");
    ASR_REQUIRE(asr_aligned(q, dtype == ASR_F32 ? 4 : 2) && asr_aligned(ctx, dtype == ASR_F32 ? 4 : 2) && asr_aligned(k_codes, 16) && asr_aligned(v_codes, 16) && asr_aligned(k_meta, 4) && asr_aligned(v_meta, 4),
                ASR_ERR_ALIGN, "cache4_attention: codes start on 16 bytes, meta on 4, q and ctx on their elements");
    const plan_t p = attn_plan(N * h_kv, h / h_kv * Lq, T);
    const int64_t need = p.splits == 1 ? 0 : (int64_t)N * h * Lq * p.splits * PART * 4;
    ASR_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && asr_aligned(workspace, 4)), ASR_ERR_ARG, "cache4_attention: workspace of %lld bytes needed, %lld given",
                (long long)need, (long long)(workspace ? workspace_bytes : 0));
    attn4_t a{q, s_n, s_head, s_tok, static_cast<const u32x4*>(k_codes), static_cast<const uint32_t*>(k_meta), static_cast<const u32x4*>(v_codes),
              static_cast<const uint32_t*>(v_meta), ctx, lse, static_cast<float*>(workspace), k_len, h, h_kv, Lq, T, p.splits, p.qtiles, p.nq,
              N * h_kv, p.waves};
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == ASR_BF16 ? attn_launch<bf16_t, 2>(s, a, p, causal != 0) : attn_launch<float, 3>(s, a, p, causal != 0);
}
