// K / V cache held in 4 bits: quantising put, reading back, attention over it, re-gathering by parent hypothesis (asr_hip.h: asr_cache4_*).
//
// A row of 64 values (one head of one token) is 32 bytes of signed codes - byte j: value 2j in the low nibble, 2j + 1 in the high one - and
// one 32-bit word, the bf16 pair (scale low, mid high): value = mid + scale * code.  scale = bf16((max - min) / 15) and mid = bf16(min + 8
// scale) put min at code -8 and max at 7 with half a step of room on either side, which is what the two bf16 roundings may use up (mid's is
// half a step only where |mid| > 256 scale: rows whose level is 17 times their spread).
#include "asr_common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(2))) int i32x2;

constexpr int CACHE4_MAX_T = 1 << 24;      // slots of a row: 32-bit offsets inside a row (32 bytes a slot), 64-bit ones in front of it

__device__ __forceinline__ uint32_t bf16_bits(float x) { return (uint32_t)__builtin_bit_cast(uint16_t, (bf16_t)x); }
__device__ __forceinline__ float meta_scale(uint32_t m) { return __builtin_bit_cast(float, m << 16); }
__device__ __forceinline__ float meta_mid(uint32_t m) { return __builtin_bit_cast(float, m & 0xffff0000u); }
__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// ---- 8 consecutive values of a row ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ void load8(const bf16_t* p, float (&v)[8]) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = meta_scale(w[i]); v[2 * i + 1] = meta_mid(w[i]); }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
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

// lane exchange inside groups of 8 lanes: xor 1, xor 2 (quad_perm), then the mirror image in the half row (the quads hold one value each by then)
template <int CTRL> __device__ __forceinline__ float dpp_f(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int CTRL> __device__ __forceinline__ void minmax_step(float& lo, float& hi, float& bad) {
    lo = fminf(lo, dpp_f<CTRL>(lo));
    hi = fmaxf(hi, dpp_f<CTRL>(hi));
    bad += dpp_f<CTRL>(bad);
}

// The codes of 8 values of a row whose 64 values lie in 8 neighbouring lanes: -> the 32-bit word of nibbles, and the row's (scale, mid).
// Every decision is that of (x - mid) / scale computed exactly.  The quick form (one subtraction, one multiplication by the reciprocal) is
// off by at most 2^-18 for quotients up to 8; only where it comes within 2^-16 of a border is the exact residual looked at.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t& meta) {
#pragma clang fp contract(off)
    float lo = x[0], hi = x[0], bad = 0.f;      // bad: 0, or NaN where a value is not finite
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        bad = __builtin_fmaf(x[i], 0.f, bad);
    }
    minmax_step<0xB1>(lo, hi, bad);
    minmax_step<0x4E>(lo, hi, bad);
    minmax_step<0x141>(lo, hi, bad);
    const float span = (hi - lo) + bad;
    if (!(span < INFINITY)) {
        meta = 0x7fc07fc0u;
        return 0u;
    }
    const float sc = span < 0x1p-100f ? 0.f : (float)(bf16_t)(span / 15.f);
    const float mid = (float)(bf16_t)(lo + 8.f * sc);
    meta = bf16_bits(sc) | (bf16_bits(mid) << 16);
    if (sc == 0.f) return 0u;
    const float rs = __builtin_amdgcn_rcpf(sc);
    float k[8], near = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = (x[i] - mid) * rs;
        k[i] = __builtin_rintf(y);
        near = fmaxf(near, fabsf(y - k[i]));
    }
    if (near > 0.5f - 0x1p-16f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = x[i] - mid, bb = d - x[i], e = (x[i] - (d - bb)) + (-mid - bb);      // d + e = x - mid exactly
            const float r = __builtin_fmaf(-k[i], sc, d);                                        // exact: k sc has 12 bits
            const float g = (fabsf(r) - 0.5f * sc) + (r > 0.f ? e : -e);                         // > 0: the neighbour is nearer
            if (g > 0.f || (g == 0.f && ((int)k[i] & 1))) k[i] += r > 0.f ? 1.f : -1.f;
        }
    }
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= (uint32_t)(int)(__builtin_amdgcn_fmed3f(k[i], -8.f, 7.f) + 8.f) << (4 * i);
    return w ^ 0x88888888u;      // offset code -> two's complement nibble
}

// Slots of one call: which rows a block works on.  A block is 32 groups of 8 lanes; `tb` (a power of two) tokens of 32 / tb rows side by
// side, so that a single token per row fills a block as well as a long chunk does; a long chunk's block walks ITER * tb tokens.
constexpr int ITER = 4;
struct slots_t {
    const int32_t* pos; const int32_t* n_tok;
    int pos_stride, N, h, L, Tmax, tb, tb_log2, chunks, rows;
};
struct strides_t { int64_t kv, n, head, tok; };

template <typename F> __device__ __forceinline__ void for_tokens(const slots_t& s, const strides_t& st, F f) {
    const int chunk = blockIdx.x % s.chunks, group = threadIdx.x >> 3;
    const int row = (int)(blockIdx.x / s.chunks) * (32 >> s.tb_log2) + (group >> s.tb_log2);
    if (row >= s.rows) return;
    const int head = row % s.h, kn = row / s.h, n = kn % s.N, kv = kn / s.N;
    const int first = s.pos ? s.pos[(int64_t)n * s.pos_stride] : 0;
    const int count = s.n_tok ? clampi(s.n_tok[n], 0, s.L) : s.L;
    const int64_t x0 = kv * st.kv + n * st.n + head * st.head;
    const int64_t c0 = (int64_t)row * s.Tmax;
    const int t0 = chunk * (s.tb * ITER) + (group & (s.tb - 1));
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
        const int i = t0 + it * s.tb;
        if (i < s.L) f(i, count, first, x0 + (int64_t)i * st.tok, c0);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void cache4_put_kernel(const T* __restrict__ x, strides_t st, uint32_t* __restrict__ codes,
                                                         uint32_t* __restrict__ meta, slots_t s) {
    const int l8 = threadIdx.x & 7;
    for_tokens(s, st, [&](int i, int count, int first, int64_t xo, int64_t c0) {
        const int64_t slot = (int64_t)first + i;
        if (i >= count || slot < 0 || slot >= s.Tmax) return;      // (one token's 8 lanes agree)
        float v[8];
        load8(x + xo + l8 * 8, v);
        uint32_t m;
        const uint32_t w = quantise8(v, m);
        codes[(c0 + slot) * 8 + l8] = w;
        if (l8 == 0) meta[c0 + slot] = m;
    });
}

template <typename T>
__global__ __launch_bounds__(256) void cache4_get_kernel(T* __restrict__ out, strides_t st, const uint32_t* __restrict__ codes,
                                                         const uint32_t* __restrict__ meta, slots_t s) {
    const int l8 = threadIdx.x & 7;
    for_tokens(s, st, [&](int i, int count, int first, int64_t xo, int64_t c0) {
        const int64_t slot = (int64_t)first + i;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (i < count && slot >= 0 && slot < s.Tmax) {
            const uint32_t w = codes[(c0 + slot) * 8 + l8], m = meta[c0 + slot];
            const float sc = meta_scale(m), mid = meta_mid(m);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __builtin_fmaf(sc, (float)((int)(w << (28 - 4 * j)) >> 28), mid);      // one rounding: sc * code is exact
        }
        store8(out + xo + l8 * 8, v);
    });
}

// ---- re-gathering by parent ------------------------------------------------------------------------------------------------------------
// A group is one (kv, utterance, head); a thread owns one piece of one position (a 16-byte half of its codes, or its meta word) for all
// `beam` rows: it reads every source row's piece before it writes any, so source and destination may be the same cache.
template <typename V> __device__ __forceinline__ void regather(const V* src, V* dst, const int (&from)[8], int64_t row_stride, int beam, bool in_place) {
    V v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r)
        if (r < beam && !(in_place && from[r] == r)) v[r] = src[(int64_t)from[r] * row_stride];
#pragma unroll
    for (int r = 0; r < 8; ++r)
        if (r < beam && !(in_place && from[r] == r)) dst[(int64_t)r * row_stride] = v[r];
}

__global__ __launch_bounds__(256) void cache4_reorder_kernel(const u32x4* codes, const uint32_t* meta, u32x4* out_codes, uint32_t* out_meta,
                                                             const int64_t* __restrict__ parent, const int32_t* __restrict__ state, int B,
                                                             int beam, int h, int Tmax, int chunks, bool in_place) {
    const int n = clampi(state[0] + 1, 0, Tmax);
    const int u = (int)(blockIdx.x % chunks) * 256 + threadIdx.x;
    if (u >= 3 * n) return;
    const int grp = blockIdx.x / chunks, hd = grp % h, kb = grp / h, b = kb % B, kv = kb / B;
    int from[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) from[r] = r < beam ? clampi((int)(parent[(int64_t)b * beam + r] - (int64_t)b * beam), 0, beam - 1) : 0;
    const int64_t row0 = (((int64_t)kv * B + b) * beam * h + hd) * Tmax;      // slots in front of the group's first row
    if (u < 2 * n) regather(codes + row0 * 2 + u, out_codes + row0 * 2 + u, from, (int64_t)h * Tmax * 2, beam, in_place);
    else regather(meta + row0 + (u - 2 * n), out_meta + row0 + (u - 2 * n), from, (int64_t)h * Tmax, beam, in_place);
}

// ---- attention ---------------------------------------------------------------------------------------------------------------------------
// With k_j = mid_j + scale_j c_j and v_j = mid'_j + scale'_j c'_j:
//     s_j = scale_j (q . c_j) + mid_j sum(q)           p_j = 2^(s_j - m)
//     o   = (sum_j p_j mid'_j + sum_j (p_j scale'_j) c'_j) / sum_j p_j
// Both products run over the codes themselves, on the int8 matrix instruction: a nibble masked in place is the byte 16 c, three VALU
// operations for eight codes, and no value of the cache is ever widened.  The other operand is cut into int8 digits of base 128: the query
// once per launch (relative to its largest element), the weights w_j = p_j scale'_j once per tile of 64 tokens (relative to the tile's
// largest, so a tile of small weights keeps its precision).  ND = 2 digits for bf16 queries (a step of 2^-14 of the largest, below the 2^-9
// that a bf16 weight is rounded by), 3 for f32 (2^-21).  The products are exact int32; softmax statistics and the output are f32.
//
// A wave owns 64 tokens at a time, token = lane: the query operand of each of a tile's four QK instructions is zero except in the four rows
// whose results land in the sixteen lanes of the right tokens, so one accumulator collects 64 tokens x (2 queries x 2 digits, or 1 x 3).
// The weights go through LDS (one byte per lane, query and digit) into the A operand of the PV product, whose rows are (query, digit) and
// whose B operand - 16 tokens of one channel per lane - is what ds_read_b64_tr_b4 makes of the tile's row-major codes.
// The running reference m of a query is renewed only when a score passes it by 2^32 (weights are f32 and scaled per tile: nothing needs
// them below 1), so a tile costs one reduction across the wave per query, the largest weight's.
template <int ND> struct Digits {
    static constexpr float UNIT = ND == 2 ? 127.f * 128.f : 127.f * 16384.f;      // the integer that the largest element becomes
    static constexpr int QPP = ND == 2 ? 2 : 1;                                   // queries per accumulator
    // digit `d` (0 = highest) of |u| <= UNIT
    static __device__ __forceinline__ int get(int u, int d) {
        if (ND == 2) return d == 0 ? (u + 64) >> 7 : (u << 25) >> 25;
        const int r = (u << 18) >> 18;
        return d == 0 ? (u + 8192) >> 14 : d == 1 ? (r + 64) >> 7 : (r << 25) >> 25;
    }
    static __device__ __forceinline__ float join(int a, int b, int c) {
        return ND == 2 ? (float)((a << 7) + b) : __builtin_fmaf((float)a, 16384.f, (float)((b << 7) + c));
    }
};

struct attn4_t {
    const void* q; int64_t q_n, q_head, q_tok;
    const u32x4* kc; const uint32_t* km; const u32x4* vc; const uint32_t* vm;
    void* ctx; float* lse; float* part;
    const int32_t* k_len;
    int N, h, h_kv, Lq, T, causal, splits, qtiles, rows, waves;
};
constexpr int PART = 66;      // floats of a partial result: 64 outputs (not divided), reference, sum

// position of element k of 16 in the byte order that unpacking leaves: low nibbles of the first word, its high ones, then the second word's
__device__ __forceinline__ int unpack_pos(int k) { return (k & 8) + (k & 1) * 4 + ((k >> 1) & 3); }
__device__ __forceinline__ i32x4 unpack16(uint32_t w0, uint32_t w1) {
    return i32x4{(int)((w0 << 4) & 0xf0f0f0f0u), (int)(w0 & 0xf0f0f0f0u), (int)((w1 << 4) & 0xf0f0f0f0u), (int)(w1 & 0xf0f0f0f0u)};
}
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp_umax(uint32_t x) {
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false));
}
// largest of 64 non-negative floats (as their bit patterns), the same for all lanes
__device__ __forceinline__ float wave_max_pos(float v) {
    uint32_t x = __builtin_bit_cast(uint32_t, v);
    x = dpp_umax<0x121, 0xf>(x);      // row_ror 1, 2, 4, 8: every lane has its row's
    x = dpp_umax<0x122, 0xf>(x);
    x = dpp_umax<0x124, 0xf>(x);
    x = dpp_umax<0x128, 0xf>(x);
    x = dpp_umax<0x142, 0xa>(x);      // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3
    x = dpp_umax<0x143, 0xc>(x);
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane((int)x, 63));
}
__device__ __forceinline__ void wave_lds_fence() {      // LDS written by other lanes of this wave
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

template <typename T, int ND, int NQ>
__global__ __launch_bounds__(512) void cache4_attn_kernel(attn4_t a) {
    using D = Digits<ND>;
    constexpr int PASSES = (NQ + D::QPP - 1) / D::QPP, SLOTS = NQ > 4 ? 2 : 1;
    static_assert(ND == 2 ? NQ <= 8 : NQ <= 4, "16 rows of (query, digit)");
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, W = a.waves, n16 = lane & 15, c = lane >> 4;
    // block -> (row, query tile, split): the query tiles of one stream of keys follow each other at a distance of 8 blocks (one XCD's L2)
    const int per8 = 8 * a.qtiles, oct = blockIdx.x / per8, rest = blockIdx.x % per8;
    const int stream = oct * 8 + (rest & 7), qt = rest >> 3;
    if (stream >= a.rows * a.splits) return;
    const int row = stream / a.splits, split = stream % a.splits, n = row / a.h_kv, hk = row % a.h_kv;
    const int klen = a.k_len ? clampi(a.k_len[n], 0, a.T) : a.T, tiles = (klen + 63) >> 6;
    if (split > 0 && split >= tiles) return;      // (the joining launch knows which splits have a tile)
    const int group = a.h / a.h_kv, Q = group * a.Lq, q0 = qt * NQ, nq = min(NQ, Q - q0);

    unsigned char* sm_v = lds + wave * 3072;              // 64 rows of 32 bytes, the halves of rows 8 .. 15 of 16 exchanged
    unsigned char* sm_p = sm_v + 2048;                    // 16 rows (query, digit) of 64 token bytes
    unsigned char* sm_q = lds + W * 3072;                 // [NQ][ND][64] digits of the queries
    float* sm_qs = reinterpret_cast<float*>(sm_q + NQ * ND * 64);      // [NQ][2]: unit of the digits (with the codes' 16), sum
    for (int j = wave; j < NQ; j += W) {
        float v = 0.f;
        if (j < nq) {
            const int qi = q0 + j, head = hk * group + qi / a.Lq, i = qi % a.Lq;
            v = to_f32(static_cast<const T*>(a.q)[n * a.q_n + head * a.q_head + i * a.q_tok + lane]);
        }
        const float top = wave_max(fabsf(v)), sum = wave_sum(v);
        const int u = top > 0.f ? (int)__builtin_rintf(v * (D::UNIT / top)) : 0;
#pragma unroll
        for (int d = 0; d < ND; ++d) sm_q[(j * ND + d) * 64 + (lane & 48) + unpack_pos(n16)] = (unsigned char)D::get(u, d);
        if (lane == 0) { sm_qs[2 * j] = top * (1.f / (16.f * D::UNIT)); sm_qs[2 * j + 1] = sum; }
    }
    __syncthreads();
    i32x4 qa[PASSES][2][2];      // [j]: tokens 32 j .. 32 j + 31 of the tile, [half]: the first or second 16 of a lane's 32 channels
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int r = n16 & 3, q = D::QPP == 2 ? 2 * p + (r >> 1) : p, d = D::QPP == 2 ? r & 1 : r;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const bool on = (n16 >> 2) == 2 * j + (c >> 1) && q < NQ && d < ND;
                const i32x4 v = *reinterpret_cast<const i32x4*>(sm_q + (min(q, NQ - 1) * ND + min(d, ND - 1)) * 64 + (2 * (c & 1) + half) * 16);
                qa[p][j][half] = on ? v : i32x4{0, 0, 0, 0};
            }
    }
    float unit[NQ], qsum[NQ], m[NQ], l[NQ], mv[NQ], acc[4][SLOTS];
    int lim[NQ];      // first token that the query does not see
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        unit[q] = sm_qs[2 * q]; qsum[q] = sm_qs[2 * q + 1];
        m[q] = -3.4028234663852886e38f; l[q] = 0.f; mv[q] = 0.f;
        lim[q] = a.causal ? klen - (a.Lq - 1) + (q0 + q) % a.Lq : klen;
    }
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) acc[d][s] = 0.f;

    const int64_t base = (int64_t)row * a.T;
    const u32x4* kc = a.kc + base * 2;
    const u32x4* vc = a.vc + base * 2;
    const uint32_t* km = a.km + base;
    const uint32_t* vm = a.vm + base;
    for (int tile = split + wave * a.splits; tile < tiles; tile += a.splits * W) {
        const int t0 = tile * 64, last = klen - 1;
        u32x4 kw[2], vw[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {      // (tokens behind the last are read as the last one: their scores are masked below)
            kw[j] = kc[(unsigned)min(t0 + 32 * j + 16 * (c >> 1) + n16, last) * 2u + (c & 1)];
            vw[j] = vc[(unsigned)min(t0 + 32 * j + (lane >> 1), last) * 2u + (lane & 1)];
        }
        const int tok = t0 + lane;
        const uint32_t kmeta = km[min(tok, last)];
        uint32_t vmeta = vm[min(tok, last)];
        if (tok >= klen) vmeta = 0u;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = 32 * j + (lane >> 1);
            *reinterpret_cast<u32x4*>(sm_v + r * 32 + (((lane & 1) ^ ((r >> 3) & 1)) << 4)) = vw[j];
        }
        // scores
        i32x4 ku[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) { ku[j][0] = unpack16(kw[j][0], kw[j][1]); ku[j][1] = unpack16(kw[j][2], kw[j][3]); }
        const float ksc = meta_scale(kmeta), kmid = meta_mid(kmeta), vsc = meta_scale(vmeta), vmid = meta_mid(vmeta);
        float s[NQ];
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            i32x4 dot = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int half = 0; half < 2; ++half) dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[p][j][half], ku[j][half], dot, 0, 0, 0);
            if (D::QPP == 2) {
                s[2 * p] = D::join(dot[0], dot[1], 0);
                if (2 * p + 1 < NQ) s[2 * p + 1] = D::join(dot[2], dot[3], 0);
            } else {
                s[p] = D::join(dot[0], dot[1], dot[2]);
            }
        }
        bool up = false;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            s[q] = __builtin_fmaf(s[q] * unit[q], ksc, kmid * qsum[q]);
            s[q] = tok < lim[q] ? s[q] : -INFINITY;
            up = up || s[q] > m[q] + 32.f;
        }
        if (__builtin_amdgcn_ballot_w64(up)) {
            float al[NQ];
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const float mn = fmaxf(m[q], wave_max(s[q]));
                al[q] = __builtin_amdgcn_exp2f(m[q] - mn);
                m[q] = mn; l[q] *= al[q]; mv[q] *= al[q];
            }
#pragma unroll
            for (int sl = 0; sl < SLOTS; ++sl) {
                float f = 1.f;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (4 * sl + q < NQ && c == q) f = al[4 * sl + q < NQ ? 4 * sl + q : 0];
#pragma unroll
                for (int d = 0; d < 4; ++d) acc[d][sl] *= f;
            }
        }
        // weights -> digits
        float wunit[SLOTS];
#pragma unroll
        for (int sl = 0; sl < SLOTS; ++sl) wunit[sl] = 0.f;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const float p = __builtin_amdgcn_exp2f(s[q] - m[q]);
            const bool seen = tok < lim[q];      // (a masked token may hold anything: 0 * NaN must not enter the sums)
            l[q] += p;
            mv[q] = __builtin_fmaf(p, seen ? vmid : 0.f, mv[q]);
            const float w = p * (seen ? vsc : 0.f);
            const float top = wave_max_pos(w);
            const float inv = top > 1e-30f ? D::UNIT * __builtin_amdgcn_rcpf(top) : 0.f;
            const int u = __builtin_bit_cast(int, __builtin_fmaf(w, inv, 12582912.f));      // round to nearest: the integer in the low 22 bits
            const int prow = 4 * (q & 3) + (ND == 2 ? 2 * (q >> 2) : 0);
#pragma unroll
            for (int d = 0; d < ND; ++d) sm_p[(prow + d) * 64 + (lane & 48) + unpack_pos(n16)] = (unsigned char)D::get(u, d);
            if (c == (q & 3)) wunit[q >> 2] = top * (1.f / (16.f * D::UNIT));
        }
        wave_lds_fence();
        const i32x4 pa = *reinterpret_cast<const i32x4*>(sm_p + n16 * 64 + c * 16);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const int r = lane;      // group c of 16 lanes: rows 16 c .. 16 c + 15, 8 bytes (16 channels) each, transposed on the way
            const i32x2 w = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i32x2*)(
                (__attribute__((address_space(3))) unsigned char*)sm_v + r * 32 + (((d >> 1) ^ ((r >> 3) & 1)) << 4) + (d & 1) * 8));
            const i32x4 o = __builtin_amdgcn_mfma_i32_16x16x64_i8(pa, unpack16((uint32_t)w[0], (uint32_t)w[1]), i32x4{0, 0, 0, 0}, 0, 0, 0);
            acc[d][0] = __builtin_fmaf(D::join(o[0], o[1], o[2]), wunit[0], acc[d][0]);
            if (SLOTS == 2) acc[d][1] = __builtin_fmaf(D::join(o[2], o[3], 0), wunit[SLOTS - 1], acc[d][SLOTS - 1]);
        }
        wave_lds_fence();
    }

    // join the waves: [W][NQ] references, sums, and outputs (with the mid part added)
    __syncthreads();
    float* sm_o = reinterpret_cast<float*>(lds);      // [W][NQ][64]
    float* sm_m = sm_o + W * NQ * 64;                 // [W][NQ][2]
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const float lw = wave_sum(l[q]), mw = wave_sum(mv[q]);
        if (lane == 0) { sm_m[(wave * NQ + q) * 2] = m[q]; sm_m[(wave * NQ + q) * 2 + 1] = lw; }
        if (c == (q & 3))
#pragma unroll
            for (int d = 0; d < 4; ++d) sm_o[(wave * NQ + q) * 64 + d * 16 + n16] = acc[d][q >> 2] + mw;
    }
    __syncthreads();
    for (int q = wave; q < nq; q += W) {
        float M = sm_m[q * 2], L = 0.f, o = 0.f;
        for (int w = 1; w < W; ++w) M = fmaxf(M, sm_m[(w * NQ + q) * 2]);
        for (int w = 0; w < W; ++w) {
            const float f = __builtin_amdgcn_exp2f(sm_m[(w * NQ + q) * 2] - M);
            L = __builtin_fmaf(sm_m[(w * NQ + q) * 2 + 1], f, L);
            o = __builtin_fmaf(sm_o[(w * NQ + q) * 64 + lane], f, o);
        }
        const int qi = q0 + q, head = hk * group + qi / a.Lq, i = qi % a.Lq;
        if (a.splits == 1) {
            static_cast<T*>(a.ctx)[(((int64_t)n * a.Lq + i) * a.h + head) * 64 + lane] = from_f32<T>(L == 0.f ? 0.f : o / L);
            if (a.lse && lane == 0) a.lse[((int64_t)n * a.h + head) * a.Lq + i] = L == 0.f ? -INFINITY : M + __log2f(L);
        } else {
            float* p = a.part + (((int64_t)row * Q + qi) * a.splits + split) * PART;
            p[lane] = o;
            if (lane == 0) { p[64] = M; p[65] = L; }
        }
    }
}

// joins the splits of one query: 4 waves take every fourth partial result
template <typename T>
__global__ __launch_bounds__(256) void cache4_join_kernel(attn4_t a) {
    __shared__ float sm[4][PART];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = a.h / a.h_kv, Q = group * a.Lq;
    const int row = blockIdx.x / Q, qi = blockIdx.x % Q, n = row / a.h_kv, hk = row % a.h_kv;
    const int klen = a.k_len ? clampi(a.k_len[n], 0, a.T) : a.T, live = max(1, min(a.splits, (klen + 63) >> 6));
    const float* part = a.part + ((int64_t)row * Q + qi) * a.splits * PART;
    float M = -3.4028234663852886e38f, L = 0.f, o = 0.f;
    for (int s = wave; s < live; s += 4) {
        const float* p = part + (int64_t)s * PART;
        const float v = p[lane], ms = p[64], ls = p[65], mn = fmaxf(M, ms);
        const float f0 = __builtin_amdgcn_exp2f(M - mn), f1 = __builtin_amdgcn_exp2f(ms - mn);
        L = __builtin_fmaf(ls, f1, L * f0);
        o = __builtin_fmaf(v, f1, o * f0);
        M = mn;
    }
    sm[wave][lane] = o;
    if (lane == 0) { sm[wave][64] = M; sm[wave][65] = L; }
    __syncthreads();
    if (wave) return;
    M = fmaxf(fmaxf(sm[0][64], sm[1][64]), fmaxf(sm[2][64], sm[3][64]));
    L = 0.f; o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(sm[w][64] - M);
        L = __builtin_fmaf(sm[w][65], f, L);
        o = __builtin_fmaf(sm[w][lane], f, o);
    }
    const int head = hk * group + qi / a.Lq, i = qi % a.Lq;
    static_cast<T*>(a.ctx)[(((int64_t)n * a.Lq + i) * a.h + head) * 64 + lane] = from_f32<T>(L == 0.f ? 0.f : o / L);
    if (a.lse && lane == 0) a.lse[((int64_t)n * a.h + head) * a.Lq + i] = L == 0.f ? -INFINITY : M + __log2f(L);
}

// How a call is cut: queries per block, splits of the keys.
struct plan_t { int nq, qtiles, splits, waves; };
plan_t attn_plan(int rows, int Q, int T, int dtype) {
    plan_t p;
    const int most = dtype == ASR_BF16 ? 8 : 4;
    p.qtiles = (Q + most - 1) / most;
    p.nq = (Q + p.qtiles - 1) / p.qtiles;
    const int tiles = (T + 63) / 64;
    p.waves = tiles < 8 ? (tiles < 4 ? (tiles < 2 ? 1 : 2) : 4) : 8;
    const int64_t blocks = (int64_t)rows * p.qtiles;
    p.splits = 1;
    if (tiles > 8 && blocks < 512) {
        const int64_t want = (512 + blocks - 1) / blocks, most_splits = (tiles + 15) / 16;
        p.splits = (int)(want < most_splits ? want : most_splits);
    }
    return p;
}

template <typename T, int ND> int attn_launch(hipStream_t s, const attn4_t& a, const plan_t& p) {
    const size_t work = (size_t)p.waves * 3072 + p.nq * (ND * 64 + 8), join = (size_t)p.waves * p.nq * 66 * 4;
    const size_t lds = work > join ? work : join;
    const int64_t octs = ((int64_t)a.rows * a.splits + 7) / 8;
    const dim3 grid((unsigned)(octs * 8 * a.qtiles)), block(p.waves * 64);
#define ASR_C4(NQ)                                                                                      \
    case NQ:                                                                                            \
        if constexpr (ND == 2 || NQ <= 4) hipLaunchKernelGGL((cache4_attn_kernel<T, ND, NQ>), grid, block, lds, s, a); \
        break;
    switch (p.nq) { ASR_C4(1) ASR_C4(2) ASR_C4(3) ASR_C4(4) ASR_C4(5) ASR_C4(6) ASR_C4(7) ASR_C4(8) }
#undef ASR_C4
    ASR_LAUNCH_CHECK("cache4_attention");
    if (a.splits > 1) {
        hipLaunchKernelGGL((cache4_join_kernel<T>), dim3((unsigned)((int64_t)a.rows * (a.h / a.h_kv) * a.Lq)), dim3(256), 0, s, a);
        ASR_LAUNCH_CHECK("cache4_attention (join)");
    }
    return 0;
}

int slots_plan(const char* name, slots_t& s, int64_t& blocks, int n_kv, int N, int h, int L, int Tmax, const int32_t* pos, int pos_stride,
               const int32_t* n_tok) {
    ASR_REQUIRE(n_kv > 0 && N > 0 && h > 0 && L > 0 && Tmax > 0, ASR_ERR_ARG, "%s: bad sizes (n_kv=%d N=%d h=%d L=%d Tmax=%d)", name, n_kv, N, h, L, Tmax);
    ASR_REQUIRE(Tmax <= CACHE4_MAX_T && L <= CACHE4_MAX_T, ASR_ERR_UNSUPPORTED, "%s: more than 2^24 slots", name);
    ASR_REQUIRE(pos_stride == 0 || pos_stride == 1, ASR_ERR_ARG, "%s: pos_stride is 0 (one position for all rows) or 1", name);
    const int64_t rows = (int64_t)n_kv * N * h;
    int tb = 1, lg = 0;
    while (tb < 32 && tb < L) { tb *= 2; ++lg; }
    const int chunks = (L + tb * ITER - 1) / (tb * ITER);
    blocks = (rows + (32 >> lg) - 1) / (32 >> lg) * chunks;
    ASR_REQUIRE(rows <= INT32_MAX && blocks <= INT32_MAX, ASR_ERR_UNSUPPORTED, "%s: too many rows", name);
    s = slots_t{pos, n_tok, pos_stride, N, h, L, Tmax, tb, lg, chunks, (int)rows};
    return 0;
}
bool strides_ok(const strides_t& st, int per16) { return st.kv % per16 == 0 && st.n % per16 == 0 && st.head % per16 == 0 && st.tok % per16 == 0; }

}  // namespace

extern "C" int asr_cache4_put(void* stream, const void* x, int x_dtype, int64_t s_kv, int64_t s_n, int64_t s_head, int64_t s_tok, void* codes,
                              void* meta, const int32_t* pos, int pos_stride, const int32_t* n_new, int n_kv, int N, int h, int L, int Tmax) {
    ASR_REQUIRE(x && codes && meta, ASR_ERR_ARG, "cache4_put: null pointer");
    ASR_REQUIRE(x_dtype == ASR_F32 || x_dtype == ASR_BF16, ASR_ERR_ARG, "cache4_put: dtype %d (ASR_F32 or ASR_BF16)", x_dtype);
    slots_t s; int64_t blocks;
    if (const int rc = slots_plan("cache4_put", s, blocks, n_kv, N, h, L, Tmax, pos, pos_stride, n_new)) return rc;
    const strides_t st{s_kv, s_n, s_head, s_tok};
    ASR_REQUIRE(asr_aligned(x, 16) && asr_aligned(codes, 16) && asr_aligned(meta, 4) && strides_ok(st, x_dtype == ASR_F32 ? 4 : 8), ASR_ERR_ALIGN,
                "cache4_put: rows of x start on 16 bytes, codes on 16, meta on 4");
    hipStream_t hs = static_cast<hipStream_t>(stream);
    if (x_dtype == ASR_F32)
        hipLaunchKernelGGL((cache4_put_kernel<float>), dim3((unsigned)blocks), dim3(256), 0, hs, static_cast<const float*>(x), st,
                           static_cast<uint32_t*>(codes), static_cast<uint32_t*>(meta), s);
    else
        hipLaunchKernelGGL((cache4_put_kernel<bf16_t>), dim3((unsigned)blocks), dim3(256), 0, hs, static_cast<const bf16_t*>(x), st,
                           static_cast<uint32_t*>(codes), static_cast<uint32_t*>(meta), s);
    ASR_LAUNCH_CHECK("cache4_put");
    return 0;
}

extern "C" int asr_cache4_get(void* stream, const void* codes, const void* meta, void* out, int out_dtype, int64_t s_kv, int64_t s_n, int64_t s_head,
                              int64_t s_tok, const int32_t* pos, int pos_stride, const int32_t* n_tok, int n_kv, int N, int h, int L, int Tmax) {
    ASR_REQUIRE(out && codes && meta, ASR_ERR_ARG, "cache4_get: null pointer");
    ASR_REQUIRE(out_dtype == ASR_F32 || out_dtype == ASR_BF16, ASR_ERR_ARG, "cache4_get: dtype %d (ASR_F32 or ASR_BF16)", out_dtype);
    slots_t s; int64_t blocks;
    if (const int rc = slots_plan("cache4_get", s, blocks, n_kv, N, h, L, Tmax, pos, pos_stride, n_tok)) return rc;
    const strides_t st{s_kv, s_n, s_head, s_tok};
    ASR_REQUIRE(asr_aligned(out, 16) && asr_aligned(codes, 16) && asr_aligned(meta, 4) && strides_ok(st, out_dtype == ASR_F32 ? 4 : 8), ASR_ERR_ALIGN,
                "cache4_get: rows of out start on 16 bytes, codes on 16, meta on 4");
    hipStream_t hs = static_cast<hipStream_t>(stream);
    if (out_dtype == ASR_F32)
        hipLaunchKernelGGL((cache4_get_kernel<float>), dim3((unsigned)blocks), dim3(256), 0, hs, static_cast<float*>(out), st,
                           static_cast<const uint32_t*>(codes), static_cast<const uint32_t*>(meta), s);
    else
        hipLaunchKernelGGL((cache4_get_kernel<bf16_t>), dim3((unsigned)blocks), dim3(256), 0, hs, static_cast<bf16_t*>(out), st,
                           static_cast<const uint32_t*>(codes), static_cast<const uint32_t*>(meta), s);
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
    const int chunks = (int)((3 * (int64_t)Tmax + 255) / 256);
    const int64_t blocks = (int64_t)n_kv * B * h * chunks;
    ASR_REQUIRE(blocks <= INT32_MAX, ASR_ERR_UNSUPPORTED, "cache4_reorder: too many rows");
    hipLaunchKernelGGL(cache4_reorder_kernel, dim3((unsigned)blocks), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const u32x4*>(codes),
                       static_cast<const uint32_t*>(meta), static_cast<u32x4*>(out_codes), static_cast<uint32_t*>(out_meta), parent, state, B, beam, h, Tmax,
                       chunks, codes == out_codes);
    ASR_LAUNCH_CHECK("cache4_reorder");
    return 0;
}

extern "C" int64_t asr_cache4_attention_workspace_bytes(int N, int h, int h_kv, int Lq, int T, int dtype) {
    if (N <= 0 || h_kv <= 0 || h <= 0 || h % h_kv || Lq <= 0 || T <= 0 || (int64_t)N * h_kv > INT32_MAX || (int64_t)(h / h_kv) * Lq > INT32_MAX) return 0;
    const plan_t p = attn_plan(N * h_kv, h / h_kv * Lq, T, dtype);
    return p.splits == 1 ? 0 : (int64_t)N * h * Lq * p.splits * PART * 4;
}

extern "C" int asr_cache4_attention(void* stream, const void* q, int dtype, int64_t s_n, int64_t s_head, int64_t s_tok, const void* k_codes,
                                    const void* k_meta, const void* v_codes, const void* v_meta, void* ctx, float* lse, int N, int h, int h_kv, int Lq,
                                    int T, const int32_t* k_len, int causal, void* workspace, int64_t workspace_bytes) {
    ASR_REQUIRE(q && k_codes && k_meta && v_codes && v_meta && ctx, ASR_ERR_ARG, "cache4_attention: null pointer");
    ASR_REQUIRE(dtype == ASR_F32 || dtype == ASR_BF16, ASR_ERR_ARG, "cache4_attention: dtype %d (ASR_F32 or ASR_BF16)", dtype);
    ASR_REQUIRE(N > 0 && h > 0 && h_kv > 0 && Lq > 0 && T > 0 && h % h_kv == 0, ASR_ERR_ARG, "cache4_attention: bad sizes (N=%d h=%d h_kv=%d Lq=%d T=%d)", N, h, h_kv, Lq, T);
    ASR_REQUIRE(T <= CACHE4_MAX_T, ASR_ERR_UNSUPPORTED, "cache4_attention: more than 2^24 slots");
    ASR_REQUIRE((int64_t)N * h * Lq <= INT32_MAX / 128, ASR_ERR_UNSUPPORTED, "cache4_attention: more than 2^24 queries");
    ASR_REQUIRE(asr_aligned(q, 4) && asr_aligned(ctx, 4) && asr_aligned(k_codes, 16) && asr_aligned(v_codes, 16) && asr_aligned(k_meta, 4) && asr_aligned(v_meta, 4),
                ASR_ERR_ALIGN, "cache4_attention: codes start on 16 bytes, the rest on 4");
    const plan_t p = attn_plan(N * h_kv, h / h_kv * Lq, T, dtype);
    const int64_t need = p.splits == 1 ? 0 : (int64_t)N * h * Lq * p.splits * PART * 4;
    ASR_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && asr_aligned(workspace, 4)), ASR_ERR_ARG, "cache4_attention: workspace of %lld bytes needed, %lld given",
                (long long)need, (long long)(workspace ? workspace_bytes : 0));
    attn4_t a{q, s_n, s_head, s_tok, static_cast<const u32x4*>(k_codes), static_cast<const uint32_t*>(k_meta), static_cast<const u32x4*>(v_codes),
              static_cast<const uint32_t*>(v_meta), ctx, lse, static_cast<float*>(workspace), k_len, N, h, h_kv, Lq, T, causal ? 1 : 0, p.splits, p.qtiles,
              N * h_kv, p.waves};
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == ASR_BF16 ? attn_launch<bf16_t, 2>(s, a, p) : attn_launch<float, 3>(s, a, p);
}
