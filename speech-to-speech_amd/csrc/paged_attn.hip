// Attention over the paged key / value cache: softmax(scale q k^T) v for ragged new rows of every session (layout: paged.h).
//
// One tile of TK positions, per wave, with the scores TRANSPOSED so that a lane keeps one query row (column) for good:
//   S^T [16 positions][16 rows] = K Q^T       A = key rows from the page, B = query rows held in registers
//   P^T = exp2(S^T * scale * log2 e - m)      running maximum m and sum l per column, l per lane until the end: nothing through LDS
//   O^T [16 channels][16 rows] += V^T P^T     A = value rows of the transposed page, B = P^T straight from the registers S^T was in
// The C layout of a 16 x 16 product puts rows 4 g + r (g = lane / 16) into lane g's registers, the B layout wants 8 neighbours per lane: the key
// row that score tile (u, t) reads at index m is chosen as position (m / 4) 8 U + 8 u + 4 t + m % 4, and lane g holds the positions 8 U g + 8 u .. + 7
// - the 8 neighbours whose values it loads as one octet.  Grouped heads: a column is a (new row, head of the KV head's group) pair, so the group
// shares one pass over the pages.
#include "paged.h"

#include <algorithm>

namespace s2s {

typedef float f32x8_t __attribute__((ext_vector_type(8)));

struct PagedAttn {
    PagedRows r;
    const void *kc, *vc;
    const _Float16 *km, *vm;
    const void* q; long q_rs;
    void* o; long o_rs;
    bool q_vec, o_vec;            // rows allow 16-byte reads / 4-element writes
    const int* kv_len;
    int H, G;                     // query heads, query heads per KV head
    unsigned g_magic;             // 2^32 / G + 1 where that gives every quotient of this call (0: divide)
    int max_kv, causal, window;
    float q_mul, scale_log2e;     // the scale times log2 e as a factor of the query rows, -1, 0 or 1, and a positive rest: see score_scale
    int n_splits, chunk;          // positions per split (multiple of 64)
    int q_tiles;
    bool tile;                    // attn_paged_tile_kernel (host side)
    bool by_length;               // tile kernel: sessions by falling kv_len
    float *po, *plse;             // n_splits > 1: [split][T][H][D], [split][T][H] (log2 of the sum of exp2)
};

template <int KIND> struct KvT;
template <> struct KvT<KV_F32> {
    typedef float row_t;
    typedef f32x8_t frag_t;
};
template <> struct KvT<KV_BF16> {
    typedef __hip_bfloat16 row_t;
    typedef bf16x8_t frag_t;
};
template <> struct KvT<KV_INT4> {  // codes become float16: (code - 8) scale + zero is rounded once, to 11 bits
    typedef __hip_bfloat16 row_t;
    typedef f16x8_t frag_t;
};
// 32-deep product steps of a tile along the positions: 64 positions, 32 where a tile of 64 would not leave room for a second one in the registers
constexpr int tile_u(int kind, int D) { return kind == KV_F32 || D == 256 ? 1 : 2; }

// 32-deep step of a 16 x 16 product: lane l holds row l % 16, elements 8 (l / 16) .. + 7 of both operands (f32: eight 4-deep products; both operands
// deal their elements out alike, so the order within the 32 does not matter)
__device__ __forceinline__ f32x4_t mma(const bf16x8_t& a, const bf16x8_t& b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4_t mma(const f16x8_t& a, const f16x8_t& b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4_t mma(const f32x8_t& a, const f32x8_t& b, f32x4_t c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

// bits of an octet's elements inside [lo, hi): positions nobody attends to may hold NaN, and 0 x NaN is NaN
template <typename F> struct OctetBits {
    static constexpr int N = sizeof(F) / 4;
    typedef unsigned bits_t __attribute__((ext_vector_type(N)));
    bits_t w;
    __device__ __forceinline__ OctetBits(int first, int lo, int hi) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (N == 8) w[i] = first + i >= lo && first + i < hi ? ~0u : 0u;
            else w[i] = (first + 2 * i >= lo && first + 2 * i < hi ? 0xffffu : 0u) | (first + 2 * i + 1 >= lo && first + 2 * i + 1 < hi ? 0xffff0000u : 0u);
        }
    }
    __device__ __forceinline__ F keep(const F& f) const { return __builtin_bit_cast(F, __builtin_bit_cast(bits_t, f) & w); }
};

__device__ __forceinline__ float max_over_groups(float x) {        // over the 4 lanes l, l ^ 16, l ^ 32, l ^ 48
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// new row of column vr (vr >= 0): vr / G
__device__ __forceinline__ int row_of(const PagedAttn& p, int vr) { return p.G == 1 ? vr : p.g_magic ? (int)__umulhi((unsigned)vr, p.g_magic) : vr / p.G; }

// where the columns of a tile of query rows stand
struct Span {
    int row0, n, rows;            // rows of the session that are computed, and uncut
    int len, past;                // positions that count; positions before the new rows' own (negative: the first rows see nothing).  A session beyond the
                                  // bounds has fewer rows and positions, but those that are left keep their places: `past` is taken from the uncut numbers
    int lo, hi;                   // positions some row of the tile sees: [lo, hi); empty where lo >= hi
    int lo_all, hi_all;           // positions every row sees
};
__device__ __forceinline__ bool tile_span(const PagedAttn& p, int b, int vr0, int nvr, Span& s) {
    const int len = max(p.kv_len[b], 0);
    s.rows = session_rows(p.r, b, s.row0, s.n);
    if (s.n <= 0 || s.row0 >= p.r.T || vr0 >= s.n * p.G) return false;
    s.len = min(len, p.max_kv);
    s.past = len - s.rows;
    const int t0 = row_of(p, vr0), t_last = row_of(p, min(vr0 + nvr, s.n * p.G) - 1);
    s.hi = p.causal ? max(0, min(s.len, s.past + t_last + 1)) : s.len;
    s.hi_all = p.causal ? max(0, min(s.len, s.past + t0 + 1)) : s.len;
    s.lo = p.window > 0 ? max(0, min(s.len, s.past + t0 + 1 - p.window)) : 0;
    s.lo_all = p.window > 0 ? max(0, s.past + t_last + 1 - p.window) : 0;
    return true;
}

// A score that a mask hides is -inf before it is scaled, so what scores are multiplied by has to be positive, or -inf would become NaN or +inf: the sign of the
// scale, or its being zero, goes to the query row, where both are exact and a NaN stays one.  4 bits: the row's power of two times the scale may leave
// the floats at either end, where it is cut (a positive factor below the smallest normal float makes every score 0 as the float itself does).
template <int KIND> __device__ __forceinline__ float score_scale(const PagedAttn& p, float mul) {
    return KIND == KV_INT4 ? fminf(fmaxf(mul * p.scale_log2e, 0x1p-126f), 0x1.fffffep127f) : p.scale_log2e;
}

// Rows of a session beyond max_new get no partial results.  The join, which goes by rows, leaves out those whose weight in split 0 is +inf, which no result is (a
// maximum of +inf comes with a NaN or an empty sum): one workgroup of the session puts it there.
__device__ __forceinline__ void leave_rows(const PagedAttn& p, const Span& s) {
    const long end = min((long)s.row0 + s.rows, (long)p.r.T) * p.H;
    for (long i = ((long)s.row0 + s.n) * p.H + threadIdx.x; i < end; i += 256) p.plse[i] = INFINITY;
}

// 4 octets of a query row per 128 channels in the operand's type, times q_mul.  4-bit caches: float16 after dividing the row by a power of two (exact), so that its
// largest value lies in [1, 2); `mul` gives it back.  bf16 values down to 2^-17 of the largest stay exact, smaller ones are off by at most 2^-25 of it.
template <int KIND, int D>
__device__ __forceinline__ void load_query(const typename KvT<KIND>::row_t* row, bool vec, float q_mul, int g, typename KvT<KIND>::frag_t (&q)[D / 32], float& mul) {
    mul = 1.f;
    typedef typename KvT<KIND>::row_t T;
    typedef typename KvT<KIND == KV_INT4 ? KV_BF16 : KIND>::frag_t raw_t;
    raw_t w[D / 32];
    if (vec) {
#pragma unroll
        for (int s = 0; s < D / 32; ++s) w[s] = *reinterpret_cast<const raw_t*>(row + s * 32 + g * 8);
    } else {
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            T one[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) one[e] = row[s * 32 + g * 8 + e];
            __builtin_memcpy(&w[s], one, sizeof(one));
        }
    }
    if (q_mul != 1.f) {
        typedef std::remove_reference_t<decltype(w[0][0])> elem_t;
#pragma unroll
        for (int s = 0; s < D / 32; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) w[s][e] = (elem_t)((float)w[s][e] * q_mul);
    }
    if constexpr (KIND == KV_INT4) {
        float m = 0.f;
#pragma unroll
        for (int s = 0; s < D / 32; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf((float)w[s][e]));
        m = max_over_groups(m);
        const int ex = m > 0.f && m < INFINITY ? ilogbf(m) : 0;
        mul = ldexpf(1.f, ex);
#pragma unroll
        for (int s = 0; s < D / 32; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) q[s][e] = (_Float16)ldexpf((float)w[s][e], -ex);
    } else {
#pragma unroll
        for (int s = 0; s < D / 32; ++s) q[s] = w[s];
    }
}

// (code - 8) scale + zero of an octet
__device__ __forceinline__ f16x8_t dequant(unsigned w, f16x2_t s0, f16x2_t s1, f16x2_t s2, f16x2_t s3, f16x2_t z0, f16x2_t z1, f16x2_t z2, f16x2_t z3) {
    f16x2_t c[4];
    codes_to_f16(w, c);
    const f16x2_t a = __builtin_elementwise_fma(c[0], s0, z0), b = __builtin_elementwise_fma(c[1], s1, z1);
    const f16x2_t d = __builtin_elementwise_fma(c[2], s2, z2), e = __builtin_elementwise_fma(c[3], s3, z3);
    return f16x8_t{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}
__device__ __forceinline__ f16x8_t dequant_key(unsigned w, unsigned meta) {
    const f16x2_t m = __builtin_bit_cast(f16x2_t, meta);
    const f16x2_t s = {m[0], m[0]}, z = {m[1], m[1]};
    return dequant(w, s, s, s, s, z, z, z, z);
}
__device__ __forceinline__ f16x8_t dequant_val(unsigned w, const f16x8_t& s, const f16x8_t& z) {
    return dequant(w, f16x2_t{s[0], s[1]}, f16x2_t{s[2], s[3]}, f16x2_t{s[4], s[5]}, f16x2_t{s[6], s[7]}, f16x2_t{z[0], z[1]}, f16x2_t{z[2], z[3]}, f16x2_t{z[4], z[5]},
                   f16x2_t{z[6], z[7]});
}

// One tile's keys / values as a wave holds them: what was loaded, and the operand of one product from it.  Addresses are a uniform base (scalar
// registers) plus one 32-bit offset per lane that never changes.
template <typename V> __device__ __forceinline__ V ld_at(const void* base, unsigned off) { return *reinterpret_cast<const V*>((const char*)base + off); }
// A code page is read once per step and a wave's load takes whole lines of it: past the caches (64 x 1500 positions of 20 heads of 64: 37.8 -> 32.2 us).
// Rows of the model type take two loads per line and need it kept in between (512 sessions of bf16: 304 us, 333 us this way).
template <typename V> __device__ __forceinline__ V ld_once(const void* base, unsigned off) {
    return __builtin_nontemporal_load(reinterpret_cast<const V*>((const char*)base + off));
}

template <int KIND, int D> struct KeyTile {       // bf16, f32: octets of the U x 2 rows this lane stands for
    static constexpr int U = tile_u(KIND, D), EB = KIND == KV_F32 ? 4 : 2;
    typename KvT<KIND>::frag_t f[U][2][D / 32];
    static __device__ __forceinline__ unsigned lane_off(int l15, int g) { return (((l15 >> 2) * 8 * U + (l15 & 3)) * D + g * 8) * EB; }
    __device__ __forceinline__ void load(const PagedAttn& p, long head, int at, unsigned off, int) {
        const char* base = (const char*)p.kc + ((head << p.r.ps_log2) + at) * D * EB;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int s = 0; s < D / 32; ++s) f[u][t][s] = ld_at<typename KvT<KIND>::frag_t>(base + ((u * 8 + t * 4) * D + s * 32) * EB, off);
    }
    __device__ __forceinline__ void ready(unsigned char*, int) {}
    __device__ __forceinline__ typename KvT<KIND>::frag_t get(const unsigned char*, int, int, int u, int t, int s) const { return f[u][t][s]; }
};
template <int KIND, int D> struct ValTile {
    static constexpr int U = tile_u(KIND, D), EB = KIND == KV_F32 ? 4 : 2;
    typename KvT<KIND>::frag_t f[D / 16][U];
    static __device__ __forceinline__ unsigned lane_off(int l15, int g, int ps_log2) { return ((l15 << ps_log2) + g * 8 * U) * EB; }
    static __device__ __forceinline__ unsigned meta_off(int, int) { return 0; }
    __device__ __forceinline__ void load(const PagedAttn& p, long head, int at, unsigned off, unsigned) {
        const char* base = (const char*)p.vc + (((head * D) << p.r.ps_log2) + at) * EB;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int u = 0; u < U; ++u) f[d][u] = ld_at<typename KvT<KIND>::frag_t>(base + ((d * 16 << p.r.ps_log2) + u * 8) * EB, off);
    }
    // edge: values outside [lo, hi) become 0
    __device__ __forceinline__ void ready(unsigned char*, int, int g, bool edge, int kb, int lo, int hi) {
        if (!edge) return;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const OctetBits<typename KvT<KIND>::frag_t> bits(kb + (g * U + u) * 8, lo, hi);
#pragma unroll
            for (int d = 0; d < D / 16; ++d) f[d][u] = bits.keep(f[d][u]);
        }
    }
    __device__ __forceinline__ typename KvT<KIND>::frag_t get(const unsigned char*, int, int d, int u) const { return f[d][u]; }
};
// 4 bits: a lane needs the scales and zeros of its key rows (shared by 4 lanes) and of its 8 U positions in every group (shared by 16).  Loaded as
// needed they would be two thirds of the lane traffic, and 80 registers at 128 channels; so the wave loads a tile's scales and zeros once, 8 or 16 bytes a
// lane, and deals them out through LDS of its own.
template <int D> struct CodeMeta {
    static constexpr int U = tile_u(KV_INT4, D), TK = 32 * U, NS = D / 32, W = TK * NS / 64;      // dwords per lane; 64 lanes: a tile's keys or values
    static constexpr int BYTES = W * 4 * 64;
    typedef unsigned words_t __attribute__((ext_vector_type(W)));
};
template <int D> struct KeyTile<KV_INT4, D> {
    typedef CodeMeta<D> M;
    static constexpr int U = M::U, NS = M::NS;
    typedef unsigned words_t __attribute__((ext_vector_type(NS)));
    words_t w[U][2];
    typename M::words_t m;
    static __device__ __forceinline__ unsigned lane_off(int l15, int g) { return ((l15 >> 2) * 8 * U + (l15 & 3)) * (D / 2) + g * NS * 4; }
    __device__ __forceinline__ void load(const PagedAttn& p, long head, int at, unsigned off, int lane) {
        const long row = (head << p.r.ps_log2) + at;
        const char* base = (const char*)p.kc + row * (D / 2);
        m = ld_once<typename M::words_t>((const char*)p.km + row * (D / 8), lane * M::W * 4);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < 2; ++t) w[u][t] = ld_once<words_t>(base + (u * 8 + t * 4) * (D / 2), off);
    }
    __device__ __forceinline__ void ready(unsigned char* own, int lane) {
        __builtin_amdgcn_wave_barrier();           // the wave's reads of the last tile come first (LDS keeps a wave's order; the compiler must)
        *reinterpret_cast<typename M::words_t*>(own + lane * M::W * 4) = m;
        __builtin_amdgcn_wave_barrier();
    }
    __device__ __forceinline__ f16x8_t get(const unsigned char* own, int l15, int, int u, int t, int s) const {
        const words_t row = *reinterpret_cast<const words_t*>(own + ((l15 >> 2) * 8 * U + (l15 & 3) + u * 8 + t * 4) * (D / 8));
        return dequant_key(w[u][t][s], row[s]);
    }
};
template <int D> struct ValTile<KV_INT4, D> {
    typedef CodeMeta<D> M;
    static constexpr int U = M::U;
    typedef unsigned words_t __attribute__((ext_vector_type(U)));
    words_t w[D / 16];
    typename M::words_t m;
    static __device__ __forceinline__ unsigned lane_off(int l15, int g, int ps_log2) { return (l15 << (ps_log2 - 1)) + g * U * 4; }
    static __device__ __forceinline__ unsigned meta_off(int lane, int ps_log2) {                  // rows of TK float16: scales, zeros of every group
        return (((unsigned)(lane * M::W * 2 / M::TK) << ps_log2) + lane * M::W * 2 % M::TK) * 2;
    }
    __device__ __forceinline__ void load(const PagedAttn& p, long head, int at, unsigned off, unsigned moff) {
        const char* base = (const char*)p.vc + ((head * D) << (p.r.ps_log2 - 1)) + (at >> 1);
        m = ld_once<typename M::words_t>((const char*)(p.vm + ((head * (D / 32) * 2) << p.r.ps_log2) + at), moff);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) w[d] = ld_once<words_t>(base + (d * 16 << (p.r.ps_log2 - 1)), off);
    }
    // edge: scale and zero 0 outside [lo, hi), a value of 0 whatever the code
    __device__ __forceinline__ void ready(unsigned char* own, int lane, int, bool edge, int kb, int lo, int hi) {
        if (edge) {
            const int first = kb + lane * M::W * 2 % M::TK;
#pragma unroll
            for (int i = 0; i < M::W; ++i)
                m[i] &= (first + 2 * i >= lo && first + 2 * i < hi ? 0xffffu : 0u) | (first + 2 * i + 1 >= lo && first + 2 * i + 1 < hi ? 0xffff0000u : 0u);
        }
        __builtin_amdgcn_wave_barrier();
        *reinterpret_cast<typename M::words_t*>(own + M::BYTES + lane * M::W * 4) = m;
        __builtin_amdgcn_wave_barrier();
    }
    __device__ __forceinline__ f16x8_t get(const unsigned char* own, int g, int d, int u) const {
        const unsigned char* row = own + M::BYTES + ((d >> 1) * 2 * M::TK + (g * U + u) * 8) * 2;
        return dequant_val(w[d][u], *reinterpret_cast<const f16x8_t*>(row), *reinterpret_cast<const f16x8_t*>(row + M::TK * 2));
    }
};

// 4 neighbouring channels of an output row
__device__ __forceinline__ void store4(float* o, const f32x4_t& v, bool vec) {
    if (vec) {
        *reinterpret_cast<f32x4_t*>(o) = v;
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = v[r];
}
__device__ __forceinline__ void store4(__hip_bfloat16* o, const f32x4_t& v, bool vec) {
    const u32x2_t w = {pack_bf16x2_hw(v[0], v[1]), pack_bf16x2_hw(v[2], v[3])};
    if (vec) {
        *reinterpret_cast<u32x2_t*>(o) = w;
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) reinterpret_cast<unsigned short*>(o)[r] = (unsigned short)(w[r >> 1] >> (16 * (r & 1)));
}

// P^T octet as product operand(s).  bf16: a second operand holds what the first rounding left (p = hi + lo to 16 bits), where the products are not
// what bounds the kernel.
__device__ __forceinline__ void probs(const float (&x)[8], f32x8_t& hi) {
#pragma unroll
    for (int e = 0; e < 8; ++e) hi[e] = x[e];
}
__device__ __forceinline__ void probs(const float (&x)[8], f16x8_t& hi) {
#pragma unroll
    for (int e = 0; e < 8; ++e) hi[e] = (_Float16)x[e];
}
__device__ __forceinline__ void probs(const float (&x)[8], bf16x8_t& hi) {
#pragma unroll
    for (int e = 0; e < 8; ++e) hi[e] = (__bf16)x[e];
}

// The running maximum is raised only when a score exceeds it by more than 8 (in log2): P stays below 2^8, sums and products are f32, so nothing is lost,
// and the usual step needs no cross-lane maximum and no rescaling.
constexpr float MAX_SLACK = 8.f;
// The maximum that is kept lies this far below the true one, so that the weights fill the upper range of float16 (up to 2^15) and a long tail of small ones does
// not fall off its lower end: 2^-32 of the largest weight is still seen.  bf16 and f32 have room on both sides.
constexpr float max_bias(int kind) { return kind == KV_INT4 ? 7.f : 0.f; }
constexpr float NO_MAX = -3e38f;                  // finite, so that masked scores (-inf) minus it stay -inf

// scores of a tile -> softmax step and products with the tile's values
template <int KIND, int D>
__device__ __forceinline__ void step_tile(const f32x4_t (&s)[tile_u(KIND, D)][2], const ValTile<KIND, D>& vt, const unsigned char* own, int g, float sc, float& m, float& l, f32x4_t (&acc)[D / 16]) {
    typedef typename KvT<KIND>::frag_t frag_t;
    constexpr int U = tile_u(KIND, D), ND = D / 16;
    float x[U][8], mx = NO_MAX;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[u][e] = fmaf(s[u][e >> 2][e & 3], sc, -m);
            mx = fmaxf(mx, x[u][e]);
        }
    if (__any(mx > MAX_SLACK + max_bias(KIND))) {
        float mn = m + max_bias(KIND);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) mn = fmaxf(mn, s[u][e >> 2][e & 3] * sc);
        mn = max_over_groups(mn) - max_bias(KIND);
        const float a = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= a;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] *= a;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[u][e] = fmaf(s[u][e >> 2][e & 3], sc, -mn);
    }
    frag_t ph[U];
    bf16x8_t pl[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[u][e] = __builtin_amdgcn_exp2f(x[u][e]);
            l += x[u][e];
        }
        probs(x[u], ph[u]);
        if constexpr (KIND == KV_BF16) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[u][e] -= (float)ph[u][e];
            probs(x[u], pl[u]);
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const frag_t v = vt.get(own, g, d, u);
            acc[d] = mma(v, ph[u], acc[d]);
            if constexpr (KIND == KV_BF16) acc[d] = mma(v, pl[u], acc[d]);
        }
    }
}

// ---- few rows per session: every wave streams its own tiles from memory into registers -----------------------------------------------------
// grid (q_tiles * n_splits, Hkv, B), W waves; wave w takes the split's tiles w, w + W, ...; their partial softmaxes meet in LDS at the end.  Bound
// by HBM: keys and values go straight into the operand registers, the loads of the next keys are issued before this tile's softmax and those of
// the next values behind this tile's products, so both are in flight while the other is used.  512 sessions of up to 1531 positions, 16 / 8 heads of 128, bf16: 304 us,
// 5.5 TB/s (a large copy reaches 4.9); 4 bits, 64 x 1500 positions of 20 heads of 64: 31.6 us, 4.9 TB/s; 7 sessions of up to 100021: 104 us, 5.0 TB/s.
template <int KIND, int D>
__global__ __launch_bounds__(256, KIND == KV_INT4 ? (D == 64 ? 4 : D == 128 ? 3 : 2) : D == 256 ? 1 : 2) void attn_paged_step_kernel(PagedAttn p) {
    typedef typename KvT<KIND>::row_t T;
    typedef typename KvT<KIND>::frag_t frag_t;
    constexpr int W = 4, U = tile_u(KIND, D), TK = 32 * U, NS = D / 32, ND = D / 16;
    __shared__ float so[W / 2][16][D + 4];
    __shared__ float sm[W][16], sl[W][16];
    __shared__ alignas(16) unsigned char meta[KIND == KV_INT4 ? W * 2 * CodeMeta<D>::BYTES : 16];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
    unsigned char* own = meta + (KIND == KV_INT4 ? wave * 2 * CodeMeta<D>::BYTES : 0);
    const int b = blockIdx.z, hk = blockIdx.y, split = blockIdx.x % p.n_splits, vr0 = (blockIdx.x / p.n_splits) * 16;
    Span sp;
    if (!tile_span(p, b, vr0, 16, sp)) return;
    if (p.n_splits > 1 && blockIdx.x == 0 && hk == 0) leave_rows(p, sp);
    // a column behind the last (row, head) does the last one's work again and stores nothing
    const bool valid = vr0 + l15 < sp.n * p.G;
    const int vr = min(vr0 + l15, sp.n * p.G - 1), t = row_of(p, vr), h = hk * p.G + vr - t * p.G;
    const int c_hi = p.causal ? min(sp.len, sp.past + t + 1) : sp.len;
    const int c_lo = p.window > 0 ? sp.past + t + 1 - p.window : 0;
    const int k0 = (sp.lo & ~63) + split * p.chunk, k1 = min(sp.hi, k0 + p.chunk);

    f32x4_t acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m = NO_MAX, l = 0.f;

    int kb = k0 + wave * TK;
    if (kb < k1) {
        KeyTile<KIND, D> kt;
        ValTile<KIND, D> vt;
        const int ps_mask = (1 << p.r.ps_log2) - 1;
        const unsigned k_off = KeyTile<KIND, D>::lane_off(l15, g), v_off = ValTile<KIND, D>::lane_off(l15, g, p.r.ps_log2);
        const unsigned m_off = ValTile<KIND, D>::meta_off(lane, p.r.ps_log2);
        int page = page_raw(p.r, b, kb), next = kb + W * TK < k1 ? page_raw(p.r, b, kb + W * TK) : -1;
        {
            const long head = (long)(page_ok(p.r, page) ? page : 0) * p.r.Hkv + hk;
            kt.load(p, head, kb & ps_mask, k_off, lane);
            vt.load(p, head, kb & ps_mask, v_off, m_off);
        }
        frag_t q[NS];                              // (behind the first tile's loads, so that they are on their way while it is waited for)
        float sc;
        load_query<KIND, D>((const T*)p.q + (sp.row0 + (long)t) * p.q_rs + (long)h * D, p.q_vec, p.q_mul, g, q, sc);
        sc = score_scale<KIND>(p, sc);
        for (; kb < k1; kb += W * TK) {
            const int nb = kb + W * TK;
            const long nhead = (long)(page_ok(p.r, next) ? next : 0) * p.r.Hkv + hk;
            const int after = nb + W * TK < k1 ? page_raw(p.r, b, nb + W * TK) : -1;
            const int nat = nb < k1 ? nb & ps_mask : 0;
            f32x4_t s[U][2];
            kt.ready(own, lane);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    s[u][tt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < NS; ++k) s[u][tt] = mma(kt.get(own, l15, g, u, tt, k), q[k], s[u][tt]);
                }
            if (nb < k1) kt.load(p, nhead, nat, k_off, lane);
            if (page_ok(p.r, page)) {
                const bool edge = kb < sp.lo_all || kb + TK > sp.hi_all;
                if (edge) {
                    const int pos = kb + g * 8 * U;
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (pos + u * 8 + e < c_lo || pos + u * 8 + e >= c_hi) s[u][e >> 2][e & 3] = -INFINITY;
                }
                vt.ready(own, lane, g, edge, kb, sp.lo, sp.hi);
                step_tile<KIND, D>(s, vt, own, g, sc, m, l, acc);
            }
            if (nb < k1) vt.load(p, nhead, nat, v_off, m_off);
            page = next;
            next = after;
        }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // W partial softmaxes of the same 16 columns -> one: common maximum first, then the upper half of the waves onto the lower, and again
    if (g == 0) {
        sm[wave][l15] = m;
        sl[wave][l15] = l;
    }
    __syncthreads();
    float M = sm[0][l15];
#pragma unroll
    for (int w = 1; w < W; ++w) M = fmaxf(M, sm[w][l15]);
    float L = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) L += sl[w][l15] * __builtin_amdgcn_exp2f(sm[w][l15] - M);
    const float mine = __builtin_amdgcn_exp2f(m - M);
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] *= mine;
#pragma unroll
    for (int half = W / 2; half >= 1; half >>= 1) {
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4_t*>(&so[wave - half][l15][d * 16 + g * 4]) = acc[d];
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[d] += *reinterpret_cast<const f32x4_t*>(&so[wave][l15][d * 16 + g * 4]);
        }
        __syncthreads();
    }
    if (wave != 0 || !valid) return;
    const float inv = L > 0.f ? 1.f / L : 0.f;
    const long row = sp.row0 + t;
    if (p.n_splits == 1) {
        T* o = (T*)p.o + row * p.o_rs + (long)h * D + g * 4;
#pragma unroll
        for (int d = 0; d < ND; ++d) store4(o + d * 16, L == 0.f ? f32x4_t{0.f, 0.f, 0.f, 0.f} : acc[d] * inv, p.o_vec);
    } else {
        const long at = ((long)split * p.r.T + row) * p.H + h;
        if (g == 0) p.plse[at] = L == 0.f ? -INFINITY : M + __builtin_amdgcn_logf(L);
        if (L == 0.f) return;      // the join reads no row of weight 0
#pragma unroll
        for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4_t*>(p.po + at * D + d * 16 + g * 4) = acc[d] * inv;
    }
}

// ---- many rows per session: a workgroup's tile of query rows shares every tile of positions through LDS ----------------------------------------
// 4 waves x NC x 16 columns.  Tiles of keys and values go from the page into LDS without passing registers (4-bit codes: through registers, as
// float16), a double buffer and one barrier per tile.  Octets are stored at index o ^ f(row), f different for the 16 lanes that read together, so that
// the 16-byte reads hit every bank once (SQ_LDS_BANK_CONFLICT 0; 53 M cycles with 8 values of f).  NC = 2: one operand read serves two products.
// Bound, at 428 GFLOP of bf16 prompts (437 us, 980 TFLOP/s, the library's 8192^3 product reaches 1210): a tile step is the 1024 cycles of its products plus the
// 800 of its softmax, which two waves per SIMD overlap only in part, at 2.0 - 2.1 GHz.  Scores of tile t + 1 beside the exponentials of tile t, in the
// compiler's order or a prescribed one, 32-position tiles at 3 waves per SIMD and 48 rows per wave (spills) were not faster.
template <int KIND, int D> struct LdsTile {
    static constexpr int U = tile_u(KIND, D), TK = 32 * U;
    static constexpr int EB = KIND == KV_F32 ? 4 : 2, OB = 8 * EB;  // bytes per element and per octet in LDS
    static constexpr int K_BYTES = TK * D * EB, BYTES = 2 * K_BYTES;
    static constexpr int FB = U == 2 ? 4 : 3;                      // position bit that l15's bit 2 is
    static constexpr int HB = D == 64 ? 1 : 2;                     // bits of f above the lowest two
    // 16 lanes read together and the banks span 256 bytes: a key row of 128 channels or more takes all 16 of f, two rows of 64 share the span (the row's
    // parity is the slot's top bit) and take 8
    static __device__ __forceinline__ int kf(int key) { return D == 64 ? ((key >> 1) & 1) | ((key >> FB) & 3) << 1 : (key & 3) | ((key >> FB) & 3) << 2; }
    static __device__ __forceinline__ int vf(int d) { return U == 2 ? (d >> 1) & 7 : KIND == KV_F32 ? d & 3 : (d >> 2) & 3; }
    // value octets trade places so that lanes of neighbouring g, which share a read cycle on opposite quarters of the rows, stay apart too
    static __device__ __forceinline__ int vs(int o) { return U == 2 ? (o & 1) << 2 | o >> 1 : KIND == KV_F32 ? o : (0x9c >> (2 * o)) & 3; }
    static __device__ __forceinline__ int vo(int s) { return U == 2 ? (s & 3) << 1 | s >> 2 : KIND == KV_F32 ? s : (0x78 >> (2 * s)) & 3; }     // back
    static __device__ __forceinline__ int k_at(int key, int o) { return (key * (D / 8) + (o ^ kf(key))) * OB; }
    static __device__ __forceinline__ int v_at(int d, int o) { return K_BYTES + (d * (TK / 8) + (vs(o) ^ vf(d))) * OB; }
};
// The reading side: f depends on l15 only, whatever the product, so a few lane offsets serve all reads and the rest are constants: octet 4 k + g of a key
// row lies 4 OB (k ^ f / 4) behind octet (g ^ f % 4).
template <int KIND, int D> struct LdsOff {
    typedef LdsTile<KIND, D> L;
    static constexpr int NK = 1 << L::HB;
    int k[NK], v[L::U];
    __device__ __forceinline__ LdsOff(int l15, int g) {
        const int key = (l15 >> 2) * 8 * L::U + (l15 & 3);
#pragma unroll
        for (int i = 0; i < NK; ++i) k[i] = L::k_at(key, 4 * i + g) - 4 * L::OB * i;
#pragma unroll
        for (int u = 0; u < L::U; ++u) v[u] = L::v_at(l15, g * L::U + u);
    }
};

// page -> LDS: 16-byte pieces in LDS order, the swizzle in the lane's source offset (a piece further on in the tile changes only the bits of f that come
// from the position bits its step reaches)
template <int KIND, int D> struct TileDma {
    typedef LdsTile<KIND, D> L;
    static constexpr int PB = L::EB / 2;                           // pieces per octet
    static constexpr int N = L::K_BYTES / 16 / 256;                // pieces per thread, keys or values
    static constexpr int KS = 256 / PB / (D / 8);                  // key rows per piece of the workgroup
    static constexpr int VS = 256 / PB / (L::TK / 8);              // value rows
    unsigned k[N], v;
    __device__ __forceinline__ TileDma(int tid, int ps_log2) {
        const int o = tid / PB, half = tid % PB;
        const int key = o / (D / 8), d = o / (L::TK / 8);
#pragma unroll
        for (int i = 0; i < N; ++i) k[i] = (key * D + ((o % (D / 8)) ^ L::kf(i * KS + key)) * 8) * L::EB + half * 16;
        v = (((unsigned)d << ps_log2) + L::vo((o % (L::TK / 8)) ^ L::vf(d)) * 8) * L::EB + half * 16;
    }
    __device__ __forceinline__ void start(const PagedAttn& p, unsigned char* buf, int page, int hk, int at, int wave) const {
        const long head = (long)page * p.r.Hkv + hk;
        const char* kb = (const char*)p.kc + ((head << p.r.ps_log2) + at) * D * L::EB;
        const char* vb = (const char*)p.vc + (((head * D) << p.r.ps_log2) + at) * L::EB;
#pragma unroll
        for (int i = 0; i < N; ++i)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(kb + i * KS * D * L::EB + k[i]),
                                             (__attribute__((address_space(3))) void*)(buf + (i * 4 + wave) * 1024), 16, 0, 0);
#pragma unroll
        for (int i = 0; i < N; ++i)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(vb + (((long)i * VS) << p.r.ps_log2) * L::EB + v),
                                             (__attribute__((address_space(3))) void*)(buf + L::K_BYTES + (i * 4 + wave) * 1024), 16, 0, 0);
    }
};
// 4-bit page -> registers: TK D / 2048 octets of one key; and as many octets of the same 8 positions, channels of one group, which share 8 scales and zeros
template <int D> struct CodeRegs {
    typedef LdsTile<KV_INT4, D> L;
    static constexpr int NS = D / 32, KN = L::TK * D / 2048, KT = NS * 4 / KN;     // octets per thread; threads per key
    static constexpr int VT = L::TK / 8;                                           // threads per channel
    typedef unsigned words_t __attribute__((ext_vector_type(KN)));
    words_t kw;
    unsigned km[KN], vw[KN];
    f16x8_t vs, vz;
    // dword i of a key row is octet 4 s + g with g = i / NS, s = i % NS
    __device__ __forceinline__ void load(const PagedAttn& p, int page, int hk, int at, int tid) {
        const long head = (long)page * p.r.Hkv + hk, row = (head << p.r.ps_log2) + at;
        const int key = tid / KT, i0 = tid % KT * KN, o = tid % VT, d0 = tid / VT * KN;
        kw = ld_at<words_t>((const char*)p.kc + row * (D / 2), key * (D / 2) + i0 * 4);
#pragma unroll
        for (int j = 0; j < KN; ++j) km[j] = ld_at<unsigned>((const char*)p.km + row * (D / 8), key * (D / 8) + (i0 + j) % NS * 4);
        const char* vb = (const char*)p.vc + ((head * D) << (p.r.ps_log2 - 1)) + (at >> 1);
#pragma unroll
        for (int j = 0; j < KN; ++j) vw[j] = ld_at<unsigned>(vb, ((d0 + j) << (p.r.ps_log2 - 1)) + o * 4);
        const char* m = (const char*)(p.vm + ((head * NS * 2) << p.r.ps_log2) + at);
        const unsigned moff = ((d0 / 32 * 2) << p.r.ps_log2) * 2 + o * 16;
        vs = ld_at<f16x8_t>(m, moff);
        vz = ld_at<f16x8_t>(m, moff + (2u << p.r.ps_log2));
    }
    __device__ __forceinline__ void store(unsigned char* buf, int tid) const {
        const int key = tid / KT, i0 = tid % KT * KN, o = tid % VT, d0 = tid / VT * KN;
#pragma unroll
        for (int j = 0; j < KN; ++j) *reinterpret_cast<f16x8_t*>(buf + L::k_at(key, 4 * ((i0 + j) % NS) + (i0 + j) / NS)) = dequant_key(kw[j], km[j]);
#pragma unroll
        for (int j = 0; j < KN; ++j) *reinterpret_cast<f16x8_t*>(buf + L::v_at(d0 + j, o)) = dequant_val(vw[j], vs, vz);
    }
};

// one tile: scores, softmax step, products with the values
template <int KIND, int D, int NC>
__device__ __forceinline__ void tile_step(const unsigned char* buf, const LdsOff<KIND, D>& off, const typename KvT<KIND>::frag_t (&q)[NC][D / 32], const float (&sc)[NC],
                                          bool edge, int pos0, const int (&c_lo)[NC], const int (&c_hi)[NC], float (&m)[NC], float (&l)[NC], f32x4_t (&acc)[NC][D / 16]) {
    typedef typename KvT<KIND>::frag_t frag_t;
    typedef LdsTile<KIND, D> L;
    constexpr int U = L::U, NS = D / 32, ND = D / 16;
    f32x4_t s[NC][U][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
            for (int c = 0; c < NC; ++c) s[c][u][tt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                const frag_t a = *reinterpret_cast<const frag_t*>(buf + off.k[k & (LdsOff<KIND, D>::NK - 1)] + ((u * 8 + tt * 4) * (D / 8) + 4 * k) * L::OB);
#pragma unroll
                for (int c = 0; c < NC; ++c) s[c][u][tt] = mma(a, q[c][k], s[c][u][tt]);
            }
        }
    if (edge) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (pos0 + u * 8 + e < c_lo[c] || pos0 + u * 8 + e >= c_hi[c]) s[c][u][e >> 2][e & 3] = -INFINITY;
    }
    float x[NC][U][8];
    bool raise = false;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float mx = NO_MAX;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[c][u][e] = fmaf(s[c][u][e >> 2][e & 3], sc[c], -m[c]);
                mx = fmaxf(mx, x[c][u][e]);
            }
        raise |= mx > MAX_SLACK + max_bias(KIND);
    }
    if (__any(raise)) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float mn = m[c] + max_bias(KIND);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) mn = fmaxf(mn, s[c][u][e >> 2][e & 3] * sc[c]);
            mn = max_over_groups(mn) - max_bias(KIND);
            const float a = __builtin_amdgcn_exp2f(m[c] - mn);
            m[c] = mn;
            l[c] *= a;
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[c][d] *= a;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[c][u][e] = fmaf(s[c][u][e >> 2][e & 3], sc[c], -mn);
        }
    }
    frag_t pr[NC][U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[c][u][e] = __builtin_amdgcn_exp2f(x[c][u][e]);
                l[c] += x[c][u][e];
            }
            probs(x[c][u], pr[c][u]);
        }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const frag_t v = *reinterpret_cast<const frag_t*>(buf + off.v[u] + d * 16 * (L::TK / 8) * L::OB);
#pragma unroll
            for (int c = 0; c < NC; ++c) acc[c][d] = mma(v, pr[c][u], acc[c][d]);
        }
}

// The session whose kv_len is the i-th largest (up to 64 sessions, a lane each: beyond that there are workgroups enough for the order not to matter).  Long
// sessions are begun first, so that what is left at the end is short (ragged prompts: 462 -> 437 us; 16 sessions over 4-bit pages, all workgroups resident at once, so
// that long ones share a CU with short ones: 142 -> 124 us).  Ranking takes 0.5 us (8 sessions) to 1.7 us (64): only where it pays, see attn_launch.
__device__ __forceinline__ int session_by_length(const PagedAttn& p, int i, int lane) {
    if (!p.by_length) return i;
    const int len = lane < p.r.B ? max(p.kv_len[lane], 0) : -1;
    int rank = 0;
    for (int j0 = 0; j0 < p.r.B; j0 += 16)
#pragma unroll
        for (int j = 0; j < 16; ++j) {             // (lanes without a session hold -1: behind all, in lane order)
            const int other = __builtin_amdgcn_readlane(len, j0 + j);
            rank += other > len || (other == len && j0 + j < lane) ? 1 : 0;
        }
    return __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(lane < p.r.B && rank == i)) - 1);
}

template <int KIND, int D, int NC>
__global__ __launch_bounds__(256, D == 256 && KIND == KV_F32 ? 1 : 2) void attn_paged_tile_kernel(PagedAttn p) {
    typedef typename KvT<KIND>::row_t T;
    typedef typename KvT<KIND>::frag_t frag_t;
    typedef LdsTile<KIND, D> L;
    constexpr int TK = L::TK, U = L::U, NS = D / 32, ND = D / 16, RW = NC * 16;
    __shared__ alignas(16) unsigned char lds[2 * L::BYTES];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l15 = lane & 15, g = lane >> 4;
    // workgroups with the same (session, KV head) read the same pages: where the count allows, they go to one XCD (ids round-robin over 8) and meet in
    // its L2.  Late query tiles see the most positions and come first.
    const int per = p.q_tiles * p.n_splits, pairs = p.r.B * p.r.Hkv;
    int pair, w;
    if (pairs % 8 == 0) {
        const int j = blockIdx.x >> 3;
        pair = (j / per) * 8 + (blockIdx.x & 7);
        w = j % per;
    } else {
        pair = blockIdx.x / per;
        w = blockIdx.x % per;
    }
    const int b = session_by_length(p, pair / p.r.Hkv, lane), hk = pair % p.r.Hkv, split = w % p.n_splits, vr0 = (p.q_tiles - 1 - w / p.n_splits) * 4 * RW;
    Span sp, sw;
    if (!tile_span(p, b, vr0, 4 * RW, sp)) return;
    if (p.n_splits > 1 && vr0 == 0 && split == 0 && hk == 0) leave_rows(p, sp);
    if (!tile_span(p, b, vr0 + wave * RW, RW, sw)) sw.lo = sw.hi = sw.lo_all = sw.hi_all = 0;      // no rows: help with the tiles only
    const int nvr = sp.n * p.G;
    const int k0 = (sp.lo & ~63) + split * p.chunk, k1 = min(sp.hi, k0 + p.chunk);

    const int ps_mask = (1 << p.r.ps_log2) - 1;
    int page = k0 < k1 ? page_raw(p.r, b, k0) : -1, next = k0 + TK < k1 ? page_raw(p.r, b, k0 + TK) : -1, cur = 0;
    CodeRegs<D> regs;
    const LdsOff<KIND, D> off(l15, g);
    const TileDma<KIND == KV_INT4 ? KV_BF16 : KIND, D> dma(tid, p.r.ps_log2);
    if constexpr (KIND == KV_INT4) {               // codes of tile t + 1 are in registers when tile t is begun
        if (page_ok(p.r, page)) regs.load(p, page, hk, k0 & ps_mask, tid);
    } else if (page_ok(p.r, page)) {
        dma.start(p, lds, page, hk, k0 & ps_mask, wave);
    }

    frag_t q[NC][NS];                              // (behind the first tile's loads, so that they are on their way while it is waited for)
    float sc[NC], m[NC], l[NC];
    int c_lo[NC], c_hi[NC];
    f32x4_t acc[NC][ND];
#pragma unroll
    for (int c = 0; c < NC; ++c) {                 // a column behind the last (row, head) does the last one's work again and stores nothing
        const int vr = min(vr0 + wave * RW + c * 16 + l15, nvr - 1), t = row_of(p, vr), h = hk * p.G + vr - t * p.G;
        load_query<KIND, D>((const T*)p.q + (sp.row0 + (long)t) * p.q_rs + (long)h * D, p.q_vec, p.q_mul, g, q[c], sc[c]);
        sc[c] = score_scale<KIND>(p, sc[c]);
        c_hi[c] = p.causal ? min(sp.len, sp.past + t + 1) : sp.len;
        c_lo[c] = p.window > 0 ? sp.past + t + 1 - p.window : 0;
        m[c] = NO_MAX;
        l[c] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[c][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    if constexpr (KIND == KV_INT4) {
        if (page_ok(p.r, page)) regs.store(lds, tid);
        if (page_ok(p.r, next)) regs.load(p, next, hk, (k0 + TK) & ps_mask, tid);
    }
    for (int kb = k0; kb < k1; kb += TK) {
        __builtin_amdgcn_s_waitcnt(0);             // this wave's part of the tile has landed (loads to LDS count as loads, not as LDS writes)
        __syncthreads();                           // everyone's has, and everyone is done with the other buffer
        unsigned char* buf = lds + cur * L::BYTES;
        unsigned char* other = lds + (cur ^ 1) * L::BYTES;
        const int after = kb + 2 * TK < k1 ? page_raw(p.r, b, kb + 2 * TK) : -1;
        if constexpr (KIND == KV_INT4) {
            if (page_ok(p.r, next)) regs.store(other, tid);
            if (page_ok(p.r, after)) regs.load(p, after, hk, (kb + 2 * TK) & ps_mask, tid);
        } else if (page_ok(p.r, next)) {
            dma.start(p, other, next, hk, (kb + TK) & ps_mask, wave);
        }
        if (kb < sp.lo || kb + TK > sp.hi) {       // the first and last tile: values nobody attends to become 0 where they lie
            for (int i = tid; i < D * TK / 8; i += 256) {
                const int d = i / (TK / 8), o = i % (TK / 8);
                frag_t* v = reinterpret_cast<frag_t*>(buf + L::v_at(d, o));
                *v = OctetBits<frag_t>(kb + o * 8, sp.lo, sp.hi).keep(*v);
            }
            __syncthreads();
        }
        if (page_ok(p.r, page) && kb < sw.hi && kb + TK > sw.lo)
            tile_step<KIND, D, NC>(buf, off, q, sc, kb < sw.lo_all || kb + TK > sw.hi_all, kb + g * 8 * U, c_lo, c_hi, m, l, acc);
        page = next;
        next = after;
        cur ^= 1;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int vr = vr0 + wave * RW + c * 16 + l15;
        l[c] += __shfl_xor(l[c], 16, 64);
        l[c] += __shfl_xor(l[c], 32, 64);
        if (vr >= nvr) continue;
        const int t = row_of(p, vr), h = hk * p.G + vr - t * p.G;
        const float inv = l[c] > 0.f ? 1.f / l[c] : 0.f;
        const bool none = l[c] == 0.f;
        const long row = sp.row0 + (long)t;
        if (p.n_splits == 1) {
            T* o = (T*)p.o + row * p.o_rs + (long)h * D + g * 4;
#pragma unroll
            for (int d = 0; d < ND; ++d) store4(o + d * 16, none ? f32x4_t{0.f, 0.f, 0.f, 0.f} : acc[c][d] * inv, p.o_vec);
        } else {
            const long at = ((long)split * p.r.T + row) * p.H + h;
            if (g == 0) p.plse[at] = none ? -INFINITY : m[c] + __builtin_amdgcn_logf(l[c]);
            if (none) continue;
#pragma unroll
            for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4_t*>(p.po + at * D + d * 16 + g * 4) = acc[c][d] * inv;
        }
    }
}

// ---- the splits' partial results of one (row, head) -> its output -------------------------------------------------------------------------------
// WAVES waves each: wave w adds the splits w, w + WAVES, ... in order, the sums meet in LDS.  Bound by the latency of its loads where there are many splits
// (4 waves), by their bytes where there are many rows (one wave, 4 rows a workgroup).
template <typename T, int D, int WAVES>
__global__ __launch_bounds__(256) void attn_paged_join_kernel(PagedAttn p) {
    constexpr int E = D / 64;
    __shared__ float so[WAVES == 4 ? 3 : 1][D], sl[4];
    typedef float vec_t __attribute__((ext_vector_type(E)));
    const int lane = threadIdx.x & 63, wave = WAVES == 4 ? threadIdx.x >> 6 : 0;
    const long n = (long)p.r.T * p.H, i = WAVES == 4 ? blockIdx.x : (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= n) return;
    const int row = (int)(i / p.H), h = (int)(i - (long)row * p.H);
    if (p.r.cu && (row < p.r.cu[0] || row >= p.r.cu[p.r.B])) return;
    float M = NO_MAX;
    for (int s = lane; s < p.n_splits; s += 64) M = fmaxf(M, p.plse[s * n + i]);
    M = wave_max(M);
    if (M == INFINITY) return;              // not computed: see leave_rows (the same in all waves of a row)
    float acc[E], L = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (int s = wave; s < p.n_splits; s += WAVES) {
        const float lse = p.plse[s * n + i];
        if (lse == -INFINITY) continue;     // nothing was written for it
        const float w = __builtin_amdgcn_exp2f(lse - M);
        L += w;
        const vec_t v = *reinterpret_cast<const vec_t*>(p.po + (s * n + i) * D + lane * E);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(w, ((const float*)&v)[e], acc[e]);
    }
    if constexpr (WAVES == 4) {
        if (lane == 0) sl[wave] = L;
        if (wave)
#pragma unroll
            for (int e = 0; e < E; ++e) so[wave - 1][lane * E + e] = acc[e];
        __syncthreads();
        if (wave) return;
        L = sl[0] + sl[1] + sl[2] + sl[3];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += so[0][lane * E + e] + so[1][lane * E + e] + so[2][lane * E + e];
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    T* o = (T*)p.o + row * p.o_rs + (long)h * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) Elem<T>::st(o + e, L == 0.f ? 0.f : acc[e] * inv);
}

// ---- host side -------------------------------------------------------------------------------------------------------------------------------
struct PagedPlan {
    int n_splits, chunk, q_tiles;
    bool tile;                    // attn_paged_tile_kernel
};
constexpr int tile_nc(int D) { return D == 256 ? 1 : 2; }           // 256 channels: what the registers hold
// Which kernel, how many query tiles and splits: enough workgroups to fill the CUs.
static PagedPlan paged_plan(const s2s_paged_kv* kv, int H, int B, int max_new, int max_kv, int causal, int window) {
    PagedPlan pl;
    const int G = H / kv->kv_heads;
    // The step kernel reads the pages again for every 16 rows; the tile kernel reads them once for 128 but leaves waves without rows idle and needs a barrier per
    // tile.  Above 64 rows the second wins everywhere, up to 16 the first; in between it goes by how many (session, KV head) pairs there are to hide
    // latencies behind.  us, step / tile: 24 rows, 128 pairs, 1500 positions, 128 channels: bf16 39 / 25, 4 bits 23 / 26, f32 69 / 85; 32 rows, 512
    // pairs: bf16 116 / 73, 4 bits 52 / 47; 40 rows, 4 pairs, 4000 positions of 64 channels: bf16 9.8 / 11.1, 4 bits 9.0 / 12.5, f32 15 / 26.
    const long rows_max = (long)max_new * G, pairs = (long)B * kv->kv_heads;
    pl.tile = rows_max > 64 || (rows_max > 16 && pairs >= (paged_kind(kv) == KV_BF16 ? 64 : 256));
    const int rows = pl.tile ? 4 * 16 * tile_nc(kv->head_dim) : 16;
    pl.q_tiles = cdiv(rows_max, rows);
    const long span = causal && window > 0 ? std::min<long>(max_kv, (long)window + cdiv(rows - 1, G) + 1 + 63) + 63 : max_kv;      // from a multiple of 64
    const long groups = pairs * pl.q_tiles;
    if (pl.tile) {
        // A split shortens the walk and costs a second launch and f32 partial rows, written and read: the number with the least time wins, in us of 128 rows
        // of 128 channels.  A tile of 64 positions takes 1.25 (bf16), 1.6 (4 bits), 8.2 (f32); two workgroups on a CU take 1.65 (bf16: 2) times as long where all
        // sessions have the same length and less in ragged batches, hence 1.5; the join takes 4.3 + 0.03 a workgroup.  Measured for 1 / 2 / 4 / 8 splits: bf16, 64
        // workgroups, 32 tiles 47 / 34 / 28 / 32; 128 and 32 48 / 40 / 42 / 57; 256 and 8 20 / 37 / 50; 256 and 64 121 / 132, ragged 85 / 75; 4 bits, 128 and
        // 64 107 / 71 / 62 / 73; 256 and 64 109 / 101, ragged 98 / 79; f32, 64 and 16 147 / 86 / 56 / 57.
        const float size = (float)(rows * kv->head_dim) / (128 * 128), fill = (float)rows_max / (float)(pl.q_tiles * rows);
        const int kind = paged_kind(kv);
        const float tile_us = (kind == KV_F32 ? 8.2f : kind == KV_BF16 ? 1.25f : 1.6f) * size, crowd = 1.5f;
        const int tiles = std::max(1, cdiv(span, 64));
        float best = 3e38f;
        int per = tiles;
        for (int n = 1; n == 1 || (n * groups <= 512 && 2 * n <= tiles); n *= 2) {
            const int each = cdiv(tiles, n);
            const float us = tile_us * (float)each * (n * groups > 256 ? crowd : 1.f) + (n > 1 ? 4.3f + 0.03f * size * fill * (float)(n * groups) : 0.f);
            if (us < best) best = us, per = each;
        }
        pl.chunk = per * 64;
    } else {
        const long want = std::max<long>(1, 1024 / std::max<long>(1, groups));
        // a split is a tile for every wave at least; where one split of 256 positions does, the second launch costs more than it saves
        const int least = 4 * 32 * tile_u(paged_kind(kv), kv->head_dim);
        pl.chunk = span <= 256 ? 256 : std::max(least, cdiv(cdiv(span, want), least) * least);
    }
    pl.n_splits = std::max(1, cdiv(span, pl.chunk));
    if (pl.n_splits == 1) pl.chunk = 1 << 30;
    return pl;
}

constexpr int64_t MAX_GROUPS = 1 << 24;       // a launch has fewer than 2^32 work-items along a dimension

template <typename T, int KIND, int D> static void attn_launch(hipStream_t st, PagedAttn& p) {
    // Sessions in the order of their lengths: where CUs get more than one workgroup and walks are long.  us without / with, lengths spread evenly up to the given one:
    // 512 workgroups, 128 positions 17.5 / 19.2, 512: 28.0 / 29.1, 1024: 39.0 / 38.5 (4 bits 42 / 39), 2048: 73 / 66 (75 / 63); 64 workgroups: 0.3 - 1 slower throughout.
    p.by_length = p.r.B <= 64 && (long)p.q_tiles * p.n_splits * p.r.Hkv * p.r.B > 256 && std::min(p.max_kv, p.chunk) >= 1024;
    if (p.tile) attn_paged_tile_kernel<KIND, D, tile_nc(D)><<<dim3(p.q_tiles * p.n_splits * p.r.Hkv * p.r.B), 256, 0, st>>>(p);
    else attn_paged_step_kernel<KIND, D><<<dim3(p.q_tiles * p.n_splits, p.r.Hkv, p.r.B), 256, 0, st>>>(p);
    if (p.n_splits > 8 && (long)p.r.T * p.H < MAX_GROUPS) attn_paged_join_kernel<T, D, 4><<<dim3(p.r.T * p.H), 256, 0, st>>>(p);
    else if (p.n_splits > 1) attn_paged_join_kernel<T, D, 1><<<cdiv((long)p.r.T * p.H, 4), 256, 0, st>>>(p);
}

}  // namespace s2s

using namespace s2s;

static int attn_paged_sizes(const s2s_paged_kv* kv, int H, int B, int T, int max_new, int max_kv, int causal, int window) {
    if (const int rc = paged_check(kv, "attn_paged")) return rc;
    S2S_REQUIRE(H >= 1 && H <= 4096 && H % kv->kv_heads == 0, "attn_paged: %d query heads over %d KV heads", H, kv->kv_heads);
    S2S_REQUIRE(B >= 0 && B <= 65535 && T >= 0 && max_new >= 1, "attn_paged: B=%d T=%d max_new=%d", B, T, max_new);
    S2S_REQUIRE(max_kv >= 0 && max_kv <= 1 << 30, "attn_paged: max_kv=%d", max_kv);
    S2S_REQUIRE(window >= 0 && (window == 0 || causal), "attn_paged: a window (%d) needs the causal mask", window);
    S2S_REQUIRE((int64_t)T * H < (1LL << 31), "attn_paged: %d rows of %d heads are too many for one call", T, H);
    if (B == 0 || T == 0) return S2S_OK;
    const PagedPlan pl = paged_plan(kv, H, B, std::min(max_new, T), max_kv, causal, window);
    const int64_t groups = (int64_t)pl.q_tiles * pl.n_splits * (pl.tile ? (int64_t)kv->kv_heads * B : 1);     // (the step kernel's heads and sessions lie along others)
    S2S_REQUIRE(groups < MAX_GROUPS, "attn_paged: %d sessions of up to %d rows are too many for one call", B, max_new);
    S2S_REQUIRE(pl.n_splits == 1 || cdiv((int64_t)T * H, 4) < MAX_GROUPS, "attn_paged: %d rows of %d heads are too many for one call", T, H);
    return S2S_OK;
}

extern "C" int64_t s2s_op_attn_paged_ws(const s2s_paged_kv* kv, int32_t H, int32_t B, int32_t T, int32_t max_new, int32_t max_kv, int32_t causal, int32_t window) {
    if (const int rc = attn_paged_sizes(kv, H, B, T, max_new, max_kv, causal, window)) return rc;
    if (B == 0 || T == 0) return 0;
    const PagedPlan pl = paged_plan(kv, H, B, std::min(max_new, T), max_kv, causal, window);
    return pl.n_splits == 1 ? 0 : (int64_t)pl.n_splits * T * H * (kv->head_dim + 1) * 4;
}

extern "C" int32_t s2s_op_attn_paged(void* stream, const s2s_paged_kv* kv, const void* q, int64_t q_rs, void* o, int64_t o_rs, int32_t H, const int32_t* table_dev,
                                     int32_t table_cols, const int32_t* kv_len_dev, const int32_t* cu_dev, int32_t B, int32_t T, int32_t max_new, int32_t max_kv,
                                     float scale, int32_t causal, int32_t window, void* ws_dev, int64_t ws_bytes) {
    int rc = attn_paged_sizes(kv, H, B, T, max_new, max_kv, causal, window);
    if (rc) return rc;
    PagedAttn p{};
    if ((rc = paged_rows(p.r, kv, table_dev, table_cols, cu_dev, B, T, max_new, "attn_paged"))) return rc;
    const float scale_log2e = fabsf(scale) * 1.44269504088896340736f;
    S2S_REQUIRE(scale_log2e < INFINITY, "attn_paged: scale %g is not finite in units of log2", (double)scale);       // (NaN too)
    S2S_REQUIRE(max_kv <= table_cols * kv->page_size, "attn_paged: max_kv=%d of %d pages per session", max_kv, table_cols);
    if (B == 0 || T == 0) return S2S_OK;
    S2S_REQUIRE(q && o && kv_len_dev, "attn_paged: null buffer");
    S2S_REQUIRE(rows_apart(T, o_rs, (int64_t)H * kv->head_dim), "attn_paged: rows of o share memory (stride %lld)", (long long)o_rs);
    const PagedPlan pl = paged_plan(kv, H, B, p.r.max_new, max_kv, causal, window);
    const int64_t need = pl.n_splits == 1 ? 0 : (int64_t)pl.n_splits * T * H * (kv->head_dim + 1) * 4;
    S2S_REQUIRE(need == 0 || (ws_dev && ws_bytes >= need && !((uintptr_t)ws_dev & 15)), "attn_paged: workspace of %lld bytes, 16-byte aligned, needed (got %lld)",
                (long long)need, (long long)ws_bytes);
    p.kc = kv->k; p.vc = kv->v; p.km = (const _Float16*)kv->k_meta; p.vm = (const _Float16*)kv->v_meta;
    p.q = q; p.q_rs = q_rs; p.o = o; p.o_rs = o_rs; p.kv_len = kv_len_dev;
    const int es = kv->dtype == S2S_F32 ? 4 : 2;
    p.q_vec = !((uintptr_t)q & 15) && (q_rs * es) % 16 == 0;
    p.o_vec = !((uintptr_t)o & 15) && (o_rs * es) % 16 == 0;
    p.H = H; p.G = H / kv->kv_heads;
    // quotients by multiplication: 2^32 / G + 1 is right up to vr G < 2^32
    p.g_magic = p.G > 1 && (int64_t)p.r.max_new * p.G * p.G < (1LL << 32) ? (unsigned)((1ULL << 32) / p.G + 1) : 0u;
    p.max_kv = max_kv; p.causal = causal != 0; p.window = std::min(window, 1 << 30);      // no cache is longer, and differences stay inside 32 bits
    p.q_mul = scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f;
    p.scale_log2e = scale == 0.f ? 1.f : scale_log2e;
    p.n_splits = pl.n_splits; p.chunk = pl.chunk; p.q_tiles = pl.q_tiles; p.tile = pl.tile;
    p.po = (float*)ws_dev;
    p.plse = p.po + (int64_t)pl.n_splits * T * H * kv->head_dim;
    S2S_PAGED_DISPATCH(attn_launch, (hipStream_t)stream, p);
    S2S_LAUNCH_CHECK();
    return S2S_OK;
}
