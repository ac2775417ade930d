// Rotary positions, and rows into and out of the paged key / value cache (layout: paged.h, include/s2s_mi355x.h).
//
// All of it is data movement: a row is read once, turned in registers and written once, 8 neighbouring channels (an octet) per lane and
// request.  Every product and sum of a rotation is rounded on its own (no contraction), so that a row turned here, in the append and in plain
// f32 arithmetic is the same row, and a 4-bit code next to a border falls on the same side.
#include "paged.h"

namespace s2s {

// ---- octets ------------------------------------------------------------------------------------------------------------------------------
template <typename T> struct Oct { u32x4_t w[sizeof(T) / 2]; };

template <typename T, bool VEC> __device__ __forceinline__ void oct_load(Oct<T>& o, const T* p) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) o.w[i] = reinterpret_cast<const u32x4_t*>(p)[i];
    } else {
        T e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = p[i];
        __builtin_memcpy(&o, e, sizeof(o));
    }
}
template <typename T, bool VEC> __device__ __forceinline__ void oct_store(T* p, const Oct<T>& o) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) reinterpret_cast<u32x4_t*>(p)[i] = o.w[i];
    } else {
        T e[8];
        __builtin_memcpy(e, &o, sizeof(o));
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = e[i];
    }
}
// for rows nobody reads before they have left the caches
template <typename T, bool VEC> __device__ __forceinline__ void oct_store_nt(T* p, const Oct<T>& o) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) __builtin_nontemporal_store(o.w[i], reinterpret_cast<u32x4_t*>(p) + i);
    } else {
        oct_store<T, VEC>(p, o);
    }
}
__device__ __forceinline__ float oct_get(const Oct<float>& o, int i) { return __uint_as_float(o.w[i >> 2][i & 3]); }
__device__ __forceinline__ float oct_get(const Oct<__hip_bfloat16>& o, int i) {
    const unsigned w = o.w[0][i >> 1];
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
}
__device__ __forceinline__ void oct_put(Oct<float>& o, const float (&y)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o.w[i >> 2][i & 3] = __float_as_uint(y[i]);
}
__device__ __forceinline__ void oct_put(Oct<__hip_bfloat16>& o, const float (&y)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o.w[0][i] = pack_bf16x2_hw(y[2 * i], y[2 * i + 1]);
}

// ---- rotation ----------------------------------------------------------------------------------------------------------------------------
struct Turn {
    const float *cosT, *sinT;     // [max_pos][rot / 2], null: rows pass
    int max_pos, rot;
    bool inter;
};
__device__ __forceinline__ float turn_a(float a, float b, float c, float s) { return __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)); }
__device__ __forceinline__ float turn_b(float a, float b, float c, float s) { return __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s)); }

// octet o of a row turned to `pos`, from the source row (a lane reads the octet its channels are paired with again: the row is in L1)
template <typename T, bool VEC>
__device__ __forceinline__ void turned_octet(const T* row, int o, const Turn& t, int pos, float (&y)[8]) {
    Oct<T> x;
    oct_load<T, VEC>(x, row + 8 * o);
    const int half = t.rot >> 1;
    if (!t.cosT || 8 * o >= t.rot) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = oct_get(x, i);
        return;
    }
    if ((unsigned)pos >= (unsigned)t.max_pos) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = 8 * o + i < t.rot ? __builtin_nanf("") : oct_get(x, i);
        return;
    }
    const float* c = t.cosT + (long)pos * half;
    const float* s = t.sinT + (long)pos * half;
    if constexpr (VEC) {           // rot % 16 == 0: an octet lies in one half, tables are read in fours
        if (t.inter) {
            const float4 cc = *reinterpret_cast<const float4*>(c + 4 * o), ss = *reinterpret_cast<const float4*>(s + 4 * o);
            const float cv[4] = {cc.x, cc.y, cc.z, cc.w}, sv[4] = {ss.x, ss.y, ss.z, ss.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = oct_get(x, 2 * i), b = oct_get(x, 2 * i + 1);
                y[2 * i] = turn_a(a, b, cv[i], sv[i]);
                y[2 * i + 1] = turn_b(a, b, cv[i], sv[i]);
            }
        } else {
            const bool first = 8 * o < half;
            const int j = first ? 8 * o : 8 * o - half;
            Oct<T> p;
            oct_load<T, VEC>(p, row + (first ? j + half : j));
            Oct<float> cc, ss;
            oct_load<float, true>(cc, c + j);
            oct_load<float, true>(ss, s + j);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float xi = oct_get(x, i), pi = oct_get(p, i), ci = oct_get(cc, i), si = oct_get(ss, i);
                y[i] = first ? turn_a(xi, pi, ci, si) : turn_b(pi, xi, ci, si);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = 8 * o + i;
            const float xi = oct_get(x, i);
            if (d >= t.rot) {
                y[i] = xi;
            } else if (t.inter) {
                const float pi = Elem<T>::ld(row + (d ^ 1));
                y[i] = d & 1 ? turn_b(pi, xi, c[d >> 1], s[d >> 1]) : turn_a(xi, pi, c[d >> 1], s[d >> 1]);
            } else {
                const bool first = d < half;
                const float pi = Elem<T>::ld(row + (first ? d + half : d - half));
                y[i] = first ? turn_a(xi, pi, c[d], s[d]) : turn_b(pi, xi, c[d - half], s[d - half]);
            }
        }
    }
}

// 16 bytes of a row: 8 bf16 or 4 f32
template <typename T> struct Piece {
    static constexpr int E = 16 / sizeof(T);
    u32x4_t w;
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    }
    __device__ __forceinline__ void put(const float (&y)[E]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(y[i]);
            else w[i] = pack_bf16x2_hw(y[2 * i], y[2 * i + 1]);
        }
    }
    template <bool STREAM> __device__ __forceinline__ void store(T* p) const {
        if constexpr (STREAM) __builtin_nontemporal_store(w, reinterpret_cast<u32x4_t*>(p));
        else *reinterpret_cast<u32x4_t*>(p) = w;
    }
};

// One unit of NH heads of one row: the channels that turn together are read before any is written, so that out may be x, and the table's values stay in
// registers over the heads.  VEC units: half layout, two pieces, piece u and its partner half a rotation on; interleaved, one piece; then what passes, in
// the same numbers of pieces and on the same path, so that lanes that turn and lanes that pass share their loads.  Else channel pairs, then single
// channels that pass.  STREAM: rows of a prompt are more than the caches hold until somebody reads them, and stores that do not stay there leave
// them to the loads (20011 f32 rows of 20 heads of 128: 95.4 -> 91.0 us).
template <typename T, bool VEC, int NH, bool STREAM>
__device__ __forceinline__ void turn_heads(const T* x, long x_hs, T* out, long o_hs, int heads, int u, const Turn& t, int pos, int D) {
    const int half = t.rot >> 1;
    const bool bad = pos >= t.max_pos;
    const float nan = __builtin_nanf("");
    const long tp = bad ? 0 : (long)pos * half;
    if constexpr (VEC) {
        constexpr int E = Piece<T>::E;
        const int turning = t.inter ? t.rot / E : half / E;
        const bool pass = u >= turning;
        if (pass && out == x) return;
        Piece<T> a[NH], b[NH];
        if (t.inter) {
            const int d = E * u;
            float cv[E / 2], sv[E / 2];
#pragma unroll
            for (int i = 0; i < E / 2; i += 2) {       // (a unit that passes reads the table's first entries)
                const float2 c = *reinterpret_cast<const float2*>(t.cosT + tp + (pass ? 0 : d / 2) + i), s = *reinterpret_cast<const float2*>(t.sinT + tp + (pass ? 0 : d / 2) + i);
                cv[i] = bad ? nan : c.x;
                cv[i + 1] = bad ? nan : c.y;
                sv[i] = s.x;
                sv[i + 1] = s.y;
            }
#pragma unroll
            for (int h = 0; h < NH; ++h)
                if (h < heads) a[h].w = *reinterpret_cast<const u32x4_t*>(x + h * x_hs + d);
#pragma unroll
            for (int h = 0; h < NH; ++h)
                if (h < heads) {
                    float y[E];
#pragma unroll
                    for (int i = 0; i < E / 2; ++i) {
                        const float p = a[h].get(2 * i), q = a[h].get(2 * i + 1);
                        y[2 * i] = turn_a(p, q, cv[i], sv[i]);
                        y[2 * i + 1] = turn_b(p, q, cv[i], sv[i]);
                    }
                    if (!pass) a[h].put(y);
                    a[h].template store<STREAM>(out + h * o_hs + d);
                }
        } else {
            const int d = pass ? t.rot + 2 * E * (u - turning) : E * u, d1 = pass ? min(d + E, D - E) : d + half, dt = pass ? 0 : d;
            float cv[E], sv[E];
#pragma unroll
            for (int i = 0; i < E; i += 4) {
                const float4 c = *reinterpret_cast<const float4*>(t.cosT + tp + dt + i), s = *reinterpret_cast<const float4*>(t.sinT + tp + dt + i);
                cv[i] = bad ? nan : c.x;
                cv[i + 1] = bad ? nan : c.y;
                cv[i + 2] = bad ? nan : c.z;
                cv[i + 3] = bad ? nan : c.w;
                sv[i] = s.x;
                sv[i + 1] = s.y;
                sv[i + 2] = s.z;
                sv[i + 3] = s.w;
            }
#pragma unroll
            for (int h = 0; h < NH; ++h)
                if (h < heads) {
                    a[h].w = *reinterpret_cast<const u32x4_t*>(x + h * x_hs + d);
                    b[h].w = *reinterpret_cast<const u32x4_t*>(x + h * x_hs + d1);
                }
#pragma unroll
            for (int h = 0; h < NH; ++h)
                if (h < heads) {
                    float ya[E], yb[E];
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        const float p = a[h].get(i), q = b[h].get(i);
                        ya[i] = turn_a(p, q, cv[i], sv[i]);
                        yb[i] = turn_b(p, q, cv[i], sv[i]);
                    }
                    if (!pass) {
                        a[h].put(ya);
                        b[h].put(yb);
                    }
                    a[h].template store<STREAM>(out + h * o_hs + d);
                    b[h].template store<STREAM>(out + h * o_hs + d1);
                }
        }
    } else {
        if (u >= half) {
            const int d = t.rot + (u - half);
#pragma unroll
            for (int h = 0; h < NH; ++h)
                if (h < heads) out[h * o_hs + d] = x[h * x_hs + d];
            return;
        }
        const int d0 = t.inter ? 2 * u : u, d1 = t.inter ? 2 * u + 1 : u + half;
        const float c = bad ? nan : t.cosT[tp + u], s = t.sinT[tp + u];
#pragma unroll
        for (int h = 0; h < NH; ++h)
            if (h < heads) {
                const float a = Elem<T>::ld(x + h * x_hs + d0), b = Elem<T>::ld(x + h * x_hs + d1);
                Elem<T>::st(out + h * o_hs + d0, turn_a(a, b, c, s));
                Elem<T>::st(out + h * o_hs + d1, turn_b(a, b, c, s));
            }
    }
}
inline int turn_units(bool vec, bool inter, int rot, int D, int es) {
    const int E = 16 / es;
    return !vec ? rot / 2 + (D - rot) : inter ? D / E : rot / 2 / E + (D - rot + 2 * E - 1) / (2 * E);
}

struct RopeParams {
    const void* x; void* out;
    long x_rs, x_hs, o_rs, o_hs;
    const int* pos;
    Turn t;
    int rows, heads, units, D;
};
template <typename T, bool VEC, int NH> __global__ __launch_bounds__(256) void rope_kernel(RopeParams p) {
    const unsigned idx = blockIdx.x * 256u + threadIdx.x;
    const unsigned r = idx / (unsigned)p.units, u = idx - r * (unsigned)p.units;
    if (r >= (unsigned)p.rows) return;
    const int pos = p.pos[r], h0 = blockIdx.y * NH;
    if (pos < 0) return;
    turn_heads<T, VEC, NH, NH == 4>((const T*)p.x + (long)r * p.x_rs + h0 * p.x_hs, p.x_hs, (T*)p.out + (long)r * p.o_rs + h0 * p.o_hs, p.o_hs, min(NH, p.heads - h0), (int)u, p.t,
                           pos, p.D);
}

// ---- 4-bit groups --------------------------------------------------------------------------------------------------------------------------
// Scale and zero of the 32 values that 4 neighbouring lanes hold (8 each), and the values cut to the range.  Every step in f32, rounded to f16 where
// the format rounds.
__device__ __forceinline__ void group_range(float (&x)[8], _Float16& scale, _Float16& zero) {
    float lo = INFINITY, hi = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        bad |= !(fabsf(x[i]) < INFINITY);
        x[i] = fminf(fmaxf(x[i], -32768.f), 32768.f);
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
    }
    int b = bad;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, o, 64));
        hi = fmaxf(hi, __shfl_xor(hi, o, 64));
        b |= __shfl_xor(b, o, 64);
    }
    scale = b ? (_Float16)0.f : (_Float16)__fdiv_rn(__fsub_rn(hi, lo), 15.f);
    zero = b ? (_Float16)__builtin_nanf("") : (_Float16)__fadd_rn(lo, 8.f * (float)scale);
}
__device__ __forceinline__ unsigned code_of(float x, float scale, float zero) {
    if (!(scale > 0.f)) return 8u;
    return (unsigned)(fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x, zero), scale)) + 8.f, 0.f), 15.f));
}
__device__ __forceinline__ float value_of(unsigned code, float scale, float zero) { return __fadd_rn(zero, __fmul_rn(scale, (float)code - 8.f)); }
__device__ __forceinline__ unsigned meta_word(_Float16 scale, _Float16 zero) {
    return (unsigned)__builtin_bit_cast(unsigned short, scale) | (unsigned)__builtin_bit_cast(unsigned short, zero) << 16;
}

// ---- append --------------------------------------------------------------------------------------------------------------------------------
struct AppendParams {
    PagedRows r;
    Turn t;
    void *kc, *vc;
    _Float16 *km, *vm;
    const void *k, *v, *q;
    void* qo;
    long k_rs, v_rs, q_rs, qo_rs;
    const int* start;
    int H;            // query heads (0: none)
    int units;        // of turn_heads
};

// key octet o of head h into its page
template <typename T, int KIND, int D>
__device__ __forceinline__ void put_key(const AppendParams& p, int page, int h, int at, int o, float (&y)[8]) {
    const long row = (((long)page * p.r.Hkv + h) << p.r.ps_log2) + at;
    Oct<T> x;
    oct_put(x, y);
    if constexpr (KIND != KV_INT4) {
        oct_store<T, true>((T*)p.kc + row * D + 8 * o, x);
    } else {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = oct_get(x, i);
        _Float16 scale, zero;
        group_range(v, scale, zero);
        unsigned w = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) w |= code_of(v[i], (float)scale, (float)zero) << (4 * code_nibble(i));
        const int s = o >> 2, g = o & 3;
        reinterpret_cast<unsigned*>(p.kc)[row * (D / 8) + g * (D / 32) + s] = w;
        if (g == 0) reinterpret_cast<unsigned*>(p.km)[row * (D / 32) + s] = meta_word(scale, zero);
    }
}

// One new row per session (a decode step): D / 8 lanes per row of a head, tasks = KV heads' keys, their values, query heads.  Bound by latency and by
// the values' scattered columns (one element, or one nibble, per channel: 64-byte sectors of the transposed page).  64 sessions of 16 / 8 heads of 128, bf16:
// 4.3 us; 512 sessions in 4 bits: 14.0 us, of which the sectors of the value columns (17 MB read, 17 MB written back) are half.
template <typename T, int KIND, int D, bool VEC>
__global__ __launch_bounds__(256) void kv_append_step_kernel(AppendParams p) {
    constexpr int LPT = D / 8;
    const int b = blockIdx.y, task = (blockIdx.x * 256 + threadIdx.x) / LPT, o = threadIdx.x % LPT;
    const int Hkv = p.r.Hkv;
    if (task >= 2 * Hkv + p.H) return;
    int row0, n;
    session_rows(p.r, b, row0, n);
    const int pos = p.start[b];
    if (n <= 0 || row0 >= p.r.T || pos < 0) return;
    if (task >= 2 * Hkv) {         // a lane reads both octets it needs before it writes; the lanes of a row are in one wave: q_out may be q
        const int h = task - 2 * Hkv;
        float y[8];
        turned_octet<T, VEC>((const T*)p.q + (long)row0 * p.q_rs + (long)h * D, o, p.t, pos, y);
        Oct<T> x;
        oct_put(x, y);
        oct_store<T, VEC>((T*)p.qo + (long)row0 * p.qo_rs + (long)h * D + 8 * o, x);
        return;
    }
    const int page = page_of(p.r, b, pos), at = pos & ((1 << p.r.ps_log2) - 1);
    if (page < 0) return;
    if (task < Hkv) {
        float y[8];
        turned_octet<T, VEC>((const T*)p.k + (long)row0 * p.k_rs + (long)task * D, o, p.t, pos, y);
        put_key<T, KIND, D>(p, page, task, at, o, y);
        return;
    }
    const int h = task - Hkv;
    Oct<T> x;
    oct_load<T, VEC>(x, (const T*)p.v + (long)row0 * p.v_rs + (long)h * D + 8 * o);
    const long head = (long)page * Hkv + h;
    if constexpr (KIND != KV_INT4) {
        T* dst = (T*)p.vc + ((head * D + 8 * o) << p.r.ps_log2) + at;
        T e[8];
        __builtin_memcpy(e, &x, sizeof(x));
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[(long)i << p.r.ps_log2] = e[i];
    } else {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = oct_get(x, i);
        _Float16 scale, zero;
        group_range(v, scale, zero);
        const unsigned nib = code_nibble(at & 7);
        unsigned char* dst = (unsigned char*)p.vc + ((head * D + 8 * o) << (p.r.ps_log2 - 1)) + (at >> 3) * 4 + (nib >> 1);
        const int sh = (nib & 1) * 4;
        unsigned char old[8];      // the other nibble is another position of the same session: nobody else writes this byte
#pragma unroll
        for (int i = 0; i < 8; ++i) old[i] = dst[(long)i << (p.r.ps_log2 - 1)];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            dst[(long)i << (p.r.ps_log2 - 1)] = (unsigned char)((old[i] & (0xf0 >> sh)) | code_of(v[i], (float)scale, (float)zero) << sh);
        if ((o & 3) == 0) {
            _Float16* m = p.vm + ((head * (D / 32) + (o >> 2)) * 2 << p.r.ps_log2) + at;
            m[0] = scale;
            m[(long)1 << p.r.ps_log2] = zero;
        }
    }
}

// Rows of a prompt: a workgroup takes the new rows that fall into one run of 64 positions (always inside one page) of: one KV head's keys; 64
// channels of one KV head's values, transposed through LDS so that every channel's positions are written as whole octets; or a query head.  HBM-bound: 25 k rows of
// 16 / 8 heads of 128, bf16: 97 us, 4.5 TB/s; in 4 bits 91 us, 3.8 TB/s (the divisions of the codes are 4 us of it).
template <typename T, int KIND, int D, bool VEC>
__global__ __launch_bounds__(256) void kv_append_block_kernel(AppendParams p) {
    constexpr int LD = sizeof(T) == 2 ? 66 : 65;      // 33 / 65 dwords per row: the column reads of 8 octets hit 4 or more different banks
    __shared__ alignas(16) T tile[64 * LD];
    __shared__ float2 meta[KIND == KV_INT4 ? 64 * 2 : 1];
    const int b = blockIdx.z, tid = threadIdx.x, Hkv = p.r.Hkv;
    int row0, n;
    session_rows(p.r, b, row0, n);
    const int pos0 = p.start[b];
    if (n <= 0 || pos0 < 0 || pos0 > (1 << 30)) return;
    const int base = (pos0 / 64 + (int)blockIdx.x) * 64;
    const int lo = max(pos0, base), hi = min(pos0 + n, base + 64);
    if (lo >= hi) return;
    const int rows = hi - lo;
    const long src0 = row0 + (lo - pos0);             // source row of position lo
    int y = blockIdx.y;
    if (y >= Hkv + Hkv * (D / 64)) {                  // queries
        const long hd = (long)(y - Hkv - Hkv * (D / 64)) * D;
        for (int i = tid; i < rows * p.units; i += 256) {
            const int r = i / p.units, u = i - r * p.units;
            const T* src = (const T*)p.q + (src0 + r) * p.q_rs + hd;
            T* dst = (T*)p.qo + (src0 + r) * p.qo_rs + hd;
            turn_heads<T, VEC, 1, true>(src, D, dst, D, 1, u, p.t, lo + r, D);
        }
        return;
    }
    const int page = page_of(p.r, b, lo), ps_mask = (1 << p.r.ps_log2) - 1;
    if (page < 0) return;
    if (y < Hkv) {                                    // keys
        for (int i = tid; i < rows * (D / 8); i += 256) {
            const int r = i / (D / 8), o = i % (D / 8);
            float v[8];
            turned_octet<T, VEC>((const T*)p.k + (src0 + r) * p.k_rs + (long)y * D, o, p.t, lo + r, v);
            put_key<T, KIND, D>(p, page, y, (lo + r) & ps_mask, o, v);
        }
        return;
    }
    y -= Hkv;
    const int h = y / (D / 64), d0 = (y % (D / 64)) * 64, first = lo - base;      // the tile's rows are positions base ..
    const long head = (long)page * Hkv + h;
    const int at0 = base & ps_mask;
    for (int i = tid; i < rows * 8; i += 256) {
        const int r = i >> 3, o = i & 7;
        Oct<T> x;
        oct_load<T, VEC>(x, (const T*)p.v + (src0 + r) * p.v_rs + (long)h * D + d0 + 8 * o);
        unsigned* dst = reinterpret_cast<unsigned*>(tile + (first + r) * LD + 8 * o);
#pragma unroll
        for (int w = 0; w < (int)sizeof(T) * 2; ++w) dst[w] = x.w[w >> 2][w & 3];
        if constexpr (KIND == KV_INT4) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = oct_get(x, e);
            _Float16 scale, zero;
            group_range(v, scale, zero);
            if ((o & 3) == 0) {
                meta[(first + r) * 2 + (o >> 2)] = make_float2((float)scale, (float)zero);
                _Float16* m = p.vm + ((head * (D / 32) + d0 / 32 + (o >> 2)) * 2 << p.r.ps_log2) + at0 + first + r;
                m[0] = scale;
                m[(long)1 << p.r.ps_log2] = zero;
            }
        }
    }
    __syncthreads();
    const int o_lo = first >> 3, o_hi = (first + rows + 7) >> 3;
    for (int i = tid; i < 64 * 8; i += 256) {
        const int d = i >> 3, o = i & 7;
        if (o < o_lo || o >= o_hi) continue;
        const bool whole = o * 8 >= first && o * 8 + 8 <= first + rows;
        if constexpr (KIND != KV_INT4) {
            T e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = tile[(o * 8 + j) * LD + d];
            T* dst = (T*)p.vc + ((head * D + d0 + d) << p.r.ps_log2) + at0 + o * 8;
            if (whole) {
                Oct<T> x;
                __builtin_memcpy(&x, e, sizeof(x));
                oct_store<T, true>(dst, x);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (o * 8 + j >= first && o * 8 + j < first + rows) dst[j] = e[j];
            }
        } else {
            unsigned w = 0, keep = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = o * 8 + j;
                const unsigned sh = 4 * code_nibble(j);
                if (r >= first && r < first + rows) {
                    const float2 m = meta[r * 2 + (d >> 5)];
                    const float x = fminf(fmaxf(Elem<T>::ld(tile + r * LD + d), -32768.f), 32768.f);
                    w |= code_of(x, m.x, m.y) << sh;
                } else {
                    keep |= 15u << sh;
                }
            }
            unsigned* dst = reinterpret_cast<unsigned*>(p.vc) + ((head * D + d0 + d) << (p.r.ps_log2 - 3)) + (at0 >> 3) + o;
            if (!whole) w |= *dst & keep;
            *dst = w;
        }
    }
}

// ---- rows back out ---------------------------------------------------------------------------------------------------------------------------
struct ReadParams {
    PagedRows r;
    const void *kc, *vc;
    const _Float16 *km, *vm;
    void *ko, *vo;
    long o_rs;
    const int* start;
};

// key octet o of a page's row
template <typename T, int KIND, int D> __device__ __forceinline__ void get_key(const ReadParams& p, long row, int o, Oct<T>& x) {
    if constexpr (KIND != KV_INT4) {
        oct_load<T, true>(x, (const T*)p.kc + row * D + 8 * o);
    } else {
        const int s = o >> 2, g = o & 3;
        const unsigned w = reinterpret_cast<const unsigned*>(p.kc)[row * (D / 8) + g * (D / 32) + s];
        const f16x2_t m = __builtin_bit_cast(f16x2_t, reinterpret_cast<const unsigned*>(p.km)[row * (D / 32) + s]);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = value_of(w >> (4 * code_nibble(j)) & 15, (float)m[0], (float)m[1]);
        oct_put(x, v);
    }
}

// the same runs of 64 positions as the append; values go back through the LDS transpose (25 k rows of 8 heads of 128 out of 4-bit pages: 25 us, 5.4 TB/s)
template <typename T, int KIND, int D, bool VEC>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadParams p) {
    constexpr int LD = sizeof(T) == 2 ? 66 : 65;
    __shared__ alignas(16) T tile[64 * LD];
    const int b = blockIdx.z, tid = threadIdx.x, Hkv = p.r.Hkv;
    int row0, n;
    session_rows(p.r, b, row0, n);
    const int pos0 = p.start[b];
    if (n <= 0 || pos0 < 0 || pos0 > (1 << 30)) return;
    const int base = (pos0 / 64 + (int)blockIdx.x) * 64;
    const int lo = max(pos0, base), hi = min(pos0 + n, base + 64);
    if (lo >= hi) return;
    const int rows = hi - lo, ps_mask = (1 << p.r.ps_log2) - 1, first = lo - base, at0 = base & ps_mask;
    const long dst0 = row0 + (lo - pos0);
    const int page = page_of(p.r, b, lo);
    int y = blockIdx.y;
    if (y < Hkv) {
        if (!p.ko) return;
        for (int i = tid; i < rows * (D / 8); i += 256) {
            const int r = i / (D / 8), o = i % (D / 8);
            const long row = (((long)(page < 0 ? 0 : page) * Hkv + y) << p.r.ps_log2) + at0 + first + r;
            Oct<T> x;
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (page < 0) {
                oct_put(x, v);
            } else {
                get_key<T, KIND, D>(p, row, o, x);
            }
            oct_store_nt<T, VEC>((T*)p.ko + (dst0 + r) * p.o_rs + (long)y * D + 8 * o, x);
        }
        return;
    }
    if (!p.vo) return;
    y -= Hkv;
    const int h = y / (D / 64), d0 = (y % (D / 64)) * 64;
    const long head = (long)(page < 0 ? 0 : page) * Hkv + h;
    const int o_lo = first >> 3, o_hi = (first + rows + 7) >> 3;
    for (int i = tid; i < 64 * 8; i += 256) {
        const int d = i >> 3, o = i & 7;
        if (o < o_lo || o >= o_hi) continue;
        Oct<T> x;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (page < 0) {
            oct_put(x, v);
        } else if constexpr (KIND != KV_INT4) {
            oct_load<T, true>(x, (const T*)p.vc + ((head * D + d0 + d) << p.r.ps_log2) + at0 + o * 8);
        } else {
            const unsigned w = (reinterpret_cast<const unsigned*>(p.vc) + ((head * D + d0 + d) << (p.r.ps_log2 - 3)) + (at0 >> 3))[o];
            const _Float16* m = p.vm + ((head * (D / 32) + (d0 + d) / 32) * 2 << p.r.ps_log2) + at0 + o * 8;
            const f16x8_t scale = *reinterpret_cast<const f16x8_t*>(m), zero = *reinterpret_cast<const f16x8_t*>(m + ((long)1 << p.r.ps_log2));
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = value_of(w >> (4 * code_nibble(j)) & 15, (float)scale[j], (float)zero[j]);
            oct_put(x, v);
        }
        T e[8];
        __builtin_memcpy(e, &x, sizeof(x));
#pragma unroll
        for (int j = 0; j < 8; ++j) tile[(o * 8 + j) * LD + d] = e[j];
    }
    __syncthreads();
    for (int i = tid; i < rows * 8; i += 256) {
        const int r = i >> 3, o = i & 7;
        Oct<T> x;
        const unsigned* src = reinterpret_cast<const unsigned*>(tile + (first + r) * LD + 8 * o);
#pragma unroll
        for (int w = 0; w < (int)sizeof(T) * 2; ++w) x.w[w >> 2][w & 3] = src[w];
        oct_store_nt<T, VEC>((T*)p.vo + (dst0 + r) * p.o_rs + (long)h * D + d0 + 8 * o, x);
    }
}

// one position per session: D / 8 lanes per row of a head, values gathered channel by channel
template <typename T, int KIND, int D, bool VEC>
__global__ __launch_bounds__(256) void kv_read_step_kernel(ReadParams p) {
    constexpr int LPT = D / 8;
    const int b = blockIdx.y, task = (blockIdx.x * 256 + threadIdx.x) / LPT, o = threadIdx.x % LPT, Hkv = p.r.Hkv;
    if (task >= 2 * Hkv || !(task < Hkv ? p.ko : p.vo)) return;
    int row0, n;
    session_rows(p.r, b, row0, n);
    const int pos = p.start[b];
    if (n <= 0 || row0 >= p.r.T || pos < 0 || pos > (1 << 30)) return;
    const int page = page_of(p.r, b, pos), at = pos & ((1 << p.r.ps_log2) - 1), h = task < Hkv ? task : task - Hkv;
    const long head = (long)max(page, 0) * Hkv + h;
    Oct<T> x;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    oct_put(x, v);
    if (page >= 0) {
        if (task < Hkv) {
            get_key<T, KIND, D>(p, (head << p.r.ps_log2) + at, o, x);
        } else if constexpr (KIND != KV_INT4) {
            T e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = ((const T*)p.vc)[((head * D + 8 * o + i) << p.r.ps_log2) + at];
            __builtin_memcpy(&x, e, sizeof(x));
        } else {
            const unsigned nib = code_nibble(at & 7);
            const unsigned char* src = (const unsigned char*)p.vc + ((head * D + 8 * o) << (p.r.ps_log2 - 1)) + (at >> 3) * 4 + (nib >> 1);
            const _Float16* m = p.vm + (((head * (D / 32) + (o >> 2)) * 2) << p.r.ps_log2) + at;
            const float scale = m[0], zero = m[(long)1 << p.r.ps_log2];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = value_of(src[(long)i << (p.r.ps_log2 - 1)] >> (nib & 1) * 4 & 15, scale, zero);
            oct_put(x, v);
        }
    }
    oct_store<T, VEC>((T*)(task < Hkv ? p.ko : p.vo) + (long)row0 * p.o_rs + (long)h * D + 8 * o, x);
}

// ---- host side -------------------------------------------------------------------------------------------------------------------------------
int paged_check(const s2s_paged_kv* kv, const char* who) {
    S2S_REQUIRE(kv, "%s: no cache", who);
    S2S_REQUIRE(kv->dtype == S2S_F32 || kv->dtype == S2S_BF16, "%s: bad dtype %d", who, kv->dtype);
    S2S_REQUIRE(kv->kind == S2S_KV_MODEL || kv->kind == S2S_KV_INT4, "%s: bad cache kind %d", who, kv->kind);
    S2S_REQUIRE(kv->kind == S2S_KV_MODEL || kv->dtype == S2S_BF16, "%s: a 4-bit cache takes bf16 rows", who);
    S2S_REQUIRE(kv->head_dim == 64 || kv->head_dim == 128 || kv->head_dim == 256, "%s: head_dim %d unsupported (64, 128, 256)", who, kv->head_dim);
    S2S_REQUIRE(kv->page_size >= 64 && kv->page_size <= 1024 && !(kv->page_size & (kv->page_size - 1)), "%s: page_size %d is no power of two in 64 .. 1024", who,
                kv->page_size);
    S2S_REQUIRE(kv->n_pages >= 1 && kv->kv_heads >= 1 && kv->kv_heads <= 1024, "%s: %d pages of %d heads", who, kv->n_pages, kv->kv_heads);
    S2S_REQUIRE(kv->k && kv->v && !((uintptr_t)kv->k & 15) && !((uintptr_t)kv->v & 15), "%s: pages are missing or not aligned to 16 bytes", who);
    S2S_REQUIRE(kv->kind == S2S_KV_MODEL || (kv->k_meta && kv->v_meta && !((uintptr_t)kv->k_meta & 15) && !((uintptr_t)kv->v_meta & 15)),
                "%s: a 4-bit cache needs k_meta and v_meta, aligned to 16 bytes", who);
    return S2S_OK;
}

static int log2_of(int x) {
    int l = 0;
    while (1 << l < x) ++l;
    return l;
}

int paged_rows(PagedRows& r, const s2s_paged_kv* kv, const int* table, int cols, const int* cu, int B, int T, int max_new, const char* who) {
    S2S_REQUIRE(B >= 0 && T >= 0 && B <= 65535, "%s: B=%d T=%d", who, B, T);
    S2S_REQUIRE(cu || T == B, "%s: without cu there is one row per session (B=%d, T=%d)", who, B, T);
    S2S_REQUIRE(max_new >= 1 && (cu || max_new == 1), "%s: max_new=%d", who, max_new);
    S2S_REQUIRE(cols >= 1 && (long)cols * kv->page_size <= 1 << 30, "%s: table_cols=%d", who, cols);
    S2S_REQUIRE(B == 0 || table, "%s: no page table", who);
    r = PagedRows{table, cols, cu, B, T, max_new < T ? max_new : (T > 0 ? T : 1), kv->n_pages, log2_of(kv->page_size), kv->kv_heads};
    return S2S_OK;
}

static bool aligned(const void* p, long rs, int es) { return !((uintptr_t)p & 15) && (rs * es) % 16 == 0; }

static int turn_check(const float* cosT, const float* sinT, int max_pos, int rot, int D, const char* who) {
    S2S_REQUIRE(cosT && sinT && max_pos >= 1, "%s: no rotary tables", who);
    S2S_REQUIRE(rot >= 2 && rot <= D && rot % 2 == 0, "%s: rotary_dim %d of head_dim %d", who, rot, D);
    return S2S_OK;
}

template <typename T, int NH>
static void rope_launch(hipStream_t st, const RopeParams& p, bool vec) {
    const dim3 grid(cdiv((long)p.rows * p.units, 256), cdiv(p.heads, NH));
    if (vec) rope_kernel<T, true, NH><<<grid, 256, 0, st>>>(p);
    else rope_kernel<T, false, NH><<<grid, 256, 0, st>>>(p);
}

template <typename T, int KIND, int D>
static void append_launch(hipStream_t st, const AppendParams& p, bool vec) {
    if (p.r.max_new == 1) {
        const dim3 grid(cdiv((long)(2 * p.r.Hkv + p.H) * (D / 8), 256), p.r.B);
        if (vec) kv_append_step_kernel<T, KIND, D, true><<<grid, 256, 0, st>>>(p);
        else kv_append_step_kernel<T, KIND, D, false><<<grid, 256, 0, st>>>(p);
        return;
    }
    const dim3 grid(cdiv((long)p.r.max_new + 63, 64), p.r.Hkv + p.r.Hkv * (D / 64) + p.H, p.r.B);
    if (vec) kv_append_block_kernel<T, KIND, D, true><<<grid, 256, 0, st>>>(p);
    else kv_append_block_kernel<T, KIND, D, false><<<grid, 256, 0, st>>>(p);
}

template <typename T, int KIND, int D>
static void read_launch(hipStream_t st, const ReadParams& p, bool vec) {
    if (p.r.max_new == 1) {
        const dim3 grid(cdiv(2L * p.r.Hkv * (D / 8), 256), p.r.B);
        if (vec) kv_read_step_kernel<T, KIND, D, true><<<grid, 256, 0, st>>>(p);
        else kv_read_step_kernel<T, KIND, D, false><<<grid, 256, 0, st>>>(p);
        return;
    }
    const dim3 grid(cdiv((long)p.r.max_new + 63, 64), p.r.Hkv + p.r.Hkv * (D / 64), p.r.B);
    if (vec) kv_read_kernel<T, KIND, D, true><<<grid, 256, 0, st>>>(p);
    else kv_read_kernel<T, KIND, D, false><<<grid, 256, 0, st>>>(p);
}

}  // namespace s2s

using namespace s2s;

extern "C" int32_t s2s_op_rope(void* stream, const void* x, int64_t x_rs, int64_t x_hs, void* out, int64_t o_rs, int64_t o_hs, const int32_t* positions_dev,
                               const float* cos_dev, const float* sin_dev, int32_t max_pos, int32_t rows, int32_t heads, int32_t head_dim, int32_t rotary_dim,
                               int32_t interleaved, int32_t dtype) {
    S2S_REQUIRE(dtype == S2S_F32 || dtype == S2S_BF16, "rope: bad dtype %d", dtype);
    S2S_REQUIRE(rows >= 0 && heads >= 0 && head_dim >= 2 && head_dim <= 1024 && heads <= 65535, "rope: rows=%d heads=%d head_dim=%d", rows, heads, head_dim);
    if (const int rc = turn_check(cos_dev, sin_dev, max_pos, rotary_dim, head_dim, "rope")) return rc;
    S2S_REQUIRE(x != out || (x_rs == o_rs && x_hs == o_hs), "rope: in place needs the same strides");
    if (rows == 0 || heads == 0) return S2S_OK;
    S2S_REQUIRE(x && out && positions_dev, "rope: null buffer");
    // heads inside rows, or rows inside heads
    S2S_REQUIRE((rows_apart(heads, o_hs, head_dim) && rows_apart(rows, o_rs, (heads - 1) * o_hs + head_dim)) ||
                    (rows_apart(rows, o_rs, head_dim) && rows_apart(heads, o_hs, (rows - 1) * o_rs + head_dim)),
                "rope: rows of out share memory (strides %lld, %lld)", (long long)o_rs, (long long)o_hs);
    const int es = dtype == S2S_F32 ? 4 : 2;
    // octets need 16-byte rows and heads, and a rotation that falls on octets in both halves
    const bool vec = rotary_dim % 16 == 0 && head_dim % 8 == 0 && aligned(x, x_rs, es) && aligned(out, o_rs, es) && (x_hs * es) % 16 == 0 && (o_hs * es) % 16 == 0 &&
                     aligned(cos_dev, 0, 4) && aligned(sin_dev, 0, 4);
    RopeParams p{x, out, x_rs, x_hs, o_rs, o_hs, positions_dev, Turn{cos_dev, sin_dev, max_pos, rotary_dim, interleaved != 0}, rows, heads,
                 turn_units(vec, interleaved != 0, rotary_dim, head_dim, es), head_dim};
    S2S_REQUIRE((long)rows * p.units < (1L << 31), "rope: %d rows of %d units are too many for one call", rows, p.units);
    const bool many = (long)rows * p.units * heads >= 256L * 1024 * 4;     // enough for every CU with 4 heads a thread
    if (dtype == S2S_F32) {
        if (many) rope_launch<float, 4>((hipStream_t)stream, p, vec);
        else rope_launch<float, 1>((hipStream_t)stream, p, vec);
    } else {
        if (many) rope_launch<__hip_bfloat16, 4>((hipStream_t)stream, p, vec);
        else rope_launch<__hip_bfloat16, 1>((hipStream_t)stream, p, vec);
    }
    S2S_LAUNCH_CHECK();
    return S2S_OK;
}

extern "C" int32_t s2s_op_kv_append_paged(void* stream, const s2s_paged_kv* kv, const void* k, int64_t k_rs, const void* v, int64_t v_rs, const void* q, int64_t q_rs,
                                          void* q_out, int64_t qo_rs, int32_t H, const int32_t* table_dev, int32_t table_cols, const int32_t* start_dev,
                                          const int32_t* cu_dev, int32_t B, int32_t T, int32_t max_new, const float* cos_dev, const float* sin_dev, int32_t max_pos,
                                          int32_t rotary_dim, int32_t interleaved) {
    int rc = paged_check(kv, "kv_append_paged");
    if (rc) return rc;
    AppendParams p{};
    if ((rc = paged_rows(p.r, kv, table_dev, table_cols, cu_dev, B, T, max_new, "kv_append_paged"))) return rc;
    if (cos_dev || sin_dev) {
        if ((rc = turn_check(cos_dev, sin_dev, max_pos, rotary_dim, kv->head_dim, "kv_append_paged"))) return rc;
        p.t = Turn{cos_dev, sin_dev, max_pos, rotary_dim, interleaved != 0};
    }
    S2S_REQUIRE(!q || (cos_dev && q_out && H >= 1 && H <= 4096), "kv_append_paged: queries need tables, q_out and 1 .. 4096 heads (H=%d)", H);
    if (B == 0 || T == 0) return S2S_OK;
    S2S_REQUIRE(k && v && start_dev, "kv_append_paged: null buffer");
    S2S_REQUIRE(!q || q != q_out || q_rs == qo_rs, "kv_append_paged: in place needs the same stride");
    S2S_REQUIRE(!q || rows_apart(T, qo_rs, (int64_t)H * kv->head_dim), "kv_append_paged: rows of q_out share memory (stride %lld)", (long long)qo_rs);
    const int es = kv->dtype == S2S_F32 ? 4 : 2;
    const bool vec = aligned(k, k_rs, es) && aligned(v, v_rs, es) && (!q || (aligned(q, q_rs, es) && aligned(q_out, qo_rs, es))) &&
                     (!cos_dev || (rotary_dim % 16 == 0 && aligned(cos_dev, 0, 4) && aligned(sin_dev, 0, 4)));
    p.kc = kv->k; p.vc = kv->v; p.km = (_Float16*)kv->k_meta; p.vm = (_Float16*)kv->v_meta;
    p.k = k; p.k_rs = k_rs; p.v = v; p.v_rs = v_rs; p.q = q; p.q_rs = q_rs; p.qo = q_out; p.qo_rs = qo_rs;
    p.start = start_dev;
    p.H = q ? H : 0;
    p.units = q ? turn_units(vec, p.t.inter, p.t.rot, kv->head_dim, es) : 1;
    S2S_PAGED_DISPATCH(append_launch, (hipStream_t)stream, p, vec);
    S2S_LAUNCH_CHECK();
    return S2S_OK;
}

extern "C" int32_t s2s_op_kv_read_paged(void* stream, const s2s_paged_kv* kv, const int32_t* table_dev, int32_t table_cols, const int32_t* start_dev,
                                        const int32_t* cu_dev, int32_t B, int32_t T, int32_t max_new, void* k_out, void* v_out, int64_t o_rs) {
    int rc = paged_check(kv, "kv_read_paged");
    if (rc) return rc;
    ReadParams p{};
    if ((rc = paged_rows(p.r, kv, table_dev, table_cols, cu_dev, B, T, max_new, "kv_read_paged"))) return rc;
    if (B == 0 || T == 0 || (!k_out && !v_out)) return S2S_OK;
    S2S_REQUIRE(start_dev, "kv_read_paged: null buffer");
    S2S_REQUIRE(rows_apart(T, o_rs, (int64_t)kv->kv_heads * kv->head_dim), "kv_read_paged: rows share memory (stride %lld)", (long long)o_rs);
    const int es = kv->dtype == S2S_F32 ? 4 : 2;
    const bool vec = (!k_out || aligned(k_out, o_rs, es)) && (!v_out || aligned(v_out, o_rs, es));
    p.kc = kv->k; p.vc = kv->v; p.km = (const _Float16*)kv->k_meta; p.vm = (const _Float16*)kv->v_meta;
    p.ko = k_out; p.vo = v_out; p.o_rs = o_rs; p.start = start_dev;
    S2S_PAGED_DISPATCH(read_launch, (hipStream_t)stream, p, vec);
    S2S_LAUNCH_CHECK();
    return S2S_OK;
}
