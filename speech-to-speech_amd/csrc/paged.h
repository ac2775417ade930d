// What the kernels of the paged key / value cache share: element types, octets (8 neighbouring elements) and the 4-bit code layout.
//
// Cache layout (include/s2s_mi355x.h, s2s_paged_kv): keys [page][Hkv][ps][D], values TRANSPOSED [page][Hkv][D][ps].  The attention reads both
// along the dimension its matrix product contracts (K along channels, V along positions), so every MFMA operand is one 16-byte load of 8
// neighbours and nothing is transposed on the reading side, which reads a row as often as the session still grows.  The writer pays: it
// transposes 64 x 64 tiles through LDS once per row.
#pragma once
#include "ops.h"

namespace s2s {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

enum { KV_F32 = 0, KV_BF16 = 1, KV_INT4 = 2 };   // template value: model-type cache of either type, or 4-bit codes under bf16 rows

// value = zero + scale * (code - 8): unsigned codes 0 .. 15 around the middle of the group's range
constexpr int KV_GROUP = 32;                     // channels of one position that share a scale and a zero = one k-step of the MFMA

// Octet of codes in one dword: element e in nibble (e >> 1) + 4 * (e & 1).  (w >> 4 i) & 0x000f000f then yields the neighbours 2 i and 2 i + 1 in
// the two halves, which is where a pair of 16-bit operands wants them.
__device__ __forceinline__ unsigned code_nibble(int e) { return (unsigned)((e >> 1) + 4 * (e & 1)); }

__device__ __forceinline__ unsigned and_or(unsigned w, unsigned mask, unsigned bits) {
    unsigned r;       // one instruction where the second constant sits in a vector register; the compiler makes it two with literals
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(mask), "v"(bits));
    return r;
}
// 8 codes -> code - 8 as float16, exact: 0x6400 | c is 1024 + c, 0x6400 | c << 4 is 1024 + 16 c (both below 2048: no rounding)
__device__ __forceinline__ void codes_to_f16(unsigned w, f16x2_t (&c)[4]) {
    const f16x2_t off = {(_Float16)-1032.f, (_Float16)-1032.f};
    const f16x2_t sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f}, off16 = {(_Float16)-72.f, (_Float16)-72.f};
    const unsigned w8 = w >> 8;
    c[0] = __builtin_bit_cast(f16x2_t, and_or(w, 0x000f000fu, 0x64006400u)) + off;
    c[1] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, and_or(w, 0x00f000f0u, 0x64006400u)), sixteenth, off16);
    c[2] = __builtin_bit_cast(f16x2_t, and_or(w8, 0x000f000fu, 0x64006400u)) + off;
    c[3] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, and_or(w8, 0x00f000f0u, 0x64006400u)), sixteenth, off16);
}

// fields of a packed cache handle, checked by paged_check (paged.hip)
int paged_check(const s2s_paged_kv* kv, const char* who);
struct PagedRows;
// rows [T][n elements] that are written, rs apart: no two share memory
inline bool rows_apart(int T, int64_t rs, int64_t n) { return T <= 1 || rs >= n; }
int paged_rows(PagedRows& r, const s2s_paged_kv* kv, const int* table, int cols, const int* cu, int B, int T, int max_new, const char* who);
inline int paged_kind(const s2s_paged_kv* kv) { return kv->kind == S2S_KV_INT4 ? KV_INT4 : kv->dtype == S2S_F32 ? KV_F32 : KV_BF16; }

// sessions' new rows and pages, as every paged kernel takes them
struct PagedRows {
    const int* table; int cols;       // [B][cols] page numbers (row b: session b's pages in order; outside [0, n_pages): no page)
    const int* cu;                    // [B + 1] first row of every session, or null: one row per session
    int B, T, max_new;                // T rows in the row buffers; a session has at most max_new
    int n_pages, ps_log2, Hkv;
};
// rows [row0, row0 + n) of session b, cut to the buffers and to max_new -> how many there are uncut
__device__ __forceinline__ int session_rows(const PagedRows& r, int b, int& row0, int& n) {
    if (!r.cu) {
        row0 = b;
        n = 1;
        return 1;
    }
    const int c0 = r.cu[b], c1 = r.cu[b + 1];
    row0 = max(c0, 0);
    n = min(min(c1, r.T) - row0, r.max_new);
    n = max(n, 0);
    return c1 - row0;
}
// The same number as a scalar load, not yet looked at: the wait for it falls where page_ok asks.  b and pos must be the same in all lanes (the table is
// only read by these kernels, so the constant address space holds).
__device__ __forceinline__ int page_raw(const PagedRows& r, int b, int pos) {
    const int col = pos >> r.ps_log2;
    if (pos < 0 || col >= r.cols) return -1;
    typedef const __attribute__((address_space(4))) int* scalar_t;
    return ((scalar_t)(uintptr_t)r.table)[(long)b * r.cols + col];
}
__device__ __forceinline__ bool page_ok(const PagedRows& r, int pg) { return (unsigned)pg < (unsigned)r.n_pages; }
__device__ __forceinline__ int page_of(const PagedRows& r, int b, int pos) {
    const int col = pos >> r.ps_log2;
    if (pos < 0 || col >= r.cols) return -1;
    const int pg = r.table[(long)b * r.cols + col];
    return (unsigned)pg < (unsigned)r.n_pages ? pg : -1;
}

}  // namespace s2s

// F<T, KIND, D>(...) for the cache at hand
#define S2S_PAGED_D(F, T, KIND, ...)                                                      \
    do {                                                                                  \
        if (kv->head_dim == 64) F<T, KIND, 64>(__VA_ARGS__);                              \
        else if (kv->head_dim == 128) F<T, KIND, 128>(__VA_ARGS__);                       \
        else F<T, KIND, 256>(__VA_ARGS__);                                                \
    } while (0)
#define S2S_PAGED_DISPATCH(F, ...)                                                        \
    do {                                                                                  \
        const int kind_ = paged_kind(kv);                                                 \
        if (kind_ == KV_F32) S2S_PAGED_D(F, float, KV_F32, __VA_ARGS__);                  \
        else if (kind_ == KV_BF16) S2S_PAGED_D(F, __hip_bfloat16, KV_BF16, __VA_ARGS__);  \
        else S2S_PAGED_D(F, __hip_bfloat16, KV_INT4, __VA_ARGS__);                        \
    } while (0)
