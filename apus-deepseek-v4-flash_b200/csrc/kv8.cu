// A cache of latent rows held in 8 bits: rows quantised as they are written, and read back (record layout: kv8.cuh).
//
// Both are one pass over the data: a warp per row, 256 channels per warp instruction, 8 per lane, so that a group of 64 is
// eight lanes and every access of a warp is one contiguous piece.  The floor is HBM; what they were bound by first was
// instructions (313 per row written), hence the conversions two and four values at a time and no 64-bit division.
#include "kernels.cuh"
#include "kv8.cuh"
#include "runtime.cuh"

namespace apus {

int kv8_check_row(const char *what, int d, int rd) {
    APUS_REQUIRE(d > 0 && d % KV8_GROUP == 0 && d <= KV8_MAX_D, "%s: d=%d must be a multiple of 64 up to 512", what, d);
    APUS_REQUIRE((rd == 0 || rd == 64) && rd < d, "%s: rd=%d must be 0 or 64 and below d=%d", what, rd, d);
    return 0;
}

namespace {

constexpr int KV8_WARPS = 8, KV8_STEP = 256, KV8_STEPS = KV8_MAX_D / KV8_STEP;

// 8 values of f32 in one access (32-byte boundaries)
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(p));
}
__device__ __forceinline__ void store8(float *p, const float (&v)[8]) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
}

// Row t of sequence b goes to entry pos[b] + t of that sequence's cache, modulo `cap` in a ring.  Of the rows of one call
// that share a place in a ring only the last is written, so that the result is that of writing them one by one.
// B200, 65,536 rows of 512, eight sets of buffers in turn so that L2 holds none: BF16 19.6 us, f32 25.7 us (5.4 and 6.7 TB/s, where a
// plain copy moves 6.55: three quarters of the f32 traffic are reads).
template <bool BF16>
__global__ void __launch_bounds__(32 * KV8_WARPS)
kv8_write_kernel(const void *x, int d, int rd, uint32_t rows, uint32_t s, const int64_t *pos, const int32_t *counts, bool ring,
                 uint8_t *cache, long long cap, long long stride) {
    APUS_PDL_WAIT();
    APUS_PDL_GO();
    const uint32_t row = blockIdx.x * KV8_WARPS + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int lane = threadIdx.x & 31, nq = d - rd;
    uint4 w[KV8_STEPS];
    float v[KV8_STEPS][8];
#pragma unroll
    for (int k = 0; k < KV8_STEPS; k++) {
        const int ch = k * KV8_STEP + lane * 8;
        w[k] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int i = 0; i < 8; i++) v[k][i] = 0.f;
        if (ch < d) {
            if (BF16) w[k] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(x) + (size_t)row * d + ch);
            else load8(static_cast<const float *>(x) + (size_t)row * d + ch, v[k]);
        }
    }
    const uint32_t b = row / s;
    const int t = (int)(row - b * s), n = counts ? min(max(counts[b], 0), (int)s) : (int)s;
    long long at = (long long)((unsigned long long)pos[b] + t);          // beyond the last of all numbers: a negative one
    if (t >= n || at < 0 || (ring ? (long long)n - t > cap && at <= INT64_MAX - cap : at >= cap)) return;     // in a ring: unless row t + cap has the place
    if (at >= cap) at = (uint64_t)(at | cap) >> 32 ? at % cap : (uint32_t)at % (uint32_t)cap;
    uint8_t *rec = cache + (size_t)(b * stride + at) * kv8_row_bytes(d, rd);
    uint32_t sc[KV8_STEPS];                                      // the row's scale bytes, in every lane
#pragma unroll
    for (int k = 0; k < KV8_STEPS; k++) {
        const int ch = k * KV8_STEP + lane * 8;
        // absolute values compare as their bits do, and a NaN's bits are above infinity's
        uint32_t m = 0;
        if (BF16) {
            const uint32_t u = max_u16x2(max_u16x2(w[k].x & 0x7fff7fffu, w[k].y & 0x7fff7fffu), max_u16x2(w[k].z & 0x7fff7fffu, w[k].w & 0x7fff7fffu));
            m = max(u << 16, u & 0xffff0000u);
            const uint32_t q[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
            for (int i = 0; i < 8; i++) v[k][i] = __uint_as_float(i & 1 ? q[i / 2] & 0xffff0000u : q[i / 2] << 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(v[k][i]) & 0x7fffffffu);
        }
#pragma unroll
        for (int o = 4; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));      // over the 8 lanes of a group
        // the least power of two not below amax / 448: a significand that is not zero carries into the exponent
        const uint32_t s1 = (__float_as_uint(__fmul_rn(fmaxf(__uint_as_float(m), 1e-4f), 1.0f / 448.0f)) + 0x7fffffu) & 0xff800000u;
        const bool odd = m >= 0x7f800000u;
        const float inv = __uint_as_float(odd ? 0x7fffffffu : 0x7f000000u - s1);         // exact; a NaN makes every code one
        if (ch < nq) {
            uint32_t c[2];
#pragma unroll
            for (int i = 0; i < 2; i++)
                c[i] = (uint32_t)e4m3x2_from_f32(v[k][4 * i] * inv, v[k][4 * i + 1] * inv) |
                       (uint32_t)e4m3x2_from_f32(v[k][4 * i + 2] * inv, v[k][4 * i + 3] * inv) << 16;
            *reinterpret_cast<uint2 *>(rec + ch) = make_uint2(c[0], c[1]);
        } else if (ch < d) {
            if (!BF16)
                w[k] = make_uint4(bf16x2_rn(v[k][0], v[k][1]), bf16x2_rn(v[k][2], v[k][3]), bf16x2_rn(v[k][4], v[k][5]), bf16x2_rn(v[k][6], v[k][7]));
            *reinterpret_cast<uint4 *>(rec + nq + 2 * (ch - nq)) = w[k];
        }
        sc[k] = __reduce_or_sync(0xffffffffu, (lane & 7) || ch >= nq ? 0u : (odd ? 255u : s1 >> 23) << lane);
    }
    if (lane == 0) *reinterpret_cast<uint4 *>(rec + kv8_scale_off(d, rd)) = make_uint4(sc[0], sc[1], 0u, 0u);
}

// B200, 65,536 rows of 512, measured likewise: to BF16 18.6 us, to f32 27.7 us (5.7 and 6.2 TB/s).
__global__ void __launch_bounds__(32 * KV8_WARPS)
kv8_read_kernel(const uint8_t *cache, int d, int rd, long long cap, long long stride, uint32_t rows, uint32_t s, const int32_t *idx,
                long long first, void *out, bool bf16) {
    APUS_PDL_WAIT();
    APUS_PDL_GO();
    const uint32_t row = blockIdx.x * KV8_WARPS + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int lane = threadIdx.x & 31, nq = d - rd;
    const uint32_t b = row / s;
    const long long e = idx ? (long long)idx[row] : (long long)((unsigned long long)first + (row - b * s));
    const bool there = e >= 0 && e < cap;
    const uint8_t *rec = cache + (size_t)(there ? b * stride + e : 0) * kv8_row_bytes(d, rd);
    uint4 raw[KV8_STEPS];
    uint32_t sc[KV8_STEPS];
#pragma unroll
    for (int k = 0; k < KV8_STEPS; k++) {
        const int ch = k * KV8_STEP + lane * 8;
        raw[k] = make_uint4(0u, 0u, 0u, 0u);
        sc[k] = 127u;
        if (there && ch < nq) {
            const uint2 u = *reinterpret_cast<const uint2 *>(rec + ch);
            raw[k].x = u.x;
            raw[k].y = u.y;
            sc[k] = rec[kv8_scale_off(d, rd) + (ch >> 6)];
        } else if (there && ch < d) {
            raw[k] = *reinterpret_cast<const uint4 *>(rec + nq + 2 * (ch - nq));
        }
    }
#pragma unroll
    for (int k = 0; k < KV8_STEPS; k++) {
        const int ch = k * KV8_STEP + lane * 8;
        if (ch >= d) continue;
        uint32_t u[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};                        // as BF16
        float v[8];
        if (ch < nq) {
            const uint32_t f = code_factor(min(sc[k], 134u));
            const uint2 p = codes_bf16x4(raw[k].x, f), q = codes_bf16x4(raw[k].y, f);
            u[0] = __byte_perm(p.x, p.y, 0x5410);
            u[1] = __byte_perm(p.x, p.y, 0x7632);
            u[2] = __byte_perm(q.x, q.y, 0x5410);
            u[3] = __byte_perm(q.x, q.y, 0x7632);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __uint_as_float(i & 1 ? u[i / 2] & 0xffff0000u : u[i / 2] << 16);
        if (ch < nq && sc[k] - 16u > 134u - 16u) {               // the products above may have left BF16's normal range
            const float f = kv8_scale(sc[k]);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = e4m3_to_f32((i < 4 ? raw[k].x : raw[k].y) >> 8 * (i & 3) & 0xffu) * f;
#pragma unroll
            for (int i = 0; i < 4; i++) u[i] = bf16x2_rn(v[2 * i], v[2 * i + 1]);
        }
        const size_t i = (size_t)row * d + ch;
        if (bf16) *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(out) + i) = make_uint4(u[0], u[1], u[2], u[3]);
        else store8(static_cast<float *>(out) + i, v);
    }
}

bool aligned(const void *p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

int check_cache(const char *what, const void *cache, int64_t cap, int64_t stride, int n_seq, int s) {
    APUS_REQUIRE(n_seq >= 0 && s >= 0, "%s: %d sequences of %d rows", what, n_seq, s);
    APUS_REQUIRE(cap >= 0 && stride >= 0, "%s: cap=%lld, stride=%lld", what, (long long)cap, (long long)stride);
    APUS_REQUIRE(cap == 0 || cache, "%s: no cache", what);
    APUS_REQUIRE(aligned(cache, 16), "%s: the cache must start on a 16-byte boundary", what);
    APUS_REQUIRE((long long)n_seq * s < (1ll << 31), "%s: %d x %d rows are too many for one call", what, n_seq, s);
    return 0;
}

}  // namespace
}  // namespace apus

using namespace apus;

extern "C" {

size_t apus_cuda_kv8_row_bytes(int d, int rd) { return kv8_check_row("kv8_row_bytes", d, rd) ? 0 : (size_t)kv8_row_bytes(d, rd); }

int apus_cuda_kv8_write_dev(const void *x, int x_bf16, int d, int rd, int n_seq, int s, const int64_t *pos, const int32_t *counts,
                            int ring, uint8_t *cache, int64_t cap, int64_t stride, void *stream) {
    if (kv8_check_row("kv8_write", d, rd) || check_cache("kv8_write", cache, cap, stride, n_seq, s)) return 1;
    // two sequences that share entries would be written by two warps at once
    APUS_REQUIRE(n_seq <= 1 || stride >= cap, "kv8_write: caches of %lld rows lie %lld rows apart", (long long)cap, (long long)stride);
    if (n_seq == 0 || s == 0 || cap == 0) return 0;
    APUS_REQUIRE(x && pos, "kv8_write: no %s", x ? "positions" : "rows");
    APUS_REQUIRE(aligned(x, x_bf16 ? 16 : 32), "kv8_write: the rows must start on a %d-byte boundary", x_bf16 ? 16 : 32);
    if (ensure_enabled()) return 1;
    const long long rows = (long long)n_seq * s;
    const dim3 grid((unsigned)ceil_div(rows, KV8_WARPS));
    if (x_bf16)
        launch_k(kv8_write_kernel<true>, grid, 32 * KV8_WARPS, 0, (cudaStream_t)stream, x, d, rd, (uint32_t)rows, (uint32_t)s, pos, counts,
                 ring != 0, cache, (long long)cap, (long long)stride);
    else
        launch_k(kv8_write_kernel<false>, grid, 32 * KV8_WARPS, 0, (cudaStream_t)stream, x, d, rd, (uint32_t)rows, (uint32_t)s, pos, counts,
                 ring != 0, cache, (long long)cap, (long long)stride);
    APUS_LAUNCHED();
    return 0;
}

int apus_cuda_kv8_read_dev(const uint8_t *cache, int d, int rd, int64_t cap, int64_t stride, int n_seq, int s, const int32_t *idx,
                           int64_t first, void *out, int out_bf16, void *stream) {
    if (kv8_check_row("kv8_read", d, rd) || check_cache("kv8_read", cache, cap, stride, n_seq, s)) return 1;
    if (n_seq == 0 || s == 0) return 0;
    APUS_REQUIRE(out && aligned(out, out_bf16 ? 16 : 32), "kv8_read: the output must start on a %d-byte boundary", out_bf16 ? 16 : 32);
    if (ensure_enabled()) return 1;
    const long long rows = (long long)n_seq * s;
    launch_k(kv8_read_kernel, dim3((unsigned)ceil_div(rows, KV8_WARPS)), 32 * KV8_WARPS, 0, (cudaStream_t)stream, cache, d, rd,
             (long long)cap, (long long)stride, (uint32_t)rows, (uint32_t)s, idx, (long long)first, out, out_bf16 != 0);
    APUS_LAUNCHED();
    return 0;
}

}  // extern "C"
