// A cache of latent rows held in 8 bits: rows quantised as they are written, and read back (record layout: kv8.cuh).
//
// Both are one pass over the data, a warp per row: a step of 128 channels per warp instruction, 4 per lane, so that a
// group of 64 is 16 lanes and every access of a warp is one contiguous piece.
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

constexpr int KV8_WARPS = 8, KV8_STEP = 128, KV8_STEPS = KV8_MAX_D / KV8_STEP;

__device__ __forceinline__ float4 load4(const void *x, bool bf16, size_t i) {
    if (!bf16) return *reinterpret_cast<const float4 *>(static_cast<const float *>(x) + i);
    const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(x) + i);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}

// Row t of sequence b goes to entry pos[b] + t of that sequence's cache, modulo `cap` in a ring.  Of the rows of one call
// that share a place in a ring only the last is written, so that the result is that of writing them one by one.
__global__ void __launch_bounds__(32 * KV8_WARPS)
kv8_write_kernel(const void *x, bool bf16, int d, int rd, long long rows, int s, const int64_t *pos, const int32_t *counts, bool ring,
                 uint8_t *cache, long long cap, long long stride) {
    APUS_PDL_WAIT();
    APUS_PDL_GO();
    const long long row = (long long)blockIdx.x * KV8_WARPS + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int lane = threadIdx.x & 31;
    const long long b = row / s;
    const int t = (int)(row - b * s), n = counts ? min(max(counts[b], 0), s) : s;
    if (t >= n) return;
    long long at = pos[b] + t;
    if (at < 0) return;
    if (ring) {
        if ((long long)n - t > cap) return;
        at %= cap;
    } else if (at >= cap) {
        return;
    }
    float4 v[KV8_STEPS];
#pragma unroll
    for (int k = 0; k < KV8_STEPS; k++) {
        const int ch = k * KV8_STEP + lane * 4;
        v[k] = ch < d ? load4(x, bf16, (size_t)row * d + ch) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    uint8_t *rec = cache + (size_t)(b * stride + at) * kv8_row_bytes(d, rd);
    const int nq = d - rd;
    uint32_t sc[2] = {0u, 0u};                                   // the row's scale bytes, in every lane
#pragma unroll
    for (int k = 0; k < KV8_STEPS; k++) {
        if (k * KV8_STEP >= nq) break;
        // absolute values compare as their bits do, and a NaN's bits are above infinity's
        uint32_t m = max(max(__float_as_uint(v[k].x) & 0x7fffffffu, __float_as_uint(v[k].y) & 0x7fffffffu),
                         max(__float_as_uint(v[k].z) & 0x7fffffffu, __float_as_uint(v[k].w) & 0x7fffffffu));
#pragma unroll
        for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));      // over the 16 lanes of a group
        const bool odd = m >= 0x7f800000u;
        const float s1 = ceil_pow2(__fmul_rn(fmaxf(__uint_as_float(m), 1e-4f), 1.0f / 448.0f));
        const float inv = __uint_as_float(0x7f000000u - __float_as_uint(s1));            // 1 / s1, exact
        const uint32_t byte = odd ? 255u : __float_as_uint(s1) >> 23;
        const int ch = k * KV8_STEP + lane * 4;
        if (ch < nq) {
            const uint32_t c = (uint32_t)e4m3x2_from_f32(v[k].x * inv, v[k].y * inv) |
                               (uint32_t)e4m3x2_from_f32(v[k].z * inv, v[k].w * inv) << 16;
            *reinterpret_cast<uint32_t *>(rec + ch) = odd ? 0x7f7f7f7fu : c;
        }
        const uint32_t lo = __shfl_sync(0xffffffffu, byte, 0), hi = __shfl_sync(0xffffffffu, byte, 16);
        sc[k >> 1] |= (lo | (k * KV8_STEP + 64 < nq ? hi << 8 : 0u)) << (16 * (k & 1));
    }
    if (lane == 0) *reinterpret_cast<uint4 *>(rec + kv8_scale_off(d, rd)) = make_uint4(sc[0], sc[1], 0u, 0u);
#pragma unroll
    for (int k = 0; k < KV8_STEPS; k++) {
        const int ch = k * KV8_STEP + lane * 4;
        if (ch >= nq && ch < d)
            *reinterpret_cast<uint2 *>(rec + nq + 2 * (ch - nq)) =
                make_uint2(bf16x2_rn(v[k].x, v[k].y), bf16x2_rn(v[k].z, v[k].w));
    }
}

__global__ void __launch_bounds__(32 * KV8_WARPS)
kv8_read_kernel(const uint8_t *cache, int d, int rd, long long cap, long long stride, long long rows, int s, const int32_t *idx,
                long long first, void *out, bool bf16) {
    APUS_PDL_WAIT();
    APUS_PDL_GO();
    const long long row = (long long)blockIdx.x * KV8_WARPS + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int lane = threadIdx.x & 31;
    const long long b = row / s, at = idx ? (long long)idx[row] : first + (row - b * s);
    const bool there = at >= 0 && at < cap;
    const uint8_t *rec = cache + (size_t)(there ? b * stride + at : 0) * kv8_row_bytes(d, rd);
    const int nq = d - rd;
    uint2 raw[KV8_STEPS];
    uint32_t sc[KV8_STEPS];
#pragma unroll
    for (int k = 0; k < KV8_STEPS; k++) {
        const int ch = k * KV8_STEP + lane * 4;
        raw[k] = make_uint2(0u, 0u);
        sc[k] = 0u;
        if (there && ch < nq) {
            raw[k].x = *reinterpret_cast<const uint32_t *>(rec + ch);
            sc[k] = rec[kv8_scale_off(d, rd) + (ch >> 6)];
        } else if (there && ch < d) {
            raw[k] = *reinterpret_cast<const uint2 *>(rec + nq + 2 * (ch - nq));
        }
    }
#pragma unroll
    for (int k = 0; k < KV8_STEPS; k++) {
        const int ch = k * KV8_STEP + lane * 4;
        if (ch >= d) continue;
        float4 v;
        if (ch < nq) {
            const float f = kv8_scale(sc[k]);
            v = make_float4(e4m3_to_f32(raw[k].x & 0xffu) * f, e4m3_to_f32(raw[k].x >> 8 & 0xffu) * f,
                            e4m3_to_f32(raw[k].x >> 16 & 0xffu) * f, e4m3_to_f32(raw[k].x >> 24) * f);
        } else {
            v = make_float4(__uint_as_float(raw[k].x << 16), __uint_as_float(raw[k].x & 0xffff0000u),
                            __uint_as_float(raw[k].y << 16), __uint_as_float(raw[k].y & 0xffff0000u));
        }
        const size_t i = (size_t)row * d + ch;
        if (bf16)
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(out) + i) =
                make_uint2(bf16x2_rn(v.x, v.y), bf16x2_rn(v.z, v.w));
        else
            *reinterpret_cast<float4 *>(static_cast<float *>(out) + i) = v;
    }
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

int check_cache(const char *what, const void *cache, int64_t cap, int64_t stride, int n_seq, int s) {
    APUS_REQUIRE(n_seq >= 0 && s >= 0, "%s: %d sequences of %d rows", what, n_seq, s);
    APUS_REQUIRE(cap >= 0 && stride >= 0, "%s: cap=%lld, stride=%lld", what, (long long)cap, (long long)stride);
    APUS_REQUIRE(cap == 0 || cache, "%s: no cache", what);
    APUS_REQUIRE(aligned16(cache), "%s: the cache must start on a 16-byte boundary", what);
    APUS_REQUIRE((long long)n_seq * s <= (1ll << 33), "%s: %d x %d rows are too many for one call", what, n_seq, s);
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
    APUS_REQUIRE(aligned16(x), "kv8_write: the rows must start on a 16-byte boundary");
    if (ensure_enabled()) return 1;
    const long long rows = (long long)n_seq * s;
    launch_k(kv8_write_kernel, dim3((unsigned)ceil_div(rows, KV8_WARPS)), 32 * KV8_WARPS, 0, (cudaStream_t)stream, x, x_bf16 != 0, d, rd,
             rows, s, pos, counts, ring != 0, cache, (long long)cap, (long long)stride);
    APUS_LAUNCHED();
    return 0;
}

int apus_cuda_kv8_read_dev(const uint8_t *cache, int d, int rd, int64_t cap, int64_t stride, int n_seq, int s, const int32_t *idx,
                           int64_t first, void *out, int out_bf16, void *stream) {
    if (kv8_check_row("kv8_read", d, rd) || check_cache("kv8_read", cache, cap, stride, n_seq, s)) return 1;
    if (n_seq == 0 || s == 0) return 0;
    APUS_REQUIRE(out && aligned16(out), "kv8_read: the output must start on a 16-byte boundary");
    if (ensure_enabled()) return 1;
    const long long rows = (long long)n_seq * s;
    launch_k(kv8_read_kernel, dim3((unsigned)ceil_div(rows, KV8_WARPS)), 32 * KV8_WARPS, 0, (cudaStream_t)stream, cache, d, rd,
             (long long)cap, (long long)stride, rows, s, idx, (long long)first, out, out_bf16 != 0);
    APUS_LAUNCHED();
    return 0;
}

}  // extern "C"
