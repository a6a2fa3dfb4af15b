// Attention over caches held in 8 bits (record layout: kv8.cuh): the decode and chunk form of the reference's sparse
// attention (c/attn.h:1308) with one latent row per token as key and value of all heads,
//
//   o[t, h] = sum_j p_j v_j / (sum_j p_j + exp(sink[h])),   p_j = exp(scale * q[t, h] . k_j),   k_j = v_j,
//
// j over the ids of row t: below na a row of kv_a (the window), from na on a row of kv_b (the compressed entries);
// a negative id, or one behind both caches, is a hole.
#include "kernels.cuh"
#include "kv8.cuh"
#include "runtime.cuh"

namespace apus {
namespace {

struct AttnKv8Args {
    const void *q;
    const float *sink;
    const int32_t *idxs;
    const uint8_t *kv_a, *kv_b;
    void *o;
    long long na, nb, a_stride, b_stride;
    int h, d, rd, idxw, rows, rows_per_seq;
    float scale;
    int q_bf16, o_bf16;
};

// The record that id `id` of sequence `seq` names, NULL for a hole.
__device__ __forceinline__ const uint8_t *kv8_record(const AttnKv8Args &a, long long seq, int id) {
    if (id < 0) return nullptr;
    const size_t rb = (size_t)kv8_row_bytes(a.d, a.rd);
    if (id < a.na) return a.kv_a + (size_t)(seq * a.a_stride + id) * rb;
    const long long j = id - a.na;
    return j < a.nb ? a.kv_b + (size_t)(seq * a.b_stride + j) * rb : nullptr;
}

// A warp per head, 32 candidates at a time: dequantised into shared memory, a candidate per lane for the scores, the
// channels over the lanes for the sum of the values.
constexpr int AK_HEADS = 8, AK_CANDS = 32, AK_LD = KV8_MAX_D + 1;
__global__ void __launch_bounds__(32 * AK_HEADS)
attn_kv8_kernel(const AttnKv8Args a) {
    APUS_PDL_WAIT();
    APUS_PDL_GO();
    extern __shared__ float sm[];
    float *kv = sm, *qs = sm + AK_CANDS * AK_LD;                 // [32][d], [8][d]
    __shared__ int s_valid[AK_CANDS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row = blockIdx.x, seq = row / a.rows_per_seq;
    const int head = (int)blockIdx.y * AK_HEADS + warp, nq = a.d - a.rd;
    const bool on = head < a.h;
    for (int i = lane; i < a.d; i += 32) {
        const size_t at = ((size_t)row * a.h + (on ? head : 0)) * a.d + i;
        qs[warp * a.d + i] = a.q_bf16 ? bf16_to_f32(static_cast<const uint16_t *>(a.q)[at]) : bf16_round(static_cast<const float *>(a.q)[at]);
    }
    float m = -INFINITY, l = 0.f, acc[KV8_MAX_D / 32];
#pragma unroll
    for (int i = 0; i < KV8_MAX_D / 32; i++) acc[i] = 0.f;
    for (int j0 = 0; j0 < a.idxw; j0 += AK_CANDS) {
        __syncthreads();
        for (int c = warp; c < AK_CANDS; c += AK_HEADS) {
            const uint8_t *rec = j0 + c < a.idxw ? kv8_record(a, seq, a.idxs[(size_t)row * a.idxw + j0 + c]) : nullptr;
            if (lane == 0) s_valid[c] = rec != nullptr;
            for (int i = lane; i < a.d; i += 32) {
                float v = 0.f;
                if (rec) v = i < nq ? e4m3_to_f32(rec[i]) * kv8_scale(rec[kv8_scale_off(a.d, a.rd) + (i >> 6)])
                                    : bf16_to_f32(*reinterpret_cast<const uint16_t *>(rec + nq + 2 * (i - nq)));
                kv[c * AK_LD + i] = v;
            }
        }
        __syncthreads();
        float x = 0.f;
        for (int i = 0; i < a.d; i++) x += qs[warp * a.d + i] * kv[lane * AK_LD + i];
        x = s_valid[lane] ? x * a.scale : -INFINITY;
        const float m2 = fmaxf(m, warp_max(x)), mm = m2 == -INFINITY ? 0.f : m2, f = expf(m - mm);
        const float p = s_valid[lane] ? expf(x - mm) : 0.f;
        l = l * f + warp_sum(p);
#pragma unroll
        for (int i = 0; i < KV8_MAX_D / 32; i++) acc[i] *= f;
        for (int c = 0; c < AK_CANDS; c++) {
            const float w = __shfl_sync(0xffffffffu, p, c);
#pragma unroll
            for (int i = 0; i < KV8_MAX_D / 32; i++)
                if (32 * i < a.d) acc[i] += w * kv[c * AK_LD + 32 * i + lane];
        }
        m = m2;
    }
    if (!on) return;
    const float sk = a.sink ? a.sink[head] : -INFINITY, m2 = fmaxf(m, sk), mm = m2 == -INFINITY ? 0.f : m2;
    const float den = l * expf(m - mm) + expf(sk - mm), f = sk == INFINITY || den == 0.f ? 0.f : expf(m - mm) / den;
#pragma unroll
    for (int i = 0; i < KV8_MAX_D / 32; i++)
        if (32 * i < a.d) {
            const size_t at = ((size_t)row * a.h + head) * a.d + 32 * i + lane;
            if (a.o_bf16) static_cast<uint16_t *>(a.o)[at] = (uint16_t)bf16x2_rn(acc[i] * f, 0.f);
            else static_cast<float *>(a.o)[at] = __uint_as_float(bf16x2_rn(acc[i] * f, 0.f) << 16);
        }
}

int attn_kv8(const AttnKv8Args &a, cudaStream_t st) {
    const size_t sm = (size_t)(AK_CANDS * AK_LD + AK_HEADS * a.d) * sizeof(float);
    if (ensure_dyn_smem((const void *)attn_kv8_kernel, sm)) return 1;
    launch_k(attn_kv8_kernel, dim3((unsigned)a.rows, (unsigned)ceil_div(a.h, AK_HEADS)), 32 * AK_HEADS, sm, st, a);
    APUS_LAUNCHED();
    return 0;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace
}  // namespace apus

using namespace apus;

extern "C" int apus_cuda_sparse_attn_kv8_dev(const void *q, int q_bf16, const float *sink, int h, int d, int rd, const int32_t *idxs, int idxw,
                                             int rows, int rows_per_seq, float scale, const uint8_t *kv_a, int64_t na, int64_t kv_a_stride,
                                             const uint8_t *kv_b, int64_t nb, int64_t kv_b_stride, void *o, int o_bf16, void *stream) {
    if (kv8_check_row("sparse_attn_kv8", d, rd)) return 1;
    APUS_REQUIRE(h > 0 && h <= 1024, "sparse_attn_kv8: h=%d must be 1 to 1024", h);
    APUS_REQUIRE(rows >= 0 && idxw >= 0, "sparse_attn_kv8: %d rows of %d ids", rows, idxw);
    APUS_REQUIRE(rows_per_seq > 0 && rows % rows_per_seq == 0, "sparse_attn_kv8: %d rows are not sequences of %d", rows, rows_per_seq);
    APUS_REQUIRE(na >= 0 && nb >= 0 && na + nb <= INT32_MAX, "sparse_attn_kv8: na=%lld, nb=%lld", (long long)na, (long long)nb);
    APUS_REQUIRE(kv_a_stride >= 0 && kv_b_stride >= 0, "sparse_attn_kv8: negative stride");
    APUS_REQUIRE((na == 0 || kv_a) && (nb == 0 || kv_b), "sparse_attn_kv8: no cache");
    APUS_REQUIRE(aligned16(kv_a) && aligned16(kv_b), "sparse_attn_kv8: the caches must start on a 16-byte boundary");
    if (rows == 0) return 0;
    APUS_REQUIRE(q && o && (idxs || idxw == 0), "sparse_attn_kv8: no %s", !q ? "queries" : !o ? "output" : "ids");
    APUS_REQUIRE(aligned16(q) && aligned16(o), "sparse_attn_kv8: queries and output must start on a 16-byte boundary");
    if (ensure_enabled()) return 1;
    const AttnKv8Args a = {q, sink, idxs, kv_a, kv_b, o, na, nb, kv_a_stride, kv_b_stride, h, d, rd, idxw, rows, rows_per_seq,
                           scale, q_bf16 != 0, o_bf16 != 0};
    return attn_kv8(a, (cudaStream_t)stream);
}
