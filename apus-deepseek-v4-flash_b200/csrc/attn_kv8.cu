// Attention over caches held in 8 bits (record layout: kv8.cuh): the decode and chunk form of the reference's sparse
// attention (c/attn.h:1308) with one latent row per token as key and value of all heads,
//
//   o[t, h] = sum_j p_j v_j / (sum_j p_j + exp(sink[h])),   p_j = exp(scale * q[t, h] . k_j),   k_j = v_j,
//
// j over the ids of row t: below na a row of kv_a (the window), from na on a row of kv_b (the compressed entries);
// a negative id, or one behind both caches, is a hole.
#include <mutex>

#include "kernels.cuh"
#include "kv8.cuh"
#include "runtime.cuh"
#include "tc_common.cuh"

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
    int cluster, unit;           // CTAs per query row, tokens per tile (a multiple of 16 up to 128)
    int *status;
};

// The record that id `id` of sequence `seq` names, NULL for a hole.
__device__ __forceinline__ const uint8_t *kv8_record(const AttnKv8Args &a, long long seq, int id) {
    if (id < 0) return nullptr;
    const size_t rb = (size_t)kv8_row_bytes(a.d, a.rd);
    if (id < a.na) return a.kv_a + (size_t)(seq * a.a_stride + id) * rb;
    const long long j = id - a.na;
    return j < a.nb ? a.kv_b + (size_t)(seq * a.b_stride + j) * rb : nullptr;
}

// ---- the kernel ------------------------------------------------------------------------------------------------------
// One query row has 64 heads on the same latent rows: 256 operations for every byte of the cache, where this GPU's ratio
// of tensor rate to memory rate is 253.  So both contractions go to the tensor cores (tcgen05, BF16 operands, f32 sums), a
// cache row is fetched and dequantised once for all heads, and it serves as key and as value from the same place:
//
//   S^T[token, head]   = K[token, ch] Q[head, ch]^T     A = 128 rows as they lie (K-major),  B = the queries
//   O^T[ch, head]     += V[token, ch]^T P[token, head]   A = the same rows (MN-major),         B = the numerators
//
// With tokens, then channels as the 128 rows of an instruction, the 64 heads are its columns and no instruction runs half
// empty.  A group of codes times its power of two is a BF16 value exactly (4 significant bits), so nothing is rounded
// before the products.  A token is a TMEM lane, so that a thread turns one token's scores into numerators for 32 heads and
// stores them as one contiguous piece of a row of P.
//
// The softmax is one pass with a reference per head instead of the running maximum: it is set to the first tile's maximum
// and stays until a score exceeds it by more than 2^AK_SLACK, which in f32 and BF16, floating as both are, costs no
// precision; only then is the accumulator scaled.  Sums of numerators stay in each thread until the end.
//
// A row's candidates are cut into tiles of at most 128, dealt in turn to the CTAs of a cluster.  At the end every CTA
// tells the others its references and sums, scales its part of O^T and stores it into the shared memory of the CTA that
// owns the channels, which adds the parts in rank order: one launch, no scratch, the same bits every time.
//
// Warps 0 to 7 fetch (into registers, a tile ahead), dequantise and do the softmax; warp 8 issues the MMAs.  Shared
// memory: 8 panels of 128 tokens x 64 channels (128-byte swizzled rows), Q as 8 panels of 64 heads x 64 channels, P.
constexpr int AK_TILE = 128, AK_HEADS = 64, AK_WORKERS = 256, AK_THREADS = AK_WORKERS + 32, AK_MAX_C = 16;
constexpr int AK_PANEL = AK_TILE * 128, AK_QPANEL = AK_HEADS * 128;
constexpr int AK_Q_OFF = 8 * AK_PANEL, AK_P_OFF = AK_Q_OFF + 8 * AK_QPANEL, AK_MISC_OFF = AK_P_OFF + AK_PANEL;
constexpr float AK_SLACK = 40.f, AK_NONE = -1.7e38f, LOG2E = 1.4426950408889634f;

struct AkMisc {
    float2 ml[AK_MAX_C][AK_HEADS];                     // reference and sum of every CTA of the cluster
    float m[AK_HEADS], f[AK_HEADS], part[4][AK_HEADS];
    uint64_t full[4], empty[4], s_full, p_ready, o_done;
    uint32_t tmem;
    int abort;
};
constexpr int AK_SMEM = AK_MISC_OFF + (int)sizeof(AkMisc) + 1024;
static_assert(AK_SMEM <= 227 * 1024, "shared memory of a CTA");

__device__ __forceinline__ void workers_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool workers_any(bool p) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)p) : "memory");
    return r != 0;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float redux_max(float x) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
          "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
          "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
// kind::f16, BF16 operands, f32 sums, 128 x 64 x 16; `mn`: both operands MN-major
__device__ __forceinline__ uint32_t ak_idesc(bool mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (mn ? (1u << 15) | (1u << 16) : 0u) | ((uint32_t)(AK_HEADS >> 3) << 17) |
           ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void ak_mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// MN-major operand of 128-byte swizzled rows, a row per k: 64 elements of M or N in a row, the next 64 a panel further
__device__ __forceinline__ uint64_t ak_desc_mn(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(AK_PANEL >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}

// Four codes -> four BF16 values times 2^-120: sign, exponent and significand bits moved to their places (the biases of
// the two formats differ by 120; a subnormal code becomes a subnormal value).
__device__ __forceinline__ uint2 codes_bf16x4(uint32_t c) {
    const uint32_t a = __byte_perm(c, 0u, 0x1404), b = __byte_perm(c, 0u, 0x3424);
    return make_uint2((a & 0x80008000u) | (a >> 4 & 0x07f007f0u), (b & 0x80008000u) | (b >> 4 & 0x07f007f0u));
}
// 16 codes of a group with scale byte `b` -> 16 BF16 values.  2^120 times the scale is a BF16 value up to byte 134 (rows of
// magnitude 57,344); larger ones take two multiplications.
__device__ __forceinline__ void dequant16(const uint4 &c, uint32_t b, uint4 &lo, uint4 &hi) {
    const uint2 w0 = codes_bf16x4(c.x), w1 = codes_bf16x4(c.y), w2 = codes_bf16x4(c.z), w3 = codes_bf16x4(c.w);
    lo = make_uint4(w0.x, w0.y, w1.x, w1.y);
    hi = make_uint4(w2.x, w2.y, w3.x, w3.y);
    uint32_t f = (b + 120u) << 7;
    if (b > 134u) {
        const uint32_t up = (247u << 7) | (247u << 23);
        lo = make_uint4(mul_bf16x2(lo.x, up), mul_bf16x2(lo.y, up), mul_bf16x2(lo.z, up), mul_bf16x2(lo.w, up));
        hi = make_uint4(mul_bf16x2(hi.x, up), mul_bf16x2(hi.y, up), mul_bf16x2(hi.z, up), mul_bf16x2(hi.w, up));
        f = b == 255u ? 0x7fffu : b << 7;
    }
    f |= f << 16;
    lo = make_uint4(mul_bf16x2(lo.x, f), mul_bf16x2(lo.y, f), mul_bf16x2(lo.z, f), mul_bf16x2(lo.w, f));
    hi = make_uint4(mul_bf16x2(hi.x, f), mul_bf16x2(hi.y, f), mul_bf16x2(hi.z, f), mul_bf16x2(hi.w, f));
}

// The ids of a tile, token 32 k + lane in id[k]; whether any of them names a record is the same in every warp.
struct TileIds {
    int id[4];
    __device__ __forceinline__ void load(const AttnKv8Args &a, const int32_t *ids, int tile, int lane) {
        const int t0 = tile * a.unit, t1 = min(t0 + a.unit, a.idxw);
#pragma unroll
        for (int k = 0; k < 4; k++) id[k] = t0 + 32 * k + lane < t1 ? ids[t0 + 32 * k + lane] : -1;
    }
    __device__ __forceinline__ bool any(const AttnKv8Args &a) {
        bool v = false;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (id[k] >= a.na + a.nb) id[k] = -1;
            v |= id[k] >= 0;
        }
        return __any_sync(0xffffffffu, v);
    }
};

// What a worker lane fetches of a tile: of its rows r0 and r0 + 8, 16 channels of every panel of codes, 16 BF16 values of
// the rotated panel and the scales.
template <bool TAIL>
struct TileRows {
    static constexpr int NC = TAIL ? 7 : 8;
    const uint8_t *rec[2];
    uint4 c[NC][2], t[TAIL ? 2 : 1][2];
    uint2 sc[2];
    __device__ __forceinline__ void find(const AttnKv8Args &a, long long seq, const TileIds &ids, int warp, int lane) {
        const int src = (warp & 1) * 16 + (lane >> 2);
        const int mine = warp >> 1 == 0 ? ids.id[0] : warp >> 1 == 1 ? ids.id[1] : warp >> 1 == 2 ? ids.id[2] : ids.id[3];
#pragma unroll
        for (int i = 0; i < 2; i++) rec[i] = kv8_record(a, seq, __shfl_sync(0xffffffffu, mine, src + 8 * i));
    }
    // panels 0 to 3 and the scales, or the others
    template <bool FIRST>
    __device__ __forceinline__ void load(const AttnKv8Args &a, int sub) {
        const int nq = a.d - a.rd;
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint8_t *r = rec[i];
#pragma unroll
            for (int p = FIRST ? 0 : 4; p < (FIRST ? 4 : NC); p++) c[p][i] = r && p * 64 < nq ? *reinterpret_cast<const uint4 *>(r + p * 64 + sub * 16) : zero;
            if (TAIL && !FIRST) {
                t[0][i] = r ? *reinterpret_cast<const uint4 *>(r + nq + sub * 32) : zero;
                t[TAIL ? 1 : 0][i] = r ? *reinterpret_cast<const uint4 *>(r + nq + sub * 32 + 16) : zero;
            }
            if (FIRST) sc[i] = r ? *reinterpret_cast<const uint2 *>(r + kv8_scale_off(a.d, a.rd)) : make_uint2(0u, 0u);
        }
    }
    // panel p of the tile into shared memory, rows r0 and r0 + 8
    __device__ __forceinline__ void store(uint8_t *panel, int p, bool rotated, int r0, int sub) const {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            uint4 lo, hi;
            if (TAIL && rotated) {
                lo = t[0][i];
                hi = t[TAIL ? 1 : 0][i];
            } else {
                dequant16(c[p < NC ? p : 0][i], (p < 4 ? sc[i].x >> 8 * (p & 3) : sc[i].y >> 8 * (p & 3)) & 0xffu, lo, hi);
            }
            uint8_t *row = panel + (r0 + 8 * i) * 128;
            *reinterpret_cast<uint4 *>(row + ((2 * sub) ^ (r0 & 7)) * 16) = lo;
            *reinterpret_cast<uint4 *>(row + ((2 * sub + 1) ^ (r0 & 7)) * 16) = hi;
        }
    }
};

// o[head][ch] of one warp: lane = channel, v[i] = head h0 + i of it, already scaled
template <int N>
__device__ __forceinline__ void ak_put(const AttnKv8Args &a, size_t at, int ch, int h0, int nh, const float (&v)[N], int lane) {
    if (!a.o_bf16) {
        float *o = static_cast<float *>(a.o) + at + ch + (size_t)h0 * a.d;
#pragma unroll
        for (int i = 0; i < N; i++, o += a.d)
            if (h0 + i < nh) *o = __uint_as_float(bf16x2_rn(v[i], 0.f) << 16);
        return;
    }
    // two lanes trade, so that each stores two channels of one of two heads
    uint16_t *o = static_cast<uint16_t *>(a.o) + at + (ch & ~1) + (size_t)(h0 + (lane & 1)) * a.d;
#pragma unroll
    for (int i = 0; i < N; i += 2, o += 2 * a.d) {
        const float other = __shfl_xor_sync(0xffffffffu, lane & 1 ? v[i] : v[i + 1], 1);
        const uint32_t w = lane & 1 ? bf16x2_rn(other, v[i + 1]) : bf16x2_rn(v[i], other);
        if (h0 + i + (lane & 1) < nh) *reinterpret_cast<uint32_t *>(o) = w;
    }
}

template <bool TAIL>
__global__ void __launch_bounds__(AK_THREADS, 1)
attn_kv8_kernel(const AttnKv8Args a) {
    APUS_PDL_WAIT();
    APUS_PDL_GO();
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    AkMisc &sm = *reinterpret_cast<AkMisc *>(smem + AK_MISC_OFF);
    volatile int *s_abort = &sm.abort;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, C = a.cluster;
    const int rank = (int)(blockIdx.x % (unsigned)C), h0 = (int)blockIdx.y * AK_HEADS, nh = min(AK_HEADS, a.h - h0);
    const long long row = blockIdx.x / (unsigned)C, seq = row / a.rows_per_seq;
    const int32_t *ids = a.idxs + (size_t)row * a.idxw;
    const int n_tiles = (a.idxw + a.unit - 1) / a.unit, NP = a.d / 64, NPAIR = (NP + 1) / 2;

    if (tid == 0) {
        for (int i = 0; i < 4; i++) { mbar_init(&sm.full[i], 8); mbar_init(&sm.empty[i], 1); }
        mbar_init(&sm.s_full, 1);
        mbar_init(&sm.p_ready, 8);
        mbar_init(&sm.o_done, 1);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid < AK_HEADS) sm.m[tid] = AK_NONE;
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&sm.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (C > 1) cluster_arrive();                        // this CTA has started: its shared memory may be stored to
    const uint32_t tmem = sm.tmem, tmem_s = tmem + 4 * AK_HEADS;

    // A wait that runs out sets the abort flag, after which every other wait gives up soon; all loops and barriers are gone
    // through all the same, so that no thread is left waiting, and nothing is written.
    int fail = 0;
    uint32_t done = 0;                                   // tiles of this CTA so far
    TileIds cur;
    int tile = rank;
    bool more = false;
    for (; tile < n_tiles; tile += C) {
        cur.load(a, ids, tile, lane);
        if ((more = cur.any(a))) break;
    }

    if (warp == 8) {
        const uint32_t id_s = ak_idesc(false), id_o = ak_idesc(true);
        const uint32_t kv = smem_u32(smem), q = smem_u32(smem + AK_Q_OFF), p = smem_u32(smem + AK_P_OFF);
        while (more) {
            const int ks = (min(a.unit, a.idxw - tile * a.unit) + 15) >> 4;      // steps of 16 tokens that hold any
            if (lane == 0) {
                for (int i = 0; i < NPAIR && !fail; i++) {
                    if (!mbar_wait(&sm.full[i], done & 1u, s_abort)) { fail = 51; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    for (int pn = 2 * i; pn < min(2 * i + 2, NP); pn++) {
                        const uint64_t da = umma_desc_sw128(kv + pn * AK_PANEL), db = umma_desc_sw128(q + pn * AK_QPANEL);
#pragma unroll
                        for (int j = 0; j < 4; j++) ak_mma(tmem_s, da + 2 * j, db + 2 * j, id_s, (pn | j) ? 1u : 0u);
                    }
                }
                if (!fail) umma_commit(&sm.s_full);
                if (!fail && !mbar_wait(&sm.p_ready, done & 1u, s_abort)) fail = 52;
                if (!fail) {
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    for (int i = 0; i < NPAIR; i++) {
                        const uint64_t da = ak_desc_mn(kv + 2 * i * AK_PANEL), db = ak_desc_mn(p);
                        for (int k = 0; k < ks; k++)
                            ak_mma(tmem + i * AK_HEADS, da + 128 * k, db + 128 * k, id_o, (done | (uint32_t)k) ? 1u : 0u);
                        umma_commit(&sm.empty[i]);
                    }
                }
                if (fail) *s_abort = 1;
            }
            __syncwarp();
            done++;
            more = false;
            for (tile += C; tile < n_tiles; tile += C) {
                cur.load(a, ids, tile, lane);
                if ((more = cur.any(a))) break;
            }
        }
        if (lane == 0 && !fail) umma_commit(&sm.o_done);
        __syncwarp();
    } else {
        const int r0 = warp * 16 + (lane >> 2), sub = lane & 3, quad = warp & 3, half = warp >> 2, token = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const float cs = a.scale * LOG2E;
        TileRows<TAIL> rows;
        rows.rec[0] = rows.rec[1] = nullptr;
        if (more) rows.find(a, seq, cur, warp, lane);
        rows.template load<true>(a, sub);
        // the queries, 8 channels at a time
        const int per_head = a.d / 8;
        for (int i0 = 0; i0 < AK_HEADS * per_head; i0 += AK_WORKERS * 4) {
            uint4 v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int i = i0 + k * AK_WORKERS + tid, head = i / per_head, c = i - head * per_head;
                v[k] = make_uint4(0u, 0u, 0u, 0u);
                if (head < nh) {
                    const size_t at = ((size_t)row * a.h + h0 + head) * a.d + c * 8;
                    if (a.q_bf16) {
                        v[k] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + at);
                    } else {
                        const float4 x = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + at);
                        const float4 y = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + at + 4);
                        v[k] = make_uint4(bf16x2_rn(x.x, x.y), bf16x2_rn(x.z, x.w), bf16x2_rn(y.x, y.y), bf16x2_rn(y.z, y.w));
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int i = i0 + k * AK_WORKERS + tid, head = i / per_head, c = i - head * per_head;
                if (head < AK_HEADS)
                    *reinterpret_cast<uint4 *>(smem + AK_Q_OFF + (c >> 3) * AK_QPANEL + head * 128 + (((c & 7) ^ (head & 7)) << 4)) = v[k];
            }
        }
        float l[32];
#pragma unroll
        for (int i = 0; i < 32; i++) l[i] = 0.f;
        while (more) {
            const int held = (min(a.unit, a.idxw - tile * a.unit) + 15) & ~15;   // rows that the MMAs read
            const int my_id = quad == 0 ? cur.id[0] : quad == 1 ? cur.id[1] : quad == 2 ? cur.id[2] : cur.id[3];
            const bool valid = my_id >= 0;
            rows.template load<false>(a, sub);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (i >= NPAIR) break;
                if (!mbar_wait(&sm.empty[i], (done & 1u) ^ 1u, s_abort)) fail = 53;
                if (r0 < held) {
#pragma unroll
                    for (int k = 0; k < 2; k++)
                        if (2 * i + k < NP) rows.store(smem + (2 * i + k) * AK_PANEL, 2 * i + k, 2 * i + k == NP - 1, r0, sub);
                }
                proxy_fence();
                mbar_arrive_warp(&sm.full[i], lane);
            }
            // the tile after this one: half of its rows are on their way while the scores are worked on (all of them, and the
            // scores, are more registers than a thread has)
            more = false;
            for (tile += C; tile < n_tiles; tile += C) {
                cur.load(a, ids, tile, lane);
                if ((more = cur.any(a))) break;
            }
            if (more) {
                rows.find(a, seq, cur, warp, lane);
                rows.template load<true>(a, sub);
            }

            if (!mbar_wait(&sm.s_full, done & 1u, s_abort)) fail = 54;
            __syncwarp();
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            uint32_t s[32];
            tmem_ld32(tmem_s + lanes + half * 32, s);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            const float4 *mp = reinterpret_cast<const float4 *>(sm.m + half * 32);
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float4 m = mp[i];
                top = fmaxf(top, fmaxf(fmaxf(fmaf(__uint_as_float(s[4 * i]), cs, -m.x), fmaf(__uint_as_float(s[4 * i + 1]), cs, -m.y)),
                                       fmaxf(fmaf(__uint_as_float(s[4 * i + 2]), cs, -m.z), fmaf(__uint_as_float(s[4 * i + 3]), cs, -m.w))));
            }
            if (workers_any(valid && top > AK_SLACK)) {
                // new references: the maxima over the tokens so far
                float keep = AK_NONE;
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    const float r = redux_max(valid ? __uint_as_float(s[i]) * cs : -INFINITY);
                    if (lane == i) keep = r;
                }
                sm.part[quad][half * 32 + lane] = keep;
                workers_sync();
                if (tid < AK_HEADS) {
                    const float old = sm.m[tid];
                    const float now = fmaxf(fmaxf(fmaxf(sm.part[0][tid], sm.part[1][tid]), fmaxf(sm.part[2][tid], sm.part[3][tid])), old);
                    sm.m[tid] = now;
                    sm.f[tid] = ex2(old - now);
                }
                workers_sync();
                const float *f = sm.f + half * 32;
#pragma unroll
                for (int i = 0; i < 32; i++) l[i] *= f[i];
                if (done) {
                    for (int i = 0; i < NPAIR; i++) {
                        uint32_t v[32];
                        tmem_ld32(tmem + lanes + i * AK_HEADS + half * 32, v);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int k = 0; k < 32; k++) v[k] = __float_as_uint(__uint_as_float(v[k]) * f[k]);
                        tmem_st32(tmem + lanes + i * AK_HEADS + half * 32, v);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
            }
            uint8_t *prow = smem + AK_P_OFF + token * 128;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const float4 m = mp[2 * c + k];
                    const int i = 8 * c + 4 * k;
                    const float p0 = valid ? ex2(fmaf(__uint_as_float(s[i]), cs, -m.x)) : 0.f;
                    const float p1 = valid ? ex2(fmaf(__uint_as_float(s[i + 1]), cs, -m.y)) : 0.f;
                    const float p2 = valid ? ex2(fmaf(__uint_as_float(s[i + 2]), cs, -m.z)) : 0.f;
                    const float p3 = valid ? ex2(fmaf(__uint_as_float(s[i + 3]), cs, -m.w)) : 0.f;
                    w[2 * k] = bf16x2_rn(p0, p1);
                    w[2 * k + 1] = bf16x2_rn(p2, p3);
                    // the sum is that of the rounded numerators: the weights then add up to one
                    l[i] += __uint_as_float(w[2 * k] << 16);
                    l[i + 1] += __uint_as_float(w[2 * k] & 0xffff0000u);
                    l[i + 2] += __uint_as_float(w[2 * k + 1] << 16);
                    l[i + 3] += __uint_as_float(w[2 * k + 1] & 0xffff0000u);
                }
                *reinterpret_cast<uint4 *>(prow + (((half * 4 + c) ^ (token & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            proxy_fence();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            mbar_arrive_warp(&sm.p_ready, lane);
            if (fail) *s_abort = 1;
            done++;
        }
        if (!mbar_wait(&sm.o_done, 0u, s_abort)) fail = 55;
        if (fail) *s_abort = 1;
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        // sums over the tokens: 32 values in 32 lanes, halved five times, lane i ends with head i
#pragma unroll
        for (int o = 16; o; o >>= 1)
#pragma unroll
            for (int i = 0; i < o; i++) {
                const bool up = lane & o;
                l[i] = (up ? l[i + o] : l[i]) + __shfl_xor_sync(0xffffffffu, up ? l[i] : l[i + o], o);
            }
        sm.part[quad][half * 32 + lane] = l[0];
        workers_sync();
    }

    const uint32_t recv = smem_u32(smem);
    // channels per receiving CTA: whole warps of 32, and the parts of all CTAs fit the panels
    const int slice = (a.d / C + 31) & ~31;
    if (C > 1) {
        cluster_wait();                                  // every CTA of the cluster has started
        if (tid < AK_HEADS) {
            const float sum = (sm.part[0][tid] + sm.part[1][tid]) + (sm.part[2][tid] + sm.part[3][tid]), m = sm.m[tid];
            for (int r = 0; r < C; r++)
                asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};"
                             ::"r"(cluster_addr(smem_u32(&sm.ml[rank][tid]), r)), "f"(m), "f"(sum) : "memory");
        }
        cluster_arrive();
        cluster_wait();                                  // all references and sums are in, all panels have been read
    } else if (tid < AK_HEADS) {
        sm.ml[0][tid] = make_float2(sm.m[tid], (sm.part[0][tid] + sm.part[1][tid]) + (sm.part[2][tid] + sm.part[3][tid]));
    }
    if (tid < AK_HEADS) {
        const float sk = a.sink && tid < nh ? a.sink[h0 + tid] : -INFINITY, sk2 = sk * LOG2E;
        float top = fmaxf(sk2, AK_NONE);
        for (int r = 0; r < C; r++) top = fmaxf(top, sm.ml[r][tid].x);
        float den = ex2(sk2 - top);
        for (int r = 0; r < C; r++) den += sm.ml[r][tid].y * ex2(sm.ml[r][tid].x - top);
        sm.f[tid] = sk2 == INFINITY || den == 0.f ? 0.f : ex2(sm.ml[rank][tid].x - top) / den;
    }
    __syncthreads();
    const size_t o_at = ((size_t)row * a.h + h0) * a.d;
    if (warp < 8) {
        const int quad = warp & 3, half = warp >> 2;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        for (int i = 0; i < NPAIR; i++) {
            const int ch = i * 128 + quad * 32 + lane;
            if (ch - lane >= a.d) break;
            float v[32];
            if (done) {
                uint32_t raw[32];
                tmem_ld32(tmem + lanes + i * AK_HEADS + half * 32, raw);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int k = 0; k < 32; k++) v[k] = __uint_as_float(raw[k]) * sm.f[half * 32 + k];
            } else {
#pragma unroll
                for (int k = 0; k < 32; k++) v[k] = 0.f;
            }
            if (C == 1) {
                if (!*s_abort) ak_put(a, o_at, ch, half * 32, nh, v, lane);
            } else {
                const int to = ch / slice;
                const uint32_t base = cluster_addr(recv, to) + ((uint32_t)rank * slice + (ch - to * slice)) * (AK_HEADS * 4);
#pragma unroll
                for (int k = 0; k < 8; k++)
                    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};"
                                 ::"r"(base + (((half * 8 + k) ^ (lane & 15)) << 4)), "f"(v[4 * k]), "f"(v[4 * k + 1]), "f"(v[4 * k + 2]),
                                   "f"(v[4 * k + 3]) : "memory");
            }
        }
    }
    if (C > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();                                  // the parts of this CTA's channels are in; nothing remote after this
        if (warp < 8 && !*s_abort) {
            for (int u = warp; u < slice / 32 * 16; u += 8) {
                const int local = (u >> 4) * 32 + lane, ch = rank * slice + local, hc = u & 15;
                if (ch - lane >= a.d) break;
                float v[4] = {0.f, 0.f, 0.f, 0.f};
                for (int r = 0; r < C; r++) {
                    const float4 x = *reinterpret_cast<const float4 *>(smem + ((size_t)r * slice + local) * (AK_HEADS * 4) + ((hc ^ (lane & 15)) << 4));
                    v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
                }
                ak_put(a, o_at, ch, hc * 4, nh, v, lane);
            }
        }
    }
    if (fail) {
        atomicCAS(a.status, 0, fail);
        for (int i = 0; i < 2000; i++) __nanosleep(1000);   // MMAs already issued end
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 8)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// CTAs per query row, and tokens per tile.  `slots`: clusters of 1, 2, 4, 8 and 16 CTAs that the GPU holds at once.
void attn_kv8_shape(int idxw, long long rows, const int (&slots)[5], int *cluster, int *unit) {
    double best = 0;
    *cluster = 1;
    *unit = 16;
    for (int i = 0; i < 5; i++) {
        const int C = 1 << i;
        if (slots[i] < 1) continue;
        const int k = idxw > AK_TILE * C ? (idxw + AK_TILE * C - 1) / (AK_TILE * C) : 1;      // tiles of the CTA with the most
        const int u = idxw ? ((idxw + C * k - 1) / (C * k) + 15) & ~15 : 16;
        const double waves = (double)((rows + slots[i] - 1) / slots[i]);
        const double t = waves * (3.0 + (C > 1 ? 2.0 : 0.0) + k * (1.0 + u / 128.0 * 1.5));
        if (i == 0 || t < best) { best = t; *cluster = C; *unit = u; }
    }
}

struct AkDevice { int slots[2][5]; bool ready; };
// Sets the kernel's attributes on the current device and asks how many clusters of each size it holds, once per device.
const AkDevice *ak_device() {
    static std::mutex mu;
    static AkDevice at[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { set_error("sparse_attn_kv8: no current device"); return nullptr; }
    std::lock_guard<std::mutex> lock(mu);
    AkDevice &d = at[dev];
    if (d.ready) return &d;
    for (int tail = 0; tail < 2; tail++) {
        const void *f = tail ? (const void *)attn_kv8_kernel<true> : (const void *)attn_kv8_kernel<false>;
        if (ensure_dyn_smem(f, AK_SMEM)) return nullptr;
        if (cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) cudaGetLastError();
        for (int i = 0; i < 5; i++) {
            cudaLaunchConfig_t cfg;
            memset(&cfg, 0, sizeof cfg);
            cudaLaunchAttribute c;
            c.id = cudaLaunchAttributeClusterDimension;
            c.val.clusterDim.x = 1u << i; c.val.clusterDim.y = 1; c.val.clusterDim.z = 1;
            cfg.gridDim = dim3(1u << i); cfg.blockDim = dim3(AK_THREADS); cfg.dynamicSmemBytes = AK_SMEM;
            cfg.attrs = &c; cfg.numAttrs = 1;
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, f, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
            d.slots[tail][i] = n;
        }
        if (d.slots[tail][0] < 1) { set_error("sparse_attn_kv8: the kernel does not fit the device"); return nullptr; }
    }
    d.ready = true;
    return &d;
}

int attn_kv8(AttnKv8Args a, cudaStream_t st) {
    const AkDevice *dev = ak_device();
    a.status = wait_word();
    if (!dev || !a.status) return 1;
    const unsigned hb = (unsigned)ceil_div(a.h, AK_HEADS);
    attn_kv8_shape(a.idxw, (long long)a.rows * hb, dev->slots[a.rd != 0], &a.cluster, &a.unit);
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)a.cluster; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)a.rows * (unsigned)a.cluster, hb); cfg.blockDim = dim3(AK_THREADS);
    cfg.dynamicSmemBytes = AK_SMEM; cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    APUS_CUDA_OK(a.rd ? cudaLaunchKernelEx(&cfg, attn_kv8_kernel<true>, a) : cudaLaunchKernelEx(&cfg, attn_kv8_kernel<false>, a));
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
                           scale, q_bf16 != 0, o_bf16 != 0, 1, 16, nullptr};
    return attn_kv8(a, (cudaStream_t)stream);
}
