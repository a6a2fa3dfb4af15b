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
    int cluster, unit;           // CTAs per query row, tokens per tile (a multiple of 16 up to 112)
    int ahead;                   // rows that the GPU works on at once
    float *part;                 // [CTA]: O^T of a part as [64][d], then its 64 references and sums; where a row has several CTAs
    int *status;
};

// Where a sequence's records lie: id i below na at a + i * bytes, others at b + i * bytes.
struct Kv8Seq {
    uintptr_t a, b;
    int na, n;                                          // ids from n on are holes
    uint32_t bytes;
    __device__ __forceinline__ Kv8Seq(const AttnKv8Args &p, long long seq) {
        bytes = (uint32_t)kv8_row_bytes(p.d, p.rd);
        a = (uintptr_t)p.kv_a + (uintptr_t)(seq * p.a_stride) * bytes;
        b = (uintptr_t)p.kv_b + (uintptr_t)(seq * p.b_stride - p.na) * bytes;
        na = (int)p.na;
        n = (int)(p.na + p.nb);
    }
    __device__ __forceinline__ const uint8_t *at(int id) const {      // id not a hole
        return reinterpret_cast<const uint8_t *>((id < na ? a : b) + (uintptr_t)(uint32_t)id * bytes);
    }
};
__device__ __forceinline__ uint4 ldg16(const uint8_t *p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// 16 or 4 bytes of global memory, or zeros; here and not where the value is first used, and without a branch
__device__ __forceinline__ uint4 ldg16_if(const uint8_t *p, bool yes) {
    uint4 v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
                 "@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
                 : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"((uint32_t)yes));
    return v;
}
__device__ __forceinline__ uint32_t ldg4_if(const uint8_t *p, bool yes) {
    uint32_t v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.u32 %0, 0;\n\t@p ld.global.u32 %0, [%1];\n\t}"
                 : "=&r"(v) : "l"(p), "r"((uint32_t)yes));
    return v;
}

// ---- the kernel ------------------------------------------------------------------------------------------------------
// One query row has 64 heads on the same latent rows: 225 operations for every byte of a record (4 x 64 x 512 over 583), where
// this GPU's ratio of tensor rate to memory rate is 253 and that of its FP32 pipes some 10.  So both contractions go to the
// tensor cores (tcgen05, BF16 operands, f32 sums), a cache row is fetched and dequantised once for all heads of a CTA, and it
// serves as key and as value from the same place:
//
//   S^T[token, head]   = K[token, ch] Q[head, ch]^T     A = 128 rows as they lie (K-major),  B = the queries
//   O^T[ch, head]     += V[token, ch]^T P[token, head]   A = the same rows (MN-major),         B = the numerators
//
// With tokens, then channels as the 128 rows of an instruction, the heads are its columns (64, 32 or 16 in a CTA:
// attn_kv8_shape).  The scores of a short tile (a CTA's share may be 16 tokens) leave rows of theirs unused, the output does not:
// its rows are channels, and its steps end with the tokens.  A group of codes times its power of two is a BF16 value exactly (4
// significant bits), so nothing is rounded before the products.  A token is a TMEM lane, so that a thread turns one token's
// scores into numerators for 32 heads and stores them as one contiguous piece of a row of P.
//
// The softmax is one pass with a reference per head instead of the running maximum: it is set AK_ABOVE powers of two above
// the first tile's maximum and stays until a score exceeds it by more than AK_SLACK of them, which in f32 and BF16, floating
// as both are, costs no precision: numerators of 2^-48 to 2^64 are as good as those around 1, and what is below 2^-126 is
// less than 2^-77 of the largest one.  Only then is the accumulator scaled, which takes 3,000 to 4,000 cycles, by a factor
// that f32 may not hold: at 2^-126, numerators of 2^64 before still are 2^-14 of the new largest one.  So it is applied as
// two.  (With the reference at the maximum itself, heads whose scores spread over some 50 powers
// of two set it anew in three of nineteen tiles: 1,024 rows of 640 candidates 223 us, 208 so; one row of 8,320 33.1 and 30.1.)
// Where a row has values of 2^32 or more, numerators of 2^64 would take the sums out of f32: from there on references are set
// so that no numerator is above 1, as in a softmax with the maximum at hand.  Sums of numerators stay in each thread until the
// end.
//
// A row's candidates are cut into tiles of at most 112, dealt in turn to the CTAs of a cluster.  At the end every CTA writes
// its part of O^T, its references and its sums to scratch, meets the others in a cluster barrier and adds up the parts of
// its share of the heads in rank order: one launch, the same bits every time.  Through L2, which takes 3,300 cycles to write
// and 3,200 to 6,800 to read 128 KB per SM; distributed shared memory moved 15 bytes a cycle into an SM, 8,700 cycles.
//
// Warps 0 to 7: softmax, two threads per token, half of the heads each (one thread with all 64: the numerators 500 cycles
// later, a tile 4 % slower).  Warps 8 to 21: rows, fetched into registers a tile ahead and dequantised into shared memory,
// the first seven of them panels 0 to 3, the others the rest: while one group waits for room to issue its loads, the other
// one dequantises.  Warp 22 issues the MMAs.  Shared memory: 8 panels of 112 tokens x 64 channels (128-byte swizzled rows),
// Q as 8 panels of the heads x 64 channels, P.  112 tokens and not the 128 of an instruction, because a load in flight
// occupies L1, and L1 is what shared memory leaves of 256 KB: with more than 195 KB of shared memory 28 KB are left, and
// gathered rows arrive at 3.4 TB/s over the GPU; with 60 KB, at 6.6.  (The 16 rows that an instruction reads behind a panel
// are the next panel's; what comes of them is masked.)
//
// A tile takes 3.2 to 3.5 us with 64 heads (2.8 to 3.1 with 32, 2.8 with 16; lists of 5 to 35 tiles), 6,200 cycles by ncu's
// count.  In 4,000 of them shared memory is busy: 60 MMAs read 6 KB each at 128 bytes a cycle, and the rows' 112 KB are written
// while the MMAs of the tile before, panel pair by panel pair, leave their place.  In the other 2,200 the tensor cores wait for the
// numerators.  (Two tiles of 64 and 48 tokens in turn, the one's scores under the other's softmax, took 7,300 where it was 6,300
// so: an instruction of 64 rows takes as long as one of 128.)
constexpr int AK_TILE = 112, AK_HEADS = 64;             // of the largest CTA
constexpr int AK_SOFT = 8, AK_ROWS = AK_TILE / 16, AK_MMA = AK_SOFT + 2 * AK_ROWS, AK_THREADS = 32 * (AK_MMA + 1);   // warps by role
constexpr int AK_PANEL = AK_TILE * 128, AK_Q_OFF = 8 * AK_PANEL;
constexpr int AK_MOST_PARTS = 1024;                     // 135 MB of scratch
constexpr uint32_t AK_SLACK = 64;                       // 2^30 products of such a numerator and a value of up to 2^32 stay in f32
constexpr float AK_ABOVE = 48.f, AK_NONE = -3.402823466e38f, LOG2E = 1.4426950408889634f;

struct AkMisc {
    alignas(16) float m[AK_HEADS];
    alignas(16) float f[AK_HEADS];
    alignas(16) float part[AK_SOFT][AK_HEADS];
    uint64_t full[4], empty[4], q_full, s_full, p_ready, o_done;
    uint32_t tmem;
    int abort, large;                                   // large: a row with values of 2^32 or more has been fetched
};
// What depends on the heads of a CTA.
template <int H>
struct Ak {
    static constexpr int ASK = (H * KV8_MAX_D / 8 + 32 * AK_MMA - 1) / (32 * AK_MMA);   // pieces of 8 query channels per thread
    static constexpr int W = H / 2;                      // heads of a softmax thread
    static constexpr int QPANEL = H * 128, P_OFF = AK_Q_OFF + 8 * QPANEL, P_ROW = H * 2, MISC_OFF = P_OFF + 128 * P_ROW;
    static constexpr int SMEM = MISC_OFF + (int)sizeof(AkMisc);
    static constexpr int COLUMNS = H == 64 ? 512 : H == 32 ? 256 : 128;                 // of tensor memory: 4 H of O^T, H of S^T
    // a row of P fills 128, 64 or 32 bytes and is swizzled as wide: its 16-byte pieces by these bits of its address
    static __device__ __forceinline__ int p_swizzle(int token) { return (token * P_ROW >> 7) & (H / 8 - 1); }
    static_assert(SMEM <= 195 * 1024, "shared memory that leaves 60 KB of L1");
    static_assert(H * KV8_MAX_D * 4 <= P_OFF, "the output as f32 in the place of panels and queries");
};

// barriers of the softmax warps
__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool soft_any(bool p) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)p) : "memory");
    return r != 0;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// A wait of a whole warp, which goes on together; false when it ran out or another one did.  One loop, not unrolled, like the
// others below: this kernel's roles run through their code once per tile, and what the instruction caches do not hold they
// wait for.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    const uint32_t addr = smem_u32(bar);
    unsigned long long t0 = 0;
    uint32_t ok = 0;
#pragma unroll 1
    for (uint32_t it = 1; !ok; it++) {
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(addr), "r"(parity) : "memory");
        if (!ok && (it & 255u) == 0u) {
            const unsigned long long now = global_ns();
            if (!t0) t0 = now;
            if (*abort_flag || now - t0 > TC_WAIT_BUDGET_NS) break;
        }
    }
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float lg2(float x) {
    float r;
    asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Squares of eight BF16 values added to two sums.  Rounding keeps order, so a sum is not below any of its squares: 2^64 or more
// (or NaN) where a value is 2^32 or more.  One instruction for two values, where magnitudes and their maximum take two.
__device__ __forceinline__ uint32_t squares_bf16x2(uint32_t s, const uint4 &v) {
    asm("fma.rn.bf16x2 %0, %1, %1, %0;\n\tfma.rn.bf16x2 %0, %2, %2, %0;\n\tfma.rn.bf16x2 %0, %3, %3, %0;\n\tfma.rn.bf16x2 %0, %4, %4, %0;"
        : "+r"(s) : "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w));
    return s;
}
__device__ __forceinline__ void ak_ld(uint32_t taddr, uint32_t (&v)[32]) { tmem_ld32(taddr, v); }
__device__ __forceinline__ void ak_ld(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void ak_ld(uint32_t taddr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void ak_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ak_st(uint32_t taddr, const uint32_t (&v)[32]) {
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
__device__ __forceinline__ void ak_st(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                   "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void ak_st(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// kind::f16, BF16 operands, f32 sums, 128 x heads x 16; `mn`: both operands MN-major
__device__ __forceinline__ uint32_t ak_idesc(int heads, bool mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (mn ? (1u << 15) | (1u << 16) : 0u) | ((uint32_t)(heads >> 3) << 17) |
           ((uint32_t)(128 >> 4) << 24);
}
// Issued by one lane of a whole, converged warp: with no branch around it the descriptors stay in uniform registers.
__device__ __forceinline__ void ak_mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void ak_commit(uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
        ::"r"(smem_u32(bar)) : "memory");
}
// MN-major operand, a row of `width` bytes per k, swizzled as wide (128, 64 or 32); where M goes on, a panel further
__device__ __forceinline__ uint64_t ak_desc_mn(uint32_t saddr, int width) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(AK_PANEL >> 4) << 16 | (uint64_t)(8 * width >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)(width == 128 ? 2 : width == 64 ? 4 : 6) << 61;
}

// 2^(scale s - reference).  The product is rounded as it was when the reference was set from it: left exact, in one instruction,
// it is some powers of two above or below from 2^27 on, and more than f32 holds from 2^31 on.  (1,024 rows of 640 candidates: one
// instruction 203.4 us, two 204.1.)
__device__ __forceinline__ float ak_numerator(uint32_t s, float cs, float reference) {
    return ex2(__fsub_rn(__fmul_rn(__uint_as_float(s), cs), reference));
}

// Where a channel of a panel of codes lies (codes_bf16x4): queries and output channels follow it.
__device__ __forceinline__ int ak_order(int ch) { return (ch & ~3) | (ch & 1) << 1 | (ch >> 1 & 1); }
// 16 codes of a group with scale byte `b` -> 16 BF16 values.  2^120 times the scale is a BF16 value up to byte 134 (rows of
// magnitude 57,344); what larger ones are above that is made up for afterwards (TileRows::enlarge).
__device__ __forceinline__ void dequant16(const uint4 c, uint32_t b, uint4 &lo, uint4 &hi) {
    const uint32_t f = code_factor(min(b, 134u));
    const uint2 w0 = codes_bf16x4(c.x, f), w1 = codes_bf16x4(c.y, f), w2 = codes_bf16x4(c.z, f), w3 = codes_bf16x4(c.w, f);
    lo = make_uint4(w0.x, w0.y, w1.x, w1.y);
    hi = make_uint4(w2.x, w2.y, w3.x, w3.y);
}
// 16 bytes to shared memory.  No memory clobber: the loads that follow in the program need not wait for it (every use of what
// is stored lies behind a fence or a barrier that has one).
__device__ __forceinline__ void sts16(void *p, const uint4 &v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(p)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w));
}

// The ids of a tile, token 32 k + lane in id[k]; whether any of them names a record is the same in every warp.
struct TileIds {
    int id[4];
    __device__ __forceinline__ void load(const AttnKv8Args &a, const int32_t *ids, int tile, int lane) {
        const int t0 = tile * a.unit, t1 = min(t0 + a.unit, a.idxw);
#pragma unroll
        for (int k = 0; k < 4; k++) id[k] = t0 + 32 * k + lane < t1 ? ids[t0 + 32 * k + lane] : -1;
    }
    __device__ __forceinline__ bool any(int n) {
#pragma unroll
        for (int k = 0; k < 4; k++) id[k] = id[k] < n ? id[k] : -1;
        return __any_sync(0xffffffffu, max(max(id[0], id[1]), max(id[2], id[3])) >= 0);
    }
};

// What a lane of the row warps holds of a tile: of its rows r0 and r0 + 8, 16 channels of each of its group's four panels, as
// they were fetched (codes in the first half of v, or the BF16 values of the rotated panel) and then as BF16 values.
template <bool TAIL>
struct TileRows {
    uint4 v[4][2][2];                                   // panel, row, half
    uint4 v1[2];                                        // as fetched: the second half of the rotated panel, row
    uint32_t sc[2];
    // `from`: of this lane's bytes in the group's first panel; the first n_codes panels hold codes, the n-th may be rotated
    __device__ __forceinline__ void load(const Kv8Seq &at, const TileIds &ids, int w, int lane, int from, int scales, int n_codes, int n) {
        const int src = (w & 1) * 16 + (lane >> 2), sub = lane & 3;
        const int mine = w >> 1 == 0 ? ids.id[0] : w >> 1 == 1 ? ids.id[1] : w >> 1 == 2 ? ids.id[2] : ids.id[3];
        const uint8_t *rec[2];
        bool is[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int id = __shfl_sync(0xffffffffu, mine, src + 8 * i);
            is[i] = id >= 0;
            rec[i] = at.at(id);
            sc[i] = ldg4_if(rec[i] + scales, is[i]);
        }
        // no branches: every register gets a value, or the loops around this would keep old ones
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < 2; i++) v[j][i][0] = ldg16_if(rec[i] + from + j * 64 + (TAIL && j >= n_codes ? sub * 16 : 0), is[i] && j < n);
        if (TAIL)
#pragma unroll
            for (int i = 0; i < 2; i++) v1[i] = ldg16_if(rec[i] + from + n_codes * 64 + sub * 16 + 16, is[i] && n_codes < n);
    }
    __device__ __forceinline__ void convert(int i2, int n_codes, volatile int *large) {  // panels 2 i2 and 2 i2 + 1
#pragma unroll
        for (int j = 2 * i2; j < 2 * i2 + 2; j++) {
            if (!TAIL || j < n_codes) {
#pragma unroll
                for (int i = 0; i < 2; i++) dequant16(v[j][i][0], sc[i] >> 8 * j & 0xffu, v[j][i][0], v[j][i][1]);
            } else {
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    v[j][i][1] = v1[i];
                    m = squares_bf16x2(squares_bf16x2(m, v[j][i][0]), v[j][i][1]);
                }
                if (max(m & 0xffffu, m >> 16) >= (127u + 64u) << 7) *large = 1;
            }
        }
    }
    // panels 2 i2 and 2 i2 + 1 of the group's n into shared memory; `to`: where this lane's part of row r0 starts in the group's
    // first panel; the halves of its 16 channels go to x0 and x1
    __device__ __forceinline__ void store(uint8_t *to, int i2, int n, int n_codes, int x0, int x1, volatile int *large) const {
#pragma unroll
        for (int j = 2 * i2; j < 2 * i2 + 2; j++)
            if (j < n)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    sts16(to + j * AK_PANEL + i * 1024 + x0, v[j][i][0]);
                    sts16(to + j * AK_PANEL + i * 1024 + x1, v[j][i][1]);
                }
        // the part of a scale above byte 134, on what has been stored (255: NaN)
        const uint32_t top = max_u16x2(max_u16x2(sc[0] & 0x00ff00ffu, sc[0] >> 8 & 0x00ff00ffu), max_u16x2(sc[1] & 0x00ff00ffu, sc[1] >> 8 & 0x00ff00ffu));
        if (__any_sync(0xffffffffu, max(top & 0xffffu, top >> 16) > 134u)) {
            if (max(top & 0xffffu, top >> 16) > 149u) *large = 1;        // a code of up to 2^9 times 2^23
#pragma unroll 1
            for (int k = 0; k < 32; k++) {
                const int j = 2 * i2 + (k >> 4), i = k >> 3 & 1;
                const uint32_t b = (i ? sc[1] : sc[0]) >> 8 * j & 0xffu, p = smem_u32(to + j * AK_PANEL + i * 1024 + (k & 4 ? x1 : x0)) + (k & 3) * 4;
                if (j < n_codes && b > 134u) {
                    uint32_t u;
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(u) : "r"(p));
                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(p), "r"(mul_bf16x2(u, b == 255u ? 0x7fff7fffu : (b - 7u) * 0x00800080u)));
                }
            }
        }
    }
};

// What a reference and the sum of the numerators relative to it add up to, in powers of two: parts and the sink are weighed
// against the largest of these and not against the largest reference, which may be far above all its scores.  So a factor that is
// zero, 2^-126 or less, makes weights zero that are below 2^(AK_SLACK - 126).
__device__ __forceinline__ float ak_weight(float2 v) { return v.x + lg2(v.y); }

// The parts of a row's C CTAs, joined for this CTA's share of the heads: U times 4 channels of a head and R of the parts at a
// time, four or eight loads in flight
template <int U, int R>
__device__ __forceinline__ void ak_join(int C, int H, float *w, const float *parts, int d, const float *sink, void *o, int o_bf16, int rank, int nh) {
    const int per = (nh + C - 1) / C, lo = rank * per, n = min(per, nh - lo), tid = threadIdx.x;
    const uint32_t part_size = H * d + 2 * H;
    if (tid < AK_HEADS) {
        // lane i of a head's C lanes: reference and sum of part i; w [head][part]: what a part is multiplied by, -1 for one
        // without tokens, which has not been written
        const int hd = tid / C, r = tid % C;
        float2 v = make_float2(AK_NONE, 0.f);
        float sk = -INFINITY;
        if (hd < n) {
            v = __ldcg(reinterpret_cast<const float2 *>(parts + r * part_size + H * d) + lo + hd);
            if (sink) sk = sink[lo + hd] * LOG2E;
        }
        float top = fmaxf(fmaxf(ak_weight(v), sk), AK_NONE);
        for (int m = 1; m < C; m <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
        float den = v.y * ex2(v.x - top);
        for (int m = 1; m < C; m <<= 1) den += __shfl_xor_sync(0xffffffffu, den, m);
        den += ex2(sk - top);
        w[tid] = v.x == AK_NONE && v.y == 0.f || sk == INFINITY || den == 0.f ? -1.f : ex2(v.x - top) / den;
    }
    __syncthreads();
    const int per_head = d / 4, total = n * per_head;
#pragma unroll 1
    for (int u0 = tid; u0 < total; u0 += U * AK_THREADS) {
        float s[U][4];
        const uint8_t *p[U];
        const float *f[U];
#pragma unroll
        for (int k = 0; k < U; k++) {
            const int u = min(u0 + k * AK_THREADS, total - 1);
            s[k][0] = s[k][1] = s[k][2] = s[k][3] = 0.f;
            p[k] = reinterpret_cast<const uint8_t *>(parts + lo * d + u * 4);
            f[k] = w + u / per_head * C;
        }
#pragma unroll 1
        for (int r0 = 0; r0 < C; r0 += R) {
            uint4 x[U][R];
#pragma unroll
            for (int k = 0; k < U; k++)
#pragma unroll
                for (int r = 0; r < R; r++) x[k][r] = ldg16_if(p[k] + (r0 + r) * (part_size * 4), !(f[k][r0 + r] < 0.f));
#pragma unroll
            for (int k = 0; k < U; k++)
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const float g = f[k][r0 + r];
                    s[k][0] += g * __uint_as_float(x[k][r].x); s[k][1] += g * __uint_as_float(x[k][r].y);
                    s[k][2] += g * __uint_as_float(x[k][r].z); s[k][3] += g * __uint_as_float(x[k][r].w);
                }
        }
#pragma unroll
        for (int k = 0; k < U; k++) {
            const int u = u0 + k * AK_THREADS;
            if (u >= total) break;
            const uint32_t x = bf16x2_rn(s[k][0], s[k][1]), y = bf16x2_rn(s[k][2], s[k][3]);
            const size_t i = (size_t)lo * d + (size_t)u * 4;
            if (o_bf16) *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(o) + i) = make_uint2(x, y);
            else *reinterpret_cast<uint4 *>(static_cast<uint32_t *>(o) + i) = make_uint4(x << 16, x & 0xffff0000u, y << 16, y & 0xffff0000u);
        }
    }
}

template <bool TAIL, int H>
__global__ void __launch_bounds__(AK_THREADS, 1)
attn_kv8_kernel(const AttnKv8Args a) {
    APUS_PDL_GO();
    using K = Ak<H>;
    constexpr int W = K::W;
    extern __shared__ __align__(1024) uint8_t smem[];
    AkMisc &sm = *reinterpret_cast<AkMisc *>(smem + K::MISC_OFF);
    volatile int *s_abort = &sm.abort, *s_large = &sm.large;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, C = a.cluster;
    const int rank = (int)(blockIdx.x % (unsigned)C), h0 = (int)blockIdx.y * H, nh = min(H, a.h - h0);
    const uint32_t row = blockIdx.x / (unsigned)C, seq = row / (uint32_t)a.rows_per_seq;
    const Kv8Seq at(a, seq);
    const size_t part_size = H * a.d + 2 * H;
    float *part = a.part + (blockIdx.y * (size_t)gridDim.x + blockIdx.x) * part_size;
    const int32_t *ids = a.idxs + (size_t)row * a.idxw;
    const int n_tiles = (a.idxw + a.unit - 1) / a.unit, NP = a.d / 64, NPAIR = (NP + 1) / 2;

    // The barriers while the kernel before this one may still run, global memory only after it.  Tensor memory too: that
    // kernel's CTAs may have yet to take theirs.
    if (tid == 0) {
#pragma unroll 1
        for (int i = 0; i < 4; i++) { mbar_init(&sm.full[i], AK_ROWS); mbar_init(&sm.empty[i], 1); }
        mbar_init(&sm.q_full, AK_MMA);
        mbar_init(&sm.s_full, 1);
        mbar_init(&sm.p_ready, AK_SOFT);
        mbar_init(&sm.o_done, 1);
        *s_large = 0;
        *s_abort = (smem_u32(smem) & 1023u) != 0;        // the swizzle goes by addresses: code 57, below
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid < H) sm.m[tid] = AK_NONE;
    APUS_PDL_WAIT();

    // What the first tile waits for: its ids, sinks, and the queries, 8 channels at a time, all at once, by all warps but the one
    // of the MMAs.  In the place of heads that there are not a CTA has the first one's queries.
    TileIds cur;                                         // of tile `tile`, which has a record in it while `more`
    int tile = rank;
    cur.load(a, ids, tile, lane);
    uint4 qv[K::ASK][2];
    const int per_head = a.d / 8, q_heads = 32 * AK_MMA / per_head, q_rest = 32 * AK_MMA % per_head;
    int q_head = tid / per_head, q_c = tid % per_head;   // of this thread's next piece
    auto ask = [&]() {
        const uint8_t *q = static_cast<const uint8_t *>(a.q) + ((size_t)row * a.h + h0) * a.d * (a.q_bf16 ? 2 : 4);
        int hd = q_head, c = q_c;
#pragma unroll
        for (int k = 0; k < K::ASK; k++) {
            const uint8_t *p = q + (uint32_t)((hd < nh ? hd * per_head : 0) + c) * (a.q_bf16 ? 16u : 32u);
            qv[k][0] = ldg16(p);
            if (!a.q_bf16) qv[k][1] = ldg16(p + 16);
            hd += q_heads;
            c += q_rest;
            if (c >= per_head) { c -= per_head; hd++; }
        }
    };
    auto place = [&]() {
#pragma unroll
        for (int k = 0; k < K::ASK; k++) {
            uint4 v = qv[k][0];
            if (!a.q_bf16)
                v = make_uint4(bf16x2_rn(__uint_as_float(v.x), __uint_as_float(v.y)), bf16x2_rn(__uint_as_float(v.z), __uint_as_float(v.w)),
                               bf16x2_rn(__uint_as_float(qv[k][1].x), __uint_as_float(qv[k][1].y)),
                               bf16x2_rn(__uint_as_float(qv[k][1].z), __uint_as_float(qv[k][1].w)));
            if (q_c * 8 < a.d - a.rd)                    // in the order of the codes
                v = make_uint4(__byte_perm(v.x, v.y, 0x5410), __byte_perm(v.x, v.y, 0x7632), __byte_perm(v.z, v.w, 0x5410),
                               __byte_perm(v.z, v.w, 0x7632));
            if (q_head < H) sts16(smem + AK_Q_OFF + (q_c >> 3) * K::QPANEL + q_head * 128 + (((q_c & 7) ^ (q_head & 7)) << 4), v);
            q_head += q_heads;
            q_c += q_rest;
            if (q_c >= per_head) { q_c -= per_head; q_head++; }
        }
    };
    if (warp != AK_MMA) ask();
    const float sink = a.sink && tid < nh ? a.sink[h0 + tid] : -INFINITY;        // of head tid

    if (warp == AK_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&sm.tmem)), "r"(K::COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0), tmem_s = tmem + 4 * H;

    // A wait that runs out sets the abort flag, after which every other wait gives up soon; all loops and barriers are gone
    // through all the same, so that no thread is left waiting, and nothing is written.
    int fail = tid == 0 && (smem_u32(smem) & 1023u) ? 57 : 0;
    uint32_t done = 0;                                   // tiles of this CTA so far
    bool more = false;
    auto settle = [&]() {                                // cur has been asked for: the first tile from it on with a record
#pragma unroll 1
        for (more = false; tile < n_tiles; ) {
            if ((more = cur.any(at.n))) break;
            tile += C;
            cur.load(a, ids, tile, lane);
        }
    };
    settle();
    const bool any = more;                               // there is an output to read

    if (warp != AK_MMA) {
        place();
        proxy_fence();
        mbar_arrive_warp(&sm.q_full, lane);
    }
    if (warp == AK_MMA) {
        const uint32_t id_s = ak_idesc(H, false), id_o = ak_idesc(H, true);
        const uint64_t dk = umma_desc_sw128(smem_u32(smem)), dq = umma_desc_sw128(smem_u32(smem + AK_Q_OFF));
        const uint64_t dv = ak_desc_mn(smem_u32(smem), 128), dp = ak_desc_mn(smem_u32(smem + K::P_OFF), K::P_ROW);
        // The queries of the row that a later CTA on this SM may have, into L2 (1,024 rows of 640 candidates: 209.6 us without, 207.0 with)
        if (rank == 0 && lane == 0 && row + (uint32_t)a.ahead < (uint32_t)a.rows) {
            const uint32_t item = a.q_bf16 ? 2u : 4u;
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;"
                         ::"l"(static_cast<const uint8_t *>(a.q) + ((size_t)(row + a.ahead) * a.h + h0) * a.d * item), "r"((uint32_t)nh * a.d * item) : "memory");
        }
        __syncwarp();
        if (!warp_wait(&sm.q_full, 0u, s_abort)) fail = 51;
        while (more) {
            const int ks = (min(a.unit, a.idxw - tile * a.unit) + 15) >> 4;      // steps of 16 tokens that hold any
            tile += C;
            cur.load(a, ids, tile, lane);
#pragma unroll 1
            for (int pn = 0; pn < NP && !fail; pn++) {
                if (!(pn & 1)) {
                    if (!warp_wait(&sm.full[pn >> 1], done & 1u, s_abort)) fail = 52;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                }
                const uint64_t da = dk + pn * (AK_PANEL >> 4), db = dq + pn * (K::QPANEL >> 4);
                if (!fail)
#pragma unroll
                    for (int j = 0; j < 4; j++) ak_mma(tmem_s, da + 2 * j, db + 2 * j, id_s, (pn | j) ? 1u : 0u);
            }
            if (!fail) ak_commit(&sm.s_full);
            if (!fail && !warp_wait(&sm.p_ready, done & 1u, s_abort)) fail = 53;
            if (!fail) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                for (int i = 0; i < NPAIR; i++) {
                    const uint64_t da = dv + 2 * i * (AK_PANEL >> 4);
                    ak_mma(tmem + i * H, da, dp, id_o, done ? 1u : 0u);
#pragma unroll
                    for (int k = 1; k < AK_TILE / 16; k++)
                        if (k < ks) ak_mma(tmem + i * H, da + 128 * k, dp + K::P_ROW * k, id_o, 1u);
                    ak_commit(&sm.empty[i]);
                }
            }
            if (fail) *s_abort = 1;
            done++;
            settle();
        }
        if (!fail) ak_commit(&sm.o_done);
    } else if (warp >= AK_SOFT) {
        const int grp = warp >= AK_SOFT + AK_ROWS, w = warp - AK_SOFT - grp * AK_ROWS, r0 = w * 16 + (lane >> 2), sub = lane & 3;
        const int nq = a.d - a.rd;
        // this group's panels: n of them, the last one rotated or not
        const int n = min(max(NP - 4 * grp, 0), 4), n_codes = min(max(nq / 64 - 4 * grp, 0), 4);
        const int from = 4 * grp * 64 + sub * 16, scales = kv8_scale_off(a.d, a.rd) + 4 * grp;
        uint8_t *to = smem + 4 * grp * AK_PANEL + r0 * 128;
        const int x0 = ((2 * sub) ^ (r0 & 7)) * 16, x1 = ((2 * sub + 1) ^ (r0 & 7)) * 16;
        TileRows<TAIL> rows;
        if (n && more) rows.load(at, cur, w, lane, from, scales, n_codes, n);
        while (n && more) {
            const int held = (min(a.unit, a.idxw - tile * a.unit) + 15) & ~15;   // rows that the MMAs read
            tile += C;
            cur.load(a, ids, tile, lane);
            rows.convert(0, n_codes, s_large);           // before there is room for it, while the tile before is worked on
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (2 * i >= n) break;
                if (!warp_wait(&sm.empty[2 * grp + i], (done & 1u) ^ 1u, s_abort)) fail = 54;
                if (w * 16 < held) rows.store(to, i, n, n_codes, x0, x1, s_large);
                proxy_fence();
                mbar_arrive_warp(&sm.full[2 * grp + i], lane);
                if (i == 0) rows.convert(1, n_codes, s_large);   // while the MMAs work on the first ones
            }
            // The next tile's rows, all at once: between the stores above their issue would hold up the second one, and the MMAs
            // that wait for it.
            settle();
            if (more) rows.load(at, cur, w, lane, from, scales, n_codes, n);
            if (fail) *s_abort = 1;
            done++;
        }
    } else {
        // a thread has one token and half of the heads
        const int quad = warp & 3, hh = (warp >> 2) * W, token = tid & 127;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const float cs = a.scale * LOG2E;
        // sums of numerators: of 8 heads, over the few tokens in a row that this thread adds up of every tile
        constexpr int PIECES = H / 8, TOKENS = H / 16;
        const int lh = tid & (PIECES - 1), lt = tid / PIECES * TOKENS;
        float l[8];
#pragma unroll
        for (int i = 0; i < 8; i++) l[i] = 0.f;
        uint8_t *prow = smem + K::P_OFF + token * K::P_ROW;
        const float4 *mp = reinterpret_cast<const float4 *>(sm.m + hh);
        while (more) {
            const bool valid = (quad == 0 ? cur.id[0] : quad == 1 ? cur.id[1] : quad == 2 ? cur.id[2] : cur.id[3]) >= 0;
            const uint32_t mask = valid ? ~0u : 0u;      // not a choice: the compiler would branch around every numerator
            tile += C;
            cur.load(a, ids, tile, lane);
            // One warp polls: the issue slots are the row warps'.  It waits for the rows, too, for what they say about their values.
            // Behind this the numerators of the tile before have been added up.
            if (warp == 0) {
#pragma unroll 1
                for (int i = 0; i <= NPAIR; i++)
                    if (!warp_wait(i < NPAIR ? &sm.full[i] : &sm.s_full, done & 1u, s_abort)) fail = 55;
            }
            soft_sync();
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t most = (127u + (*s_large ? 0u : AK_SLACK)) << 7;
            for (bool set = done == 0;; set = true) {
                uint32_t s[W];
                ak_ld(tmem_s + lanes + hh, s);
                ak_ld_wait();
                if (set) {
                    // New references from the maxima over the tokens so far, folded over the lanes, after which lane i has that of
                    // this warp's head i.
#pragma unroll
                    for (int i = 0; i < W; i++) s[i] = (__float_as_uint(__uint_as_float(s[i]) * cs) & mask) | (0xff800000u & ~mask);
#pragma unroll
                    for (int o = W / 2; o; o >>= 1)
#pragma unroll
                        for (int i = 0; i < o; i++) {
                            const bool up = lane & o;
                            s[i] = __float_as_uint(fmaxf(__uint_as_float(up ? s[i + o] : s[i]), __uint_as_float(__shfl_xor_sync(0xffffffffu, up ? s[i] : s[i + o], o))));
                        }
#pragma unroll
                    for (int o = W; o < 32; o <<= 1)
                        s[0] = __float_as_uint(fmaxf(__uint_as_float(s[0]), __uint_as_float(__shfl_xor_sync(0xffffffffu, s[0], o))));
                    if (lane < W) sm.part[quad][hh + lane] = __uint_as_float(s[0]);
                    soft_sync();
                    if (tid < H) {
                        const float old = sm.m[tid];
                        const float now = fmaxf(fmaxf(fmaxf(sm.part[0][tid], sm.part[1][tid]), fmaxf(sm.part[2][tid], sm.part[3][tid])) + AK_ABOVE, old);
                        sm.m[tid] = now;
                        sm.f[tid] = ex2(0.5f * (old - now));     // its square is the factor, which may be below 2^-126
                    }
                    soft_sync();
                    if (done) {
                        const float4 *f = reinterpret_cast<const float4 *>(sm.f + hh);
#pragma unroll
                        for (int i = 0; i < 8; i++) { const float g = sm.f[8 * lh + i]; l[i] = l[i] * g * g; }
#pragma unroll 1
                        for (int i = 0; i < NPAIR; i++) {
                            const uint32_t o = tmem + lanes + i * H + hh;
                            ak_ld(o, s);
                            ak_ld_wait();
#pragma unroll
                            for (int k = 0; k < W / 4; k++) {
                                const float4 g = f[k];
                                s[4 * k] = __float_as_uint(__uint_as_float(s[4 * k]) * g.x * g.x);
                                s[4 * k + 1] = __float_as_uint(__uint_as_float(s[4 * k + 1]) * g.y * g.y);
                                s[4 * k + 2] = __float_as_uint(__uint_as_float(s[4 * k + 2]) * g.z * g.z);
                                s[4 * k + 3] = __float_as_uint(__uint_as_float(s[4 * k + 3]) * g.w * g.w);
                            }
                            ak_st(o, s);
                        }
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    }
                    ak_ld(tmem_s + lanes + hh, s);       // again: registers are few
                    ak_ld_wait();
                }
                // all references before the first store: a load behind a store waits for it to issue, one piece after another
                uint32_t top = 0, w[W / 2];              // the largest numerator: as BF16 bits they compare like numbers
#pragma unroll
                for (int c = 0; c < W / 4; c++) {
                    const float4 r = mp[c];
                    w[2 * c] = mask & bf16x2_rn(ak_numerator(s[4 * c], cs, r.x), ak_numerator(s[4 * c + 1], cs, r.y));
                    w[2 * c + 1] = mask & bf16x2_rn(ak_numerator(s[4 * c + 2], cs, r.z), ak_numerator(s[4 * c + 3], cs, r.w));
                    top = max_u16x2(top, max_u16x2(w[2 * c], w[2 * c + 1]));
                }
#pragma unroll
                for (int c = 0; c < W / 8; c++)
                    sts16(prow + ((((hh >> 3) + c) ^ K::p_swizzle(token)) << 4), make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]));
                // a numerator above 2^AK_SLACK, or above 1 where values are large: once more with new references
                if (!soft_any(max(top & 0xffffu, top >> 16) > most) || set) break;
            }
            proxy_fence();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            mbar_arrive_warp(&sm.p_ready, lane);
            // while the MMAs run: the sums of the numerators, as they were rounded, so that the weights add up to one
#pragma unroll
            for (int k = 0; k < TOKENS; k++) {
                const uint4 w = *reinterpret_cast<const uint4 *>(smem + K::P_OFF + (lt + k) * K::P_ROW + ((lh ^ K::p_swizzle(lt + k)) << 4));
                l[0] += __uint_as_float(w.x << 16); l[1] += __uint_as_float(w.x & 0xffff0000u);
                l[2] += __uint_as_float(w.y << 16); l[3] += __uint_as_float(w.y & 0xffff0000u);
                l[4] += __uint_as_float(w.z << 16); l[5] += __uint_as_float(w.z & 0xffff0000u);
                l[6] += __uint_as_float(w.w << 16); l[7] += __uint_as_float(w.w & 0xffff0000u);
            }
            if (fail) *s_abort = 1;
            done++;
            settle();
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
#pragma unroll
            for (int o = PIECES; o < 32; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
            if (lane < PIECES) sm.part[warp][8 * lane + i] = l[i];
        }
        soft_sync();
        if (tid < H) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < AK_SOFT; i++) sum += sm.part[i][tid];
            const float m = sm.m[tid];
            if (C > 1) reinterpret_cast<float2 *>(part + H * a.d)[tid] = make_float2(m, sum);
            // the only CTA of its row: what its part is multiplied by, while the last MMAs run
            const float sk = sink * LOG2E, top = fmaxf(fmaxf(ak_weight(make_float2(m, sum)), sk), AK_NONE), den = ex2(sk - top) + sum * ex2(m - top);
            sm.f[tid] = sk == INFINITY || den == 0.f ? 0.f : ex2(m - top) / den;
        }
    }
    // A CTA that writes its part to global memory takes every pair of panels as its MMAs end (a CTA of its own uses the panels'
    // place and waits for all of them); a warp that has not gone through the tiles, because d is small, waits for all too.
    const bool by_pairs = C > 1 && done;
    if (warp < AK_MMA && !by_pairs) {
        if (!warp_wait(&sm.o_done, 0u, s_abort)) fail = 56;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
    if (fail) *s_abort = 1;
    if (C == 1) __syncthreads();

    const size_t o_at = ((size_t)row * a.h + h0) * a.d;
    if (warp < 16 && (any || C == 1)) {
        const int quad = warp & 3, hh = (warp >> 2 & 1) * W;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        constexpr int E = W < 16 ? W : 16;
        const int heads = min(nh - hh, W), item = C == 1 && a.o_bf16 ? 2 : 4;
        // 16 heads at a time and not 32: half the code, which has to be fetched for few rounds of it
#pragma unroll 1
        for (int k0 = 0; k0 < heads; k0 += E) {
            float f[E];
#pragma unroll
            for (int k = 0; k < E; k++) f[k] = sm.f[hh + k0 + k];
#pragma unroll 1
            for (int i = warp >> 3; i < NPAIR; i += 2) {
                const int ch0 = i * 128 + quad * 32;
                if (ch0 >= a.d) break;
                const int ch = ch0 + (ch0 < a.d - a.rd ? ak_order(lane) : lane); // panels of codes have an order of their own
                if (by_pairs && k0 == 0) {
                    if (!warp_wait(&sm.empty[i], (done - 1) & 1u, s_abort)) fail = 56;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                }
                uint32_t v[E];
                if (any) {
                    ak_ld(tmem + lanes + i * H + hh + k0, v);
                    ak_ld_wait();
                }
                if (C > 1) {
                    float *p = part + (hh + k0) * a.d + ch;
#pragma unroll
                    for (int k = 0; k < E; k++, p += a.d)
                        if (k0 + k < heads) __stcg(p, __uint_as_float(v[k]));
                } else {                                 // the output's rows in shared memory, a warp's 32 channels of a head at a time
                    const uint32_t base = smem_u32(smem) + ((hh + k0) * a.d + ch) * item, step = a.d * item;
#pragma unroll
                    for (int k = 0; k < E; k++) {
                        const uint32_t u = any ? bf16x2_rn(0.f, __uint_as_float(v[k]) * f[k]) : 0u;
                        if (a.o_bf16) asm volatile("st.shared.u16 [%0], %1;" ::"r"(base + k * step), "h"((uint16_t)(u >> 16)));
                        else asm volatile("st.shared.u32 [%0], %1;" ::"r"(base + k * step), "r"(u));
                    }
                }
            }
        }
    }
    if (C > 1) {
        // the other CTAs of a row must not join what a wait that ran out has left
        if (fail) *s_abort = 1;
        __syncthreads();
        if (tid < H && *s_abort) reinterpret_cast<float2 *>(part + H * a.d)[tid] = make_float2(NAN, NAN);
        __syncwarp();
        cluster_arrive();
        cluster_wait();                                  // the parts of all CTAs are written
        if (!*s_abort) {
            const float *parts = part - (size_t)rank * part_size, *sinks = a.sink ? a.sink + h0 : nullptr;
            void *o = static_cast<uint8_t *>(a.o) + o_at * (a.o_bf16 ? 2 : 4);
            // as many parts at a time as the pieces of the share leave threads for (16 rows of 640 candidates, 32 heads of 4 CTAs:
            // 16.5 us with four pieces of two parts, 15.6 with two of four)
            if (C > 4) ak_join<1, 8>(C, H, sm.f, parts, a.d, sinks, o, a.o_bf16, rank, nh);
            else if (H < 64 && C == 4) ak_join<H == 16 ? 1 : 2, 4>(C, H, sm.f, parts, a.d, sinks, o, a.o_bf16, rank, nh);
            else ak_join<H == 16 ? 2 : 4, 2>(C, H, sm.f, parts, a.d, sinks, o, a.o_bf16, rank, nh);
        }
    } else {
        proxy_fence();
        __syncthreads();
        // the heads of this CTA are one piece of the output
        if (tid == 0 && !*s_abort) {
            const uint32_t bytes = (uint32_t)(nh * a.d) * (a.o_bf16 ? 2u : 4u);
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n\tcp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;"
                         ::"l"(static_cast<uint8_t *>(a.o) + o_at * (a.o_bf16 ? 2 : 4)), "r"(smem_u32(smem)), "r"(bytes) : "memory");
        }
    }
    if (fail) {
        atomicCAS(a.status, 0, fail);
#pragma unroll 1
        for (int i = 0; i < 2000; i++) __nanosleep(1000);   // MMAs already issued end
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == AK_MMA)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(K::COLUMNS) : "memory");
}

using AkKernel = void (*)(AttnKv8Args);
// A CTA of 64, 32 or 16 heads.  Its times in microseconds, fitted to measurements: start and end; the join of a row's CTAs; a tile
// of 112 tokens beside 1.2 for one of none.
struct AkSize { int heads, smem; AkKernel kernel[2]; double start, join, tile; };
constexpr int AK_SIZES = 3;
const AkSize ak_sizes[AK_SIZES] = {{64, Ak<64>::SMEM, {attn_kv8_kernel<false, 64>, attn_kv8_kernel<true, 64>}, 8.4, 3.9, 1.8},
                                   {32, Ak<32>::SMEM, {attn_kv8_kernel<false, 32>, attn_kv8_kernel<true, 32>}, 6.2, 3.0, 1.5},
                                   {16, Ak<16>::SMEM, {attn_kv8_kernel<false, 16>, attn_kv8_kernel<true, 16>}, 5.8, 2.8, 1.5}};

// Heads of a CTA (which of ak_sizes), CTAs per query row and block of heads, tokens per tile.  `slots`: clusters of 1, 2, 4, 8 and
// 16 CTAs that the GPU holds at once (148, 74, 33, 15 and 7).  Fewer heads per CTA do the work on the candidates' rows once
// more for every block of heads, but where SMs would have nothing to do every step of a row is shorter; more CTAs per row take
// fewer tiles each and have a join.  The rule takes the least of: turns in which the GPU takes all clusters, times start, join and
// tiles of one.  Measured microseconds, 1 / 2 / 4 / 8 / 16 CTAs, * where the rule goes (when its times were fitted, its choice was
// within 1 % of the fastest in 17 of 18 shapes, 5 % behind in one; of these eight it is the fastest in seven, 2 % behind in one).
//                              64 heads per CTA                    32                                  16
//   1 row of 640 candidates   27.1   21.4   18.7   14.2   14.0    23.2   17.8   15.0   11.6   11.9    22.1   16.8   13.5   10.8*  11.1
//   6 of 640                  28.4   22.4   19.7   15.2   15.0    23.6   18.1   15.2   12.0*  23.1    22.4   17.2   13.7   21.0   42.1
//   16 of 640                 29.9   24.1   19.8   29.4   42.9    24.4   19.1   15.4*  33.3   56.3    22.9   17.7   26.2   51.0    104
//   32 of 640                 29.9   24.2   20.0   43.7   73.4    24.5   19.3*  29.1   55.4    113    23.1   33.7   51.3   91.5
//   1,024 of 640             204.1*                                336                                 631
//   1 of 8,320                 249    134   73.7   43.3   28.9     217    117   63.6   37.3   24.6     212    114   61.1   36.2   23.4*
//   32 of 8,320                252    138   78.8*   130    145     222    120    134    187    243     212    224    248    319
//   5 of 128, 8 heads         12.8   12.7   12.7   12.5   12.7    10.8   11.1   10.6   10.9   11.1    10.2*  10.5   10.0   10.4   10.6
int attn_kv8_shape(int idxw, int h, int rows, const int (&slots)[AK_SIZES][5], int *cluster, int *unit, int *ahead) {
    double best = 0;
    int which = 0;
    for (int z = 0; z < AK_SIZES; z++) {
        const AkSize &size = ak_sizes[z];
        const long long units = (long long)rows * ceil_div(h, size.heads);
        for (int i = 0; i < 5; i++) {
            const int C = 1 << i;
            if (slots[z][i] < 1 || (i && units << i > AK_MOST_PARTS)) continue;
            const int k = idxw > AK_TILE * C ? (idxw + AK_TILE * C - 1) / (AK_TILE * C) : 1;  // tiles of the CTA with the most
            const int u = idxw ? ((idxw + C * k - 1) / (C * k) + 15) & ~15 : 16;
            const double turns = (double)((units + slots[z][i] - 1) / slots[z][i]);
            const double t = turns * (size.start + (C > 1 ? size.join + 0.06 * C : 0.0) + k * (1.2 + u / 112.0 * size.tile));
            if (best == 0 || t < best) { best = t; which = z; *cluster = C; *unit = u; *ahead = slots[z][i]; }
        }
    }
    return which;
}

struct AkDevice { int slots[2][AK_SIZES][5]; bool ready; };
// Sets the kernel's attributes on the current device and asks how many clusters of each size it holds, once per device.
const AkDevice *ak_device() {
    static std::mutex mu;
    static AkDevice at[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { set_error("sparse_attn_kv8: no current device"); return nullptr; }
    std::lock_guard<std::mutex> lock(mu);
    AkDevice &d = at[dev];
    if (d.ready) return &d;
    for (int k = 0; k < 2 * AK_SIZES; k++) {
        const int tail = k & 1;
        const AkSize &size = ak_sizes[k >> 1];
        const void *f = (const void *)size.kernel[tail];
        if (ensure_dyn_smem(f, size.smem)) return nullptr;
        if (cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) cudaGetLastError();
        for (int i = 0; i < 5; i++) {
            cudaLaunchConfig_t cfg;
            memset(&cfg, 0, sizeof cfg);
            cudaLaunchAttribute c;
            c.id = cudaLaunchAttributeClusterDimension;
            c.val.clusterDim.x = 1u << i; c.val.clusterDim.y = 1; c.val.clusterDim.z = 1;
            cfg.gridDim = dim3(1u << i); cfg.blockDim = dim3(AK_THREADS); cfg.dynamicSmemBytes = size.smem;
            cfg.attrs = &c; cfg.numAttrs = 1;
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, f, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
            d.slots[tail][k >> 1][i] = n;
        }
        if (d.slots[tail][k >> 1][0] < 1) { set_error("sparse_attn_kv8: the kernel does not fit the device"); return nullptr; }
    }
    d.ready = true;
    return &d;
}

int attn_kv8(AttnKv8Args a, cudaStream_t st) {
    const AkDevice *dev = ak_device();
    a.status = wait_word();
    if (!dev || !a.status) return 1;
    const AkSize &size = ak_sizes[attn_kv8_shape(a.idxw, a.h, a.rows, dev->slots[a.rd != 0], &a.cluster, &a.unit, &a.ahead)];
    const unsigned hb = (unsigned)ceil_div(a.h, size.heads);
    CallScratch scratch(st);
    if (a.cluster > 1 && scratch.get((size_t)a.rows * hb * a.cluster * size.heads * (a.d + 2) * sizeof(float))) return 1;
    a.part = static_cast<float *>(scratch.p);
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)a.cluster; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)a.rows * (unsigned)a.cluster, hb); cfg.blockDim = dim3(AK_THREADS);
    cfg.dynamicSmemBytes = size.smem; cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    APUS_CUDA_OK(cudaLaunchKernelEx(&cfg, size.kernel[a.rd != 0], a));
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
    APUS_REQUIRE(rows >= 0 && idxw >= 0 && idxw <= 1 << 30, "sparse_attn_kv8: %d rows of %d ids", rows, idxw);
    APUS_REQUIRE(rows_per_seq > 0 && rows % rows_per_seq == 0, "sparse_attn_kv8: %d rows are not sequences of %d", rows, rows_per_seq);
    APUS_REQUIRE(na >= 0 && nb >= 0 && na <= INT32_MAX && nb <= INT32_MAX - na, "sparse_attn_kv8: na=%lld, nb=%lld", (long long)na, (long long)nb);
    APUS_REQUIRE(kv_a_stride >= 0 && kv_b_stride >= 0, "sparse_attn_kv8: negative stride");
    APUS_REQUIRE((na == 0 || kv_a) && (nb == 0 || kv_b), "sparse_attn_kv8: no cache");
    APUS_REQUIRE(aligned16(kv_a) && aligned16(kv_b), "sparse_attn_kv8: the caches must start on a 16-byte boundary");
    if (rows == 0) return 0;
    APUS_REQUIRE(q && o && (idxs || idxw == 0), "sparse_attn_kv8: no %s", !q ? "queries" : !o ? "output" : "ids");
    APUS_REQUIRE(aligned16(q) && aligned16(o), "sparse_attn_kv8: queries and output must start on a 16-byte boundary");
    if (ensure_enabled()) return 1;
    const AttnKv8Args a = {q, sink, idxs, kv_a, kv_b, o, na, nb, kv_a_stride, kv_b_stride, h, d, rd, idxw, rows, rows_per_seq,
                           scale, q_bf16 != 0, o_bf16 != 0, 1, 16, 0, nullptr, nullptr};
    return attn_kv8(a, (cudaStream_t)stream);
}
