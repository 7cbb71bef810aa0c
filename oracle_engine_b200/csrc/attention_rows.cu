// Attention of many rows at a time over the paged cache in its 8-bit forms (kv8.cuh), and of the rows of all sequences that begin
// with the same pages over those pages (8-bit or bfloat16), on the 5th-generation tensor cores; compiled for one head size: -DOE_HD=64
// or 128.
//
// A row is a (token, query head of the group) pair.  A CTA has MT tiles of 128 rows of one KV head and a run of cache pages (64 keys
// each); the tiles share every page's K and V.  Per page and tile:
//   S = Q K^T      tcgen05.mma M=128 N=64 K=HD, float32 in tensor memory (two buffers);
//   softmax        128 threads, one row each, or of a single tile 256, half a row's keys each: the scores from tensor memory, times
//                  the keys' scales, mask, maximum and sum in float32, P back into the buffer's columns;
//   O += P V       tcgen05.mma M=128 N=HD K=64, P from tensor memory, O float32 in tensor memory for the whole run.
// A row's reference maximum moves only when its maximum has grown by more than 2^7 since it was set; O and the sum are rescaled
// then, before the page's P V is issued, and the factor cancels in O / l.
// 8-bit forms: a code is a float16 exactly.  The pages' codes come by bulk copies; a warpgroup turns them into the swizzled float16 tiles
// that the products read, once for all MT tiles.  The keys' scales multiply the float32 scores, the values' scales the weights.
// Queries and weights are rounded to float16 (2^-12 of themselves): a query row is scaled by a power of two into [1, 2) first,
// weights are relative to R, the power of two above the largest value scale so far, and times 2^8 (what float16 cannot hold is
// then below 2^-33 of a row's largest weight).  R grows for the whole CTA at once, with the rescaling of O.
// bfloat16: K and V as they are (TMA); queries and weights are sums of two bfloat16, a second product each.
// Roles (warps): 0 asks for the pages, 1 issues the products, 2 prepares the scales, 4-11 turn codes into float16 (8-bit forms),
// the last 8 load and turn the queries, then do the softmax and store.
// A page number outside the cache counts as a page without keys; a row at a position without an angle comes out undefined; a member that is no
// sequence of the step reads and writes nothing, and what its group gets is undefined then.
// Few tiles: the pages are cut into `splits` runs, whose parts (O, m, l) are joined by the kernel that runs next.
// Measured (us; 8 KV heads of 128, int8):  a page takes a CTA 0.98 with one tile and 1.38 with two, besides 10 to 13 to start and end.  No
// unit is full then (two tiles: issue slots 56 %, exponentials and tensor cores 39 % each); the time is the chain that a page's
// scores, weights and products are, with two buffers of scores, and the waits between its warps: leaving out the exponentials, the scales'
// loads, half of either product or half of the conversion's stores changes it by 3 % at most.  One tile, whose chain nothing else
// hides: two threads a row 0.98, one 1.06; two tiles: 1.52 and 1.38.  Two CTAs of one tile an SM: 2,048 tokens in 90 instead of 74.  A
// warp for each tile's products: 1.44 instead of 1.38.  A prompt of 2,048 tokens with 24 heads takes 66 (390 TFLOP/s of causal
// work), 192 tokens with 32 heads behind 12,005 of e4m3 73 (518 TFLOP/s), joined from 6 runs, both with the cache write; 64 members with 32 heads behind
// 8,192 common tokens 50 with the kernel of their own keys (177 TFLOP/s).
// The 16-bit cache's kernel takes that prompt in 46 with its rotation and write: it turns no codes, so that two of its CTAs fit an SM.
// Every wait on an mbarrier is bounded in time; one that runs out raises an error flag, every role leaves its loop, copies in
// flight get a fixed time, and tensor memory is freed.
#include <cuda.h>
#include <cudaTypedefs.h>
#include "kv8.cuh"
#include <mutex>

#ifndef OE_HD
#define OE_HD 128
#endif

namespace {

constexpr int HD = OE_HD;
static_assert(HD == 64 || HD == 128, "built for head_dim 64 or 128");
constexpr int BM = 128, BN = OE_PAGE, SUB = HD / 64;
constexpr int Q_BYTES = BM * HD * 2;             // SUB sub-tiles of [128][64] 16-bit values
constexpr int T_BYTES = BN * HD * 2;             // K or V of a page, SUB sub-tiles of [64][64] 16-bit values
constexpr int RAW = BN * HD;                     // codes of a page's K or V
static_assert(OE_PAGE == 64, "a block of keys is a page");
constexpr int STAGES = 2, RAW_STAGES = 4, SC_SLOTS = 6;
constexpr float RESCALE_STEP = 7.f, LOG2E = 1.4426950408889634f;
constexpr unsigned long long WAIT_LIMIT_NS = 2000000000ull;

__device__ int g_error = 0;

struct Scales {
    float k[BN], v[BN];                          // as copied; v then relative to R (0 where no key is)
    float grown, ref;                            // R before / R, and R
    int mapped, pad;
};
struct Ctl {
    Scales sc[SC_SLOTS];
    uint64_t q_full, raw_full[RAW_STAGES], raw_empty[RAW_STAGES], k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
    uint64_t sc_full[SC_SLOTS], sc_ready[SC_SLOTS], sc_empty[SC_SLOTS];
    uint64_t s_full[2][2], p_ready[2][2], pv_done[2], o_done[2];
    uint32_t tmem_base;
    int abort_flag;
    float up[2 * BM];                            // what a row of queries was divided by
    float swap[2][BM];                           // what the two threads of a row tell each other
};

template <int KIND, int MT>
struct Shape {
    static constexpr bool EIGHT = KIND != OE_KV_BF16;
    static constexpr int Q_ALL = MT * Q_BYTES * (EIGHT ? 1 : 2);
    static constexpr int K_AT = Q_ALL, V_AT = K_AT + STAGES * T_BYTES, RAW_AT = V_AT + STAGES * T_BYTES;
    static constexpr int CTL_AT = RAW_AT + (EIGHT ? RAW_STAGES * 2 * RAW : 0);
    static constexpr int BYTES = CTL_AT + (int)sizeof(Ctl);
    static constexpr int CONVERT = EIGHT ? 8 : 0;                      // warps: four for keys, four for values
    static constexpr int FIRST = 4 + CONVERT;                          // the first softmax warp
    static constexpr int SPLIT = MT == 1 ? 2 : 1;                      // softmax threads of a row
    static constexpr int KEYS = BN / SPLIT;                            // that each has of a page
    static constexpr int SOFTMAX = 4 * MT * SPLIT;                     // warps
    static constexpr int THREADS = (FIRST + SOFTMAX) * 32;
    // 8-bit forms: the launch gives each thread of the five warpgroups 96 registers, 480 for a lane of each; the softmax's need more
    static constexpr int SOFTMAX_REGISTERS = 144, CONVERT_REGISTERS = 56, OTHER_REGISTERS = 80;
    static constexpr int ALL_REGISTERS = OTHER_REGISTERS + 2 * CONVERT_REGISTERS + SOFTMAX / 4 * SOFTMAX_REGISTERS;
    static constexpr uint32_t S_COLS = MT * 2 * BN, O_COLS = MT * HD;
    static constexpr uint32_t COLS = S_COLS + O_COLS <= 128 ? 128 : S_COLS + O_COLS <= 256 ? 256 : 512;
    static constexpr float HEADROOM = EIGHT ? 8.f : 0.f;
};

struct Args {
    bf16* out;                 // [T, H*HD]
    const bf16* q;             // rows of q_stride elements: the projections, queries first, not yet turned
    long long q_stride;
    const float* cos_tab;      // [max_pos, HD/2] or null
    const float* sin_tab;
    const uint8_t* codes;      // 8-bit forms
    const float* scales;
    long long n_pages;
    const int* tables;
    int max_pages;
    const int* cu_q;
    const int* seq_start;
    const int* seq_qlen;
    int H, KVH, window;
    int n_positions;           // that the angles are there for
    float scale_log2;
    int ahead;
    const int* members;        // prefixes, as in attention_kv8.cu
    const int* first;
    const int* pages;
    int n_members, n_seqs;     // that `members` holds, and that its numbers are below
    int splits;
    float* part_o;             // [rows, splits, HD]: row = (sequence or packed token) * H + head
    float* part_ml;            // [rows, splits, 2]
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ unsigned long long global_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, Ctl* ctl, int code) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = global_ns();
    for (uint32_t spin = 0;; spin++) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((spin & 255u) == 255u) {
            if (*(volatile int*)&ctl->abort_flag) return false;
            if (global_ns() - t0 > WAIT_LIMIT_NS) {
                atomicExch(&ctl->abort_flag, 1);
                atomicCAS(&g_error, 0, code);
                return false;
            }
        }
    }
}
// All lanes of the warp wait and take the same decision.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, Ctl* ctl, int code) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, ctl, code));
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_u32(dst)), "l"((uint64_t)map), "r"(smem_u32(bar)), "r"(c0), "r"(c1) : "memory");
}
// Shared-memory operand descriptor, 128-byte swizzle, version 1 (sm_100).  K-major: rows of 128 bytes along K, stride 1024 between
// groups of 8 rows.  MN-major: rows of 128 bytes along N, one row per k, stride 1024 between groups of 8 k, leading offset between
// column groups of 64.
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t lead_bytes, uint32_t stride_bytes) {
    uint64_t d = 0;
    d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)((lead_bytes >> 4) & 0x3FFFu) << 16;
    d |= (uint64_t)((stride_bytes >> 4) & 0x3FFFu) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// kind::f16 instruction descriptor: D float32, A and B both float16 or both bfloat16, A K-major, B K-major or MN-major.
__device__ __forceinline__ uint32_t umma_idesc(int m, int n, bool b_mn_major, bool bf) {
    return (1u << 4) | (bf ? (1u << 7) | (1u << 10) : 0u) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, float* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
// (no "memory": loads of the scales may move across it; tmem_st_wait orders it)
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ bool elect_one() {
    uint32_t pred;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred));
    return pred != 0;
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Two float32 at once.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(*(uint64_t*)&d) : "l"(*(uint64_t*)&a), "l"(*(uint64_t*)&b));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(*(uint64_t*)&d) : "l"(*(uint64_t*)&a), "l"(*(uint64_t*)&b));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(*(uint64_t*)&d) : "l"(*(uint64_t*)&a), "l"(*(uint64_t*)&b), "l"(*(uint64_t*)&c));
    return d;
}
// The registers of this warpgroup's threads from here on.
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <bool EIGHT>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if (EIGHT) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *(const uint32_t*)&h;
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t rest_bf16(float lo, float hi, uint32_t h) {
    return pack16<false>(lo - __uint_as_float(h << 16), hi - __uint_as_float(h & 0xffff0000u));
}

// A page's codes to the swizzled 16-bit tile, by four warps.  A lane takes 16 codes at a time; the lanes of the second sub-tile store their
// two pieces in the other order, so that 8 lanes fill 8 different bank groups.  SOME: keys from `keys` on become zeros.
template <int KIND, bool SOME>
__device__ __forceinline__ void convert_tile(const uint8_t* raw, uint8_t* tile, int t, int keys) {
    constexpr int PER_ROW = HD / 16;
#pragma unroll
    for (int u = t; u < BN * PER_ROW; u += 128) {
        const int key = u / PER_ROW, g = u % PER_ROW;
        uint4 w = *(const uint4*)(raw + u * 16);
        if (SOME && key >= keys) w = make_uint4(0u, 0u, 0u, 0u);
        const uint32_t in[4] = {kv8_word<KIND>(w.x), kv8_word<KIND>(w.y), kv8_word<KIND>(w.z), kv8_word<KIND>(w.w)};
        uint4 o[2];
        o[0] = make_uint4(kv8_pair<KIND>(in[0], 0), kv8_pair<KIND>(in[0], 2), kv8_pair<KIND>(in[1], 0), kv8_pair<KIND>(in[1], 2));
        o[1] = make_uint4(kv8_pair<KIND>(in[2], 0), kv8_pair<KIND>(in[2], 2), kv8_pair<KIND>(in[3], 0), kv8_pair<KIND>(in[3], 2));
        uint8_t* row = tile + (g / 4) * (BN * 128) + key * 128;
        const int c = (g % 4) * 2, x = key & 7, odd = g / 4;
        *(uint4*)(row + (((c + odd) ^ x) << 4)) = odd ? o[1] : o[0];
        *(uint4*)(row + (((c + 1 - odd) ^ x) << 4)) = odd ? o[0] : o[1];
    }
}

// A row's weights of a page, or of the half that the thread has: P into tensor memory, their sum.  GONE: some scores are -infinity,
// whose weights are zero whatever the values' scales are.
template <bool EIGHT, bool GONE, int KEYS>
__device__ __forceinline__ float page_weights(const float (&s)[KEYS], const float* vscale, float scale, float neg_m, uint32_t p_addr) {
    const float2 scale2 = make_float2(scale, scale), neg2 = make_float2(neg_m, neg_m);
    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int k0 = 0; k0 < KEYS; k0 += 16) {
        uint32_t w[8], rest[8];
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
            float4 f = make_float4(1.f, 1.f, 1.f, 1.f);
            if (EIGHT) f = *(const float4*)(vscale + k0 + k);
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float2 x = make_float2(s[k0 + k + e], s[k0 + k + e + 1]);
                float2 p = fma2(x, scale2, neg2);
                p.x = fast_exp2(p.x);
                p.y = fast_exp2(p.y);
                sum[e / 2] = add2(sum[e / 2], p);
                if (EIGHT) {
                    p = mul2(p, e ? make_float2(f.z, f.w) : make_float2(f.x, f.y));
                    if (GONE) {
                        p.x = x.x == -INFINITY ? 0.f : p.x;
                        p.y = x.y == -INFINITY ? 0.f : p.y;
                    }
                }
                w[(k + e) / 2] = pack16<EIGHT>(p.x, p.y);
                if (!EIGHT) rest[(k + e) / 2] = rest_bf16(p.x, p.y, w[(k + e) / 2]);
            }
        }
        tmem_st8(p_addr + (uint32_t)(k0 / 2), w);
        if (!EIGHT) tmem_st8(p_addr + (uint32_t)(BN / 2 + k0 / 2), rest);
    }
    const float2 all = add2(sum[0], sum[1]);
    return all.x + all.y;
}
// Two warps' decision: true for all 64 threads if it is true for one.
__device__ __forceinline__ bool either(int barrier, bool mine) {
    uint32_t all;
    __syncwarp();
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(all) : "r"((uint32_t)mine), "r"(barrier) : "memory");
    return all != 0;
}

// PREFIX false: the tiles are those of one sequence's tokens, keys up to each row's position.  PREFIX true: the rows are those of all
// members of a group, the keys the group's common pages.
template <int KIND, bool PREFIX, int MT>
__global__ void __launch_bounds__(Shape<KIND, MT>::THREADS, 1)
attn_rows_kernel(const __grid_constant__ CUtensorMap map_kv, const Args a) {
    using Z = Shape<KIND, MT>;
    constexpr bool EIGHT = Z::EIGHT;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    {   // the swizzled tiles need a 1024-byte boundary; the launch leaves less than 1024 bytes of slack
        uint32_t dyn;
        asm volatile("mov.u32 %0, %%dynamic_smem_size;" : "=r"(dyn));
        if ((uint32_t)(smem - smem_raw) + (uint32_t)Z::BYTES > dyn) {
            if (threadIdx.x == 0) atomicCAS(&g_error, 0, 9);
            return;
        }
    }
    uint8_t* q_s = smem;
    uint8_t* k_s = smem + Z::K_AT;
    uint8_t* v_s = smem + Z::V_AT;
    uint8_t* raw_s = smem + Z::RAW_AT;
    Ctl* ctl = (Ctl*)(smem + Z::CTL_AT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.H / a.KVH, tpt = BM / G;               // tokens, or members, of a tile
    const int kvh = blockIdx.x % a.KVH, split = blockIdx.x / a.KVH;
    auto member = [&](int i) {                             // the sequence of the group's i-th member, -1: none
        const int at = a.first[blockIdx.y] + i, sq = (unsigned)at < (unsigned)a.n_members ? a.members[at] : -1;
        return (unsigned)sq < (unsigned)a.n_seqs ? sq : -1;
    };
    // the tiles' rows and the CTA's pages (the step's integers were written before its first kernel)
    int b, count, t0, start = 0, key_lo = 0, j_lo, n_blocks[MT];
    if (PREFIX) {
        const int g = blockIdx.y;
        count = a.first[g + 1] - a.first[g];
        t0 = blockIdx.z * MT * tpt;
        b = t0 < count ? member(0) : 0;
        if (b < 0) count = 0;
    } else {
        b = blockIdx.y;
        count = a.seq_qlen[b];
        t0 = ((int)gridDim.z - 1 - (int)blockIdx.z) * MT * tpt;     // the heaviest tiles first
    }
    if (t0 >= count) {
        pdl_wait();
        pdl_launch_dependents();
        return;
    }
    int any = 0;                                           // the most pages a tile has
    {
        int hi = 0;
        if (PREFIX) {
            const int n = a.pages[blockIdx.y];
            j_lo = (int)((long long)n * split / a.splits);
            hi = (int)((long long)n * (split + 1) / a.splits);
        } else {
            start = a.seq_start[b];
            key_lo = oe_first_key(start + t0, a.window);
            j_lo = key_lo / BN;
            const int n = (start + min(t0 + MT * tpt, count) - 1) / BN - j_lo + 1;
            hi = j_lo + (int)((long long)n * (split + 1) / a.splits);
            j_lo += (int)((long long)n * split / a.splits);
        }
#pragma unroll
        for (int t = 0; t < MT; t++) {
            int last = hi;
            if (!PREFIX) last = min(hi, (start + min(t0 + (t + 1) * tpt, count) - 1) / BN + 1);
            n_blocks[t] = t0 + t * tpt < count ? max(0, last - j_lo) : 0;
            any = max(any, n_blocks[t]);
        }
    }
    const int* trow = a.tables + (size_t)b * a.max_pages;
    if (threadIdx.x == 0) {
        mbar_init(&ctl->q_full, Z::CONVERT + Z::SOFTMAX);
        for (int s = 0; s < RAW_STAGES; s++) { mbar_init(&ctl->raw_full[s], 1); mbar_init(&ctl->raw_empty[s], 8); }
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&ctl->k_full[s], EIGHT ? 4 : 1); mbar_init(&ctl->k_empty[s], 1);
            mbar_init(&ctl->v_full[s], EIGHT ? 4 : 1); mbar_init(&ctl->v_empty[s], 1);
        }
        for (int s = 0; s < SC_SLOTS; s++) {
            mbar_init(&ctl->sc_full[s], 1); mbar_init(&ctl->sc_ready[s], 1); mbar_init(&ctl->sc_empty[s], Z::SOFTMAX);
        }
        for (int t = 0; t < MT; t++) {
            mbar_init(&ctl->s_full[t][0], 1); mbar_init(&ctl->s_full[t][1], 1);
            mbar_init(&ctl->p_ready[t][0], 4 * Z::SPLIT); mbar_init(&ctl->p_ready[t][1], 4 * Z::SPLIT);
            mbar_init(&ctl->pv_done[t], 1); mbar_init(&ctl->o_done[t], 1);
        }
        ctl->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)), "r"(Z::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem_base = *(volatile uint32_t*)&ctl->tmem_base;
    // prefixes: where the caller says so, the pages are asked for before the wait; the queries come from the kernel before.  The kernel
    // of the own keys may start when that one is done: it waits for this one only where it needs the parts
    if (!PREFIX) pdl_launch_dependents();
    const bool ahead = PREFIX && a.ahead;
    if (!ahead || warp >= 4) pdl_wait();
    if (PREFIX && warp >= 4) pdl_launch_dependents();

    // The queries, turned, by all warps from 4 on: HD / 16 lanes have a row, 8 dimensions of its lower half and the 8 that they are
    // turned with each.  Several rows' pieces are asked for before the first is used: the start of a CTA is these loads.
    if (warp >= 4) {
        constexpr int PER = HD / 16, AT_ONCE = 32 / PER, WARPS = Z::CONVERT + Z::SOFTMAX, GROUPS = MT * BM / AT_ONCE;
        constexpr int NEEDED = (GROUPS + WARPS - 1) / WARPS, MOST = Z::THREADS > 384 ? 2 : 4, ROUND = NEEDED < MOST ? NEEDED : MOST;     // (what the registers hold)
        const int d = lane % PER * 8;
        // where the rows are, of all rounds
        constexpr int ALL = (GROUPS + WARPS - 1) / WARPS;
        const bf16* src[ALL];
        int pos_of[ALL];
#pragma unroll
        for (int k = 0; k < ALL; k++) {
            const int g = warp - 4 + k * WARPS, rr = g * AT_ONCE + lane / PER, r = rr % BM, tok = t0 + rr / BM * tpt + r / G;
            src[k] = nullptr;
            pos_of[k] = 0;
            if (g < GROUPS && r < tpt * G && tok < count) {
                long long at;
                int pos;
                if (PREFIX) {
                    const int sq = member(tok);
                    if (sq < 0) continue;
                    at = a.cu_q[sq];
                    pos = a.seq_start[sq];
                } else {
                    at = a.cu_q[b] + tok;
                    pos = start + tok;
                }
                pos_of[k] = (unsigned)pos < (unsigned)a.n_positions ? pos : -1;
                src[k] = a.q + at * a.q_stride + (long long)(kvh * G + r % G) * HD + d;
            }
        }
#pragma unroll
        for (int k0 = 0; k0 < ALL; k0 += ROUND) {
            const int g0 = warp - 4 + k0 * WARPS;
            uint4 u[ROUND], v[ROUND];
            int pos[ROUND];
#pragma unroll
            for (int k = 0; k < ROUND; k++) {
                const bf16* from = k0 + k < ALL ? src[k0 + k < ALL ? k0 + k : 0] : nullptr;
                pos[k] = k0 + k < ALL ? pos_of[k0 + k < ALL ? k0 + k : 0] : 0;
                u[k] = v[k] = make_uint4(0u, 0u, 0u, 0u);
                if (from != nullptr) {
                    u[k] = *(const uint4*)from;
                    v[k] = *(const uint4*)(from + HD / 2);
                }
            }
            float cs[ROUND][8], sn[ROUND][8];
            if (a.cos_tab != nullptr) {
#pragma unroll
                for (int k = 0; k < ROUND; k++) {
#pragma unroll
                    for (int j = 0; j < 8; j += 4) {
                        *(float4*)&cs[k][j] = *(const float4*)(a.cos_tab + (long long)max(pos[k], 0) * (HD / 2) + d + j);
                        *(float4*)&sn[k][j] = *(const float4*)(a.sin_tab + (long long)max(pos[k], 0) * (HD / 2) + d + j);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < ROUND; k++) {
                if (g0 + k * WARPS >= GROUPS) break;         // (the warp's)
                const int rr = (g0 + k * WARPS) * AT_ONCE + lane / PER, tile = rr / BM, r = rr % BM;
                const uint32_t uw[4] = {u[k].x, u[k].y, u[k].z, u[k].w}, vw[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
                float x[2][8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    x[0][e] = kv8_from_bits((uw[e / 2] >> (16 * (e & 1))) & 0xffffu);
                    x[1][e] = kv8_from_bits((vw[e / 2] >> (16 * (e & 1))) & 0xffffu);
                }
                if (a.cos_tab != nullptr) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float lo = x[0][e], hi = x[1][e];
                        x[0][e] = lo * cs[k][e] - hi * sn[k][e];
                        x[1][e] = lo * sn[k][e] + hi * cs[k][e];
                    }
                }
                float down = 1.f, up = 1.f;
                if (EIGHT) {
                    float most = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; e++) most = fmaxf(most, fmaxf(fabsf(x[0][e]), fabsf(x[1][e])));
#pragma unroll
                    for (int o = PER / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                    down = kv8_row_factor(most, &up);
                }
                if (d == 0) ctl->up[rr] = pos[k] < 0 ? __uint_as_float(0x7fc00000u) : up;      // (no angle: an undefined row)
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const int dim = d + half * (HD / 2);
                    uint32_t w[4], rest[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float q0 = x[half][2 * e] * down, q1 = x[half][2 * e + 1] * down;
                        w[e] = pack16<EIGHT>(q0, q1);
                        if (!EIGHT) rest[e] = rest_bf16(q0, q1, w[e]);
                    }
                    uint8_t* to = q_s + tile * (EIGHT ? 1 : 2) * Q_BYTES + (dim / 64) * (BM * 128) + r * 128 + ((((dim % 64) / 8) ^ (r & 7)) << 4);
                    *(uint4*)to = make_uint4(w[0], w[1], w[2], w[3]);
                    if (!EIGHT) *(uint4*)(to + Q_BYTES) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
                }
            }
        }
        fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->q_full);
    }
    if (EIGHT && warp < 4) fewer_registers<Z::OTHER_REGISTERS>();
    if (warp == 0) {
        // ---------------- the pages ----------------
        if (lane == 0) {
            bool ok = true;
            auto row_of = [&](int i, int which) -> long long {      // the first row of page i's K or V, -1: not mapped
                const int j = j_lo + i, page = j < a.max_pages ? trow[j] : -1;
                return (unsigned)page < (unsigned long long)a.n_pages ? (((long long)page * 2 + which) * a.KVH + kvh) * BN : -1;
            };
            if (EIGHT) {
                for (int i = 0; i < any && ok; i++) {
                    const int s = i % RAW_STAGES, c = i % SC_SLOTS;
                    ok = mbar_wait(&ctl->raw_empty[s], ((uint32_t)(i / RAW_STAGES) & 1u) ^ 1u, ctl, 1);
                    if (ok) ok = mbar_wait(&ctl->sc_empty[c], ((uint32_t)(i / SC_SLOTS) & 1u) ^ 1u, ctl, 2);
                    if (!ok) break;
                    fence_async();                         // the slot's scales were written by threads before
                    long long kr = row_of(i, 0), vr = row_of(i, 1);
                    ctl->sc[c].mapped = kr >= 0;
                    if (kr < 0) { kr = (long long)kvh * BN; vr = kr + (long long)a.KVH * BN; }      // (any rows: none of them counts)
                    mbar_expect_tx(&ctl->raw_full[s], 2 * RAW);
                    bulk_load(raw_s + s * 2 * RAW, a.codes + kr * HD, RAW, &ctl->raw_full[s]);
                    bulk_load(raw_s + s * 2 * RAW + RAW, a.codes + vr * HD, RAW, &ctl->raw_full[s]);
                    mbar_expect_tx(&ctl->sc_full[c], 2 * BN * 4);
                    bulk_load(ctl->sc[c].k, a.scales + kr, BN * 4, &ctl->sc_full[c]);
                    bulk_load(ctl->sc[c].v, a.scales + vr, BN * 4, &ctl->sc_full[c]);
                }
            } else {
                auto load = [&](int i, int which, uint64_t* full, uint64_t* empty, uint8_t* ring, int code) -> bool {
                    const int s = i % STAGES;
                    if (!mbar_wait(&empty[s], ((uint32_t)(i / STAGES) & 1u) ^ 1u, ctl, code)) return false;
                    long long r = row_of(i, which);
                    if (r < 0) r = a.n_pages * 2 * a.KVH * BN;       // outside the map: zeros
                    mbar_expect_tx(&full[s], (uint32_t)T_BYTES);
                    for (int sb = 0; sb < SUB; sb++)
                        tma_load_2d(ring + s * T_BYTES + sb * (BN * 128), &map_kv, &full[s], sb * 64, (int)r);
                    return true;
                };
                if (any > 0) ok = load(0, 0, ctl->k_full, ctl->k_empty, k_s, 1);
                for (int i = 0; i < any && ok; i++) {
                    if (i + 1 < any) ok = load(i + 1, 0, ctl->k_full, ctl->k_empty, k_s, 1);
                    if (ok) ok = load(i, 1, ctl->v_full, ctl->v_empty, v_s, 10);
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- the products: the whole warp waits, one elected lane issues ----------------
        const uint32_t idesc_s = umma_idesc(BM, BN, false, !EIGHT), idesc_o = umma_idesc(BM, HD, true, !EIGHT);
        const uint64_t q_desc = umma_desc(smem_u32(q_s), 16, 1024), k_desc = umma_desc(smem_u32(k_s), 16, 1024);
        const uint64_t v_desc = umma_desc(smem_u32(v_s), BN * 128, 1024);
        bool ok = warp_wait(&ctl->q_full, 0, ctl, 3);
        auto issue_s = [&](int t, int i) {                   // S_i of tile t, into its buffer i & 1
            const uint64_t kd = k_desc + (uint64_t)(i % STAGES * (T_BYTES >> 4));
            const uint32_t d = tmem_base + (uint32_t)((t * 2 + (i & 1)) * BN);
            if (elect_one()) {
#pragma unroll
                for (int h = 0; h < (EIGHT ? 1 : 2); h++) {
                    const uint64_t qd = q_desc + (uint64_t)((t * (EIGHT ? 1 : 2) + h) * (Q_BYTES >> 4));
#pragma unroll
                    for (int k = 0; k < HD / 16; k++) {
                        const uint32_t sb = k / 4, kk = k % 4;
                        umma(d, qd + (uint64_t)((sb * (BM * 128) + kk * 32) >> 4), kd + (uint64_t)((sb * (BN * 128) + kk * 32) >> 4),
                             idesc_s, (k > 0 || h > 0) ? 1u : 0u);
                    }
                }
                umma_commit(&ctl->s_full[t][i & 1]);
            }
            __syncwarp();
        };
        auto release = [&](uint64_t* bar) {                  // when everything issued so far is done
            if (elect_one()) umma_commit(bar);
            __syncwarp();
        };
        // A tile's S of page i + 2 is issued right behind its P V of page i, whose buffer it takes: neither waits for the other tile.
        for (int i = 0; i < min(any, 2) && ok; i++) {
            ok = warp_wait(&ctl->k_full[i % STAGES], (uint32_t)(i / STAGES) & 1u, ctl, 4);
            fence_after();
            if (!ok) break;
#pragma unroll
            for (int t = 0; t < MT; t++)
                if (i < n_blocks[t]) issue_s(t, i);
            release(&ctl->k_empty[i % STAGES]);
        }
        for (int i = 0; i < any && ok; i++) {
            const int s = i % STAGES;
            ok = warp_wait(&ctl->v_full[s], (uint32_t)(i / STAGES) & 1u, ctl, 5);
            if (!ok) break;
            const uint64_t vd = v_desc + (uint64_t)(s * (T_BYTES >> 4));
            bool keys = false;                               // page i + 2's are there
#pragma unroll
            for (int t = 0; t < MT; t++) {
                if (i >= n_blocks[t] || !ok) continue;
                ok = warp_wait(&ctl->p_ready[t][i & 1], (uint32_t)(i >> 1) & 1u, ctl, 6);
                if (!ok) continue;
                fence_after();
                const uint32_t p = tmem_base + (uint32_t)((t * 2 + (i & 1)) * BN), o = tmem_base + Z::S_COLS + (uint32_t)(t * HD);
                if (elect_one()) {
#pragma unroll
                    for (int h = 0; h < (EIGHT ? 1 : 2); h++) {
#pragma unroll
                        for (int k = 0; k < BN / 16; k++)
                            umma_ts(o, p + (uint32_t)(h * (BN / 2) + k * 8), vd + (uint64_t)((k * (16 * 128)) >> 4), idesc_o,
                                    (i > 0 || k > 0 || h > 0) ? 1u : 0u);
                    }
                    umma_commit(&ctl->pv_done[t]);
                    if (i == n_blocks[t] - 1) umma_commit(&ctl->o_done[t]);
                }
                __syncwarp();
                if (i + 2 < n_blocks[t]) {
                    if (!keys) ok = warp_wait(&ctl->k_full[s], (uint32_t)((i + 2) / STAGES) & 1u, ctl, 4);
                    if (!ok) continue;
                    keys = true;
                    fence_after();
                    issue_s(t, i + 2);
                }
            }
            if (!ok) break;
            release(&ctl->v_empty[s]);
            if (i + 2 < any) release(&ctl->k_empty[s]);
        }
    } else if (warp == 2) {
        // ---------------- the scales: relative to R, and what R grew by ----------------
        if (EIGHT) {
            float ref = kv8_above(0.f);
            const int key_hi = PREFIX ? 0x7fffffff : start + min(t0 + MT * tpt, count) - 1;
            for (int i = 0; i < any; i++) {
                const int c = i % SC_SLOTS;
                if (!warp_wait(&ctl->sc_full[c], (uint32_t)(i / SC_SLOTS) & 1u, ctl, 11)) break;
                Scales* sc = &ctl->sc[c];
                const bool mapped = *(volatile int*)&sc->mapped != 0;
                float2 v = *(const float2*)&sc->v[lane * 2];
                const int key = (j_lo + i) * BN + lane * 2;
                if (!mapped || key < key_lo || key > key_hi) v.x = 0.f;
                if (!mapped || key + 1 < key_lo || key + 1 > key_hi) v.y = 0.f;
                float most = fmaxf(fmaxf(v.x, 0.f), v.y);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                const float next = fmaxf(ref, kv8_above(most)), inv = kv8_inverse(next);
                *(float2*)&sc->v[lane * 2] = make_float2(v.x * inv, v.y * inv);
                if (lane == 0) { sc->grown = ref * inv; sc->ref = next; }
                ref = next;
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->sc_ready[c]);
            }
        }
    } else if (EIGHT && warp >= 4 && warp < Z::FIRST) {
        // ---------------- codes to 16-bit tiles: four warps the keys', four the values' ----------------
        fewer_registers<Z::CONVERT_REGISTERS>();
        const int t = threadIdx.x & 127;
        const bool values = warp >= 8;
        uint64_t *full = values ? ctl->v_full : ctl->k_full, *empty = values ? ctl->v_empty : ctl->k_empty;
        for (int i = 0; i < any; i++) {
            const int s = i % STAGES, rs = i % RAW_STAGES;
            if (!warp_wait(&ctl->raw_full[rs], (uint32_t)(i / RAW_STAGES) & 1u, ctl, 12)) break;
            if (!warp_wait(&empty[s], ((uint32_t)(i / STAGES) & 1u) ^ 1u, ctl, 13)) break;
            // a value behind the last token may hold e4m3 codes that are no numbers, and a weight of 0 times that is not 0
            int keys = BN;
            if (KIND == OE_KV_E4M3 && values) {
                if (*(volatile int*)&ctl->sc[i % SC_SLOTS].mapped == 0) keys = 0;
                else if (!PREFIX) keys = start + count - (j_lo + i) * BN;
            }
            uint8_t* to = (values ? v_s : k_s) + s * T_BYTES;
            if (KIND == OE_KV_E4M3 && keys < BN) convert_tile<KIND, true>(raw_s + (rs * 2 + values) * RAW, to, t, keys);
            else convert_tile<KIND, false>(raw_s + (rs * 2 + values) * RAW, to, t, BN);
            fence_async();
            __syncwarp();
            if (lane == 0) { mbar_arrive(&full[s]); mbar_arrive(&ctl->raw_empty[rs]); }
        }
    } else if (warp >= Z::FIRST) {
        // ---------------- softmax, output: one row a thread, or two threads a row ----------------
        if (EIGHT) more_registers<Z::SOFTMAX_REGISTERS>();
        constexpr int SPLIT = Z::SPLIT, KEYS = Z::KEYS;
        const int tile = (warp - Z::FIRST) / (4 * SPLIT), half = SPLIT == 2 ? (warp - Z::FIRST) / 4 & 1 : 0, quarter = warp & 3, pair = 1 + tile * 4 + quarter;
        const int r = quarter * 32 + lane;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const uint32_t s_addr = lane_addr + (uint32_t)(tile * 2 * BN), o_addr = lane_addr + Z::S_COLS + (uint32_t)(tile * HD + half * (HD / SPLIT));
        const int tok = t0 + tile * tpt + r / G, head = kvh * G + r % G;
        bool valid = r < tpt * G && tok < count;
        int pos = 0, low = 0;
        long long row = 0;                                 // the packed row of q and out
        long long part = 0;
        if (valid) {
            if (PREFIX) {
                const int sq = member(tok);
                valid = sq >= 0;
                if (valid) {
                    row = a.cu_q[sq];
                    pos = a.seq_start[sq];
                    part = (long long)sq * a.H + head;
                }
            } else {
                row = a.cu_q[b] + tok;
                pos = start + tok;
                low = oe_first_key(pos, a.window);
                part = row * a.H + head;
            }
        }
        const int nb = n_blocks[tile];
        bool ok = true;
        float scale = a.scale_log2;
        if (nb > 0) {
            ok = warp_wait(&ctl->q_full, 0, ctl, 17);
            scale *= ctl->up[tile * BM + r];
        }
        float m_run = -INFINITY, l_run = 0.f, ref = 1.f;
        float* tell = &ctl->swap[half][r];                 // (two threads a row: one tile)
        const float* told = &ctl->swap[half ^ 1][r];
        // (a wait that runs out is told to the warp with the other half of the rows, so that neither waits for the other)
        for (int i = 0; i < nb; i++) {
            const int c = i % SC_SLOTS;
            const Scales* sc = &ctl->sc[c];
            const uint32_t sc_parity = (uint32_t)(i / SC_SLOTS) & 1u, s_parity = (uint32_t)(i >> 1) & 1u;
            const bool scales = !EIGHT || mbar_try_wait(&ctl->sc_ready[c], sc_parity), scores = mbar_try_wait(&ctl->s_full[tile][i & 1], s_parity);
            if (!__all_sync(0xffffffffu, scales && scores)) {
                if (ok && !scales) ok = mbar_wait(&ctl->sc_ready[c], sc_parity, ctl, 15);
                if (ok && !scores) ok = mbar_wait(&ctl->s_full[tile][i & 1], s_parity, ctl, 7);
                ok = __all_sync(0xffffffffu, ok);
            }
            if (SPLIT == 1 && !ok) break;
            fence_after();
            float s[KEYS];
#pragma unroll
            for (int c0 = 0; c0 < KEYS; c0 += 16) tmem_ld16_nowait(s_addr + (uint32_t)((i & 1) * BN + half * KEYS + c0), &s[c0]);
            tmem_ld_wait();
            const int key0 = (j_lo + i) * BN + half * KEYS;
            bool mapped;
            float grown = 1.f;
            if (EIGHT) {
                mapped = sc->mapped != 0;
                grown = sc->grown;
                ref = sc->ref;
#pragma unroll
                for (int k = 0; k < KEYS; k += 4) {
                    const float4 f = *(const float4*)&sc->k[half * KEYS + k];
                    const float2 x = mul2(make_float2(s[k], s[k + 1]), make_float2(f.x, f.y));
                    const float2 y = mul2(make_float2(s[k + 2], s[k + 3]), make_float2(f.z, f.w));
                    s[k] = x.x; s[k + 1] = x.y; s[k + 2] = y.x; s[k + 3] = y.y;
                }
            } else {
                const int j = j_lo + i, page = j < a.max_pages ? trow[j] : -1;
                mapped = (unsigned)page < (unsigned long long)a.n_pages;
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            // keys wholly before a row's position, inside its window and of the cache need no mask; the decision is the warp's, and
            // rows without a token, whose results nobody stores, take no part in it
            const bool masked = __any_sync(0xffffffffu, !mapped || (!PREFIX && valid && !(key0 + KEYS - 1 <= pos && key0 >= low)));
            if (masked) {
                const int hi = !mapped ? -1 : PREFIX ? KEYS - 1 : min(pos - key0, KEYS - 1), lo = PREFIX ? 0 : max(low - key0, 0);
                const unsigned span = hi >= lo ? (unsigned)(hi - lo) : 0u;
                const bool some = hi >= lo;
#pragma unroll
                for (int k = 0; k < KEYS; k++) s[k] = some && (unsigned)(k - lo) <= span ? s[k] : -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < KEYS; k += 2) mx4[k / 2 & 3] = max3(mx4[k / 2 & 3], s[k], s[k + 1]);
            float m_new = fmaxf(m_run, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale);
            // Both halves of the scores have been read behind this: P may take their place.
            bool move = !ok || i == 0 || grown != 1.f || (valid && m_new > m_run + RESCALE_STEP);
            if (SPLIT == 2) {
                fence_before();
                move = either(pair, move);
                fence_after();
            } else {
                move = __any_sync(0xffffffffu, move);
            }
            if (move) {
                // P_{i-1} V_{i-1} must have been added to O before O is rescaled (S_i is complete, hence P_{i-2} V_{i-2} too)
                if (ok && i > 0) ok = mbar_wait(&ctl->pv_done[tile], (uint32_t)(i - 1) & 1u, ctl, 8);
                if (SPLIT == 2) *tell = m_new;
                ok = SPLIT == 2 ? !either(pair, !ok) : __all_sync(0xffffffffu, ok);
                if (!ok) break;
                fence_after();
                if (SPLIT == 2) m_new = fmaxf(m_new, *told);
                if (i > 0) {
                    const float alpha = fast_exp2(m_run - (m_new == -INFINITY ? 0.f : m_new)), beta = alpha * grown;
#pragma unroll
                    for (int c0 = 0; c0 < HD / SPLIT; c0 += 16) {
                        float ob[16];
                        uint32_t ow[16];
                        tmem_ld16_nowait(o_addr + (uint32_t)c0, ob);
                        tmem_ld_wait();
#pragma unroll
                        for (int d = 0; d < 16; d++) ow[d] = __float_as_uint(ob[d] * beta);
                        tmem_st16(o_addr + (uint32_t)c0, ow);
                    }
                    tmem_st_wait();
                    l_run *= alpha;
                }
                m_run = m_new;
            }
            const float neg_m = (m_run == -INFINITY ? 0.f : -m_run) + Z::HEADROOM;
            const uint32_t p_addr = s_addr + (uint32_t)((i & 1) * BN + half * (KEYS / 2));
            const float* vs = EIGHT ? sc->v + half * KEYS : nullptr;
            l_run += EIGHT && masked ? page_weights<EIGHT, true, KEYS>(s, vs, scale, neg_m, p_addr) : page_weights<EIGHT, false, KEYS>(s, vs, scale, neg_m, p_addr);
            tmem_st_wait();
            fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&ctl->p_ready[tile][i & 1]);
                if (EIGHT) mbar_arrive(&ctl->sc_empty[c]);
            }
        }
        // pages that only the other tile has: their scales' slots are given back all the same
        if (EIGHT && ok) {
            for (int i = nb; i < any; i++) {
                const int c = i % SC_SLOTS;
                if (!warp_wait(&ctl->sc_ready[c], (uint32_t)(i / SC_SLOTS) & 1u, ctl, 15)) break;
                if (lane == 0) mbar_arrive(&ctl->sc_empty[c]);
            }
        }
        if (SPLIT == 2 && nb > 0) {
            // (m is told in the last page's round at the latest, which the barrier of that page's P, or of this, has behind it)
            either(pair, false);
            *tell = l_run;
            if (either(pair, !ok)) ok = false;
            l_run = half ? *told + l_run : l_run + *told;
        }
        if (ok) {
            if (nb > 0) {
                ok = mbar_wait(&ctl->o_done[tile], 0, ctl, 16);
                ok = __all_sync(0xffffffffu, ok);
                fence_after();
            }
            if (ok && nb > 0) {
                // COLS columns of the warp's rows at a time go through the tile of its queries, which nothing reads any more, so that a
                // row's values are stored side by side: LANES lanes have a row
                constexpr int COLS = SPLIT == 2 ? HD / 4 : 32, LANES = COLS / 4, ROWS = 32 / LANES;
                auto place = [](int rl, int c) { return LANES == 8 ? c ^ (rl & 7) : c ^ (rl >> 1 & 3); };      // (16 bytes: no two of 8 lanes in a bank)
                const bool parts = PREFIX || a.splits > 1;
                const float f = parts ? ref : l_run > 0.f ? ref / l_run : l_run == 0.f ? 0.f : l_run;
                uint8_t* stage = q_s + tile * (EIGHT ? 1 : 2) * Q_BYTES + (half * 4 + quarter) * (32 * COLS * 4);
                const long long mine = (parts ? (part * a.splits + split) * HD : row * (long long)(a.H * HD) + (long long)head * HD) + half * (HD / SPLIT);
                const uint32_t there = __ballot_sync(0xffffffffu, valid);
                long long to[LANES];                        // of the rows whose values this lane stores
#pragma unroll
                for (int k = 0; k < LANES; k++) to[k] = __shfl_sync(0xffffffffu, mine, k * ROWS + lane / LANES) + lane % LANES * 4;
#pragma unroll 1
                for (int c0 = 0; c0 < HD / SPLIT; c0 += COLS) {
                    float ob[COLS];
#pragma unroll
                    for (int c = 0; c < COLS; c += 16) tmem_ld16_nowait(o_addr + (uint32_t)(c0 + c), ob + c);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < COLS / 4; c++)
                        *(float4*)(stage + lane * (COLS * 4) + (place(lane, c) << 4)) = make_float4(ob[4 * c] * f, ob[4 * c + 1] * f, ob[4 * c + 2] * f, ob[4 * c + 3] * f);
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < LANES; k++) {
                        const int rl = k * ROWS + lane / LANES, c = lane % LANES;
                        const float4 x = *(const float4*)(stage + rl * (COLS * 4) + (place(rl, c) << 4));
                        if (there >> rl & 1u) {
                            if (parts) *(float4*)(a.part_o + to[k] + c0) = x;
                            else *(uint2*)(a.out + to[k] + c0) = make_uint2(pack16<false>(x.x, x.y), pack16<false>(x.z, x.w));
                        }
                    }
                    __syncwarp();
                }
            }
            if (ok && valid && half == 0 && (PREFIX || a.splits > 1)) *(float2*)(a.part_ml + (part * a.splits + split) * 2) = make_float2(m_run, l_run);
        }
        fence_before();
    }

    __syncthreads();
    if (*(volatile int*)&ctl->abort_flag) {
        const unsigned long long t0w = global_ns();
        while (global_ns() - t0w < 2000000ull) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Z::COLS) : "memory");
    }
}

// Rows' parts joined, in their order: a warp per row.  The step's padding rows, from token *n_real on, have no parts.  Its time is that
// of starting a kernel and of two dependent loads: 3 us for 24 to 6,000 rows of 6 to 36 parts, which are in the L2.
__global__ void __launch_bounds__(256)
join_parts_kernel(bf16* out, const float* part_o, const float* part_ml, const int* n_real, int H, long long rows, int n) {
    pdl_launch_dependents();
    const long long real = (long long)*n_real * H;
    pdl_wait();
    const long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (r >= min(rows, real)) return;
    constexpr int PER = HD / 32;
    const float2* ml = (const float2*)part_ml + r * n;
    float m = -INFINITY;
    for (int q = lane; q < n; q += 32) m = fmaxf(m, ml[q].x);
    m = warp_max(m);
    const float mu = m == -INFINITY ? 0.f : m;
    float o[PER] = {}, l = 0.f;
    for (int q0 = 0; q0 < n; q0 += 32) {
        const float2 mine = q0 + lane < n ? ml[q0 + lane] : make_float2(-INFINITY, 0.f);
        const bool none = mine.x == -INFINITY && mine.y == 0.f;             // no key of this row: its O was not stored
        const float w = none ? -1.f : exp2f(mine.x - mu);
        if (!none) l += mine.y * w;
        const float* p = part_o + (r * n + q0) * HD + lane * PER;
        const int here = min(32, n - q0);
        for (int q = 0; q < here; q += 8) {                 // (eight at a time, whether they count or not: their loads overlap)
            float v[8][PER];
#pragma unroll
            for (int k = 0; k < 8; k++) {
#pragma unroll
                for (int x = 0; x < PER; x += 2) *(float2*)&v[k][x] = *(const float2*)(p + min(q + k, here - 1) * HD + x);
            }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float e = q + k < here ? __shfl_sync(0xffffffffu, w, q + k) : -1.f;
#pragma unroll
                for (int x = 0; x < PER; x++) o[x] = e < 0.f ? o[x] : o[x] + v[k][x] * e;
            }
        }
    }
    l = warp_sum(l);
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
#pragma unroll
    for (int x = 0; x < PER; x += 2) *(uint32_t*)(out + r * HD + lane * PER + x) = pack16<false>(o[x] * inv, o[x + 1] * inv);
}

PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::mutex g_mutex;

int get_encode() {
    std::lock_guard<std::mutex> lock(g_mutex);
    if (g_encode) return 0;
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qres;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres);
    if (e != cudaSuccess || qres != cudaDriverEntryPointSuccess || fn == nullptr) return e != cudaSuccess ? (int)e : 999;
    g_encode = (PFN_cuTensorMapEncodeTiled_v12000)fn;
    return 0;
}

template <int KIND, bool PREFIX, int MT>
int launch(const CUtensorMap& map, const Args& a, dim3 grid, cudaStream_t st) {
    using Z = Shape<KIND, MT>;
    const size_t smem = (size_t)Z::BYTES + 1024;
    static Kv8Devices set;
    if (set.first()) {
        const cudaError_t e = cudaFuncSetAttribute(attn_rows_kernel<KIND, PREFIX, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        if (Z::EIGHT) {                                    // the warpgroups' shares have to fit what the launch gives
            cudaFuncAttributes f;
            const cudaError_t g = cudaFuncGetAttributes(&f, attn_rows_kernel<KIND, PREFIX, MT>);
            if (g != cudaSuccess) return (int)g;
            if (f.numRegs * (Z::THREADS / 128) < Z::ALL_REGISTERS) return OE_ERR_UNSUPPORTED;
        }
        set.done();
    }
    return oe_launch(attn_rows_kernel<KIND, PREFIX, MT>, grid, dim3(Z::THREADS), smem, st, map, a);
}
template <int KIND, bool PREFIX>
int launch_tiles(int mt, const CUtensorMap& map, const Args& a, dim3 grid, cudaStream_t st) {
    return mt == 1 ? launch<KIND, PREFIX, 1>(map, a, grid, st) : launch<KIND, PREFIX, 2>(map, a, grid, st);
}

Args arguments(const Kv8Call& c) {
    Args a = {};
    a.out = c.out; a.q = c.qkv; a.q_stride = c.stride; a.cos_tab = c.cos_tab; a.sin_tab = c.sin_tab; a.codes = (const uint8_t*)c.cache;
    a.scales = c.scales; a.n_pages = c.n_pages; a.tables = c.tables; a.max_pages = c.max_pages; a.cu_q = c.cu_q; a.seq_start = c.seq_start;
    a.seq_qlen = c.seq_qlen; a.H = c.H; a.KVH = c.KVH; a.window = c.window; a.n_positions = c.n_positions; a.n_members = c.n_members; a.n_seqs = c.n_seqs;
    a.scale_log2 = c.scale * LOG2E; a.ahead = c.ahead;
    a.members = c.members; a.first = c.first; a.pages = c.pages; a.splits = c.splits; a.part_o = c.part_o; a.part_ml = c.part_ml;
    return a;
}
bool operands_ok(const Args& a, const void* cache) {
    return a.KVH > 0 && a.H % a.KVH == 0 && a.H / a.KVH <= BM && a.q_stride % 8 == 0 && !((uintptr_t)a.q & 15) && !((uintptr_t)cache & 15) &&
           !((uintptr_t)a.scales & 15) && !((uintptr_t)a.cos_tab & 15) && !((uintptr_t)a.sin_tab & 15) && a.splits >= 1 && a.n_pages >= 1 && a.n_positions >= 1;
}

}  // namespace

extern "C" {

// out from each row's parts, as many as `shares`, or else `splits`, says.  cu_q[n_seqs] of the tokens are real; the rows of the others are
// left as they are.
int oe_join_parts(const Kv8Call* call) {
    const Kv8Call& c = *call;
    if (c.bytes != (int)sizeof(Kv8Call)) return OE_ERR_UNSUPPORTED;
    const long long rows = (long long)c.n_tokens * c.H;
    if (rows <= 0) return 0;
    const int n = c.shares > 1 ? c.shares : c.splits;
    if (n < 1 || (rows + 7) / 8 > 0x7fffffffLL) return OE_ERR_UNSUPPORTED;
    return oe_launch(join_parts_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, c.stream, c.out, (const float*)c.part_o, (const float*)c.part_ml,
                     c.cu_q + c.n_seqs, c.H, rows, n);
}

// Attention of the step's tokens over the 8-bit cache (kind OE_KV_INT8 or OE_KV_E4M3), which has their rows already.  mt: tiles of 128
// rows a CTA has (1 or 2); splits > 1: the pages of a tile are cut into as many runs, whose parts are joined.
int oe_attn_rows(const Kv8Call* call) {
    const Kv8Call& c = *call;
    if (c.bytes != (int)sizeof(Kv8Call)) return OE_ERR_UNSUPPORTED;
    if (c.n_seqs <= 0 || c.max_qlen <= 0) return 0;
    const Args a = arguments(c);
    if (!operands_ok(a, c.cache) || ((uintptr_t)c.out & 15) || (c.mt != 1 && c.mt != 2)) return OE_ERR_UNSUPPORTED;
    if (c.splits > 1 && (c.part_o == nullptr || c.part_ml == nullptr)) return OE_ERR_UNSUPPORTED;
    const int tpt = BM / (c.H / c.KVH) * c.mt;
    const long long tiles = ((long long)c.max_qlen + tpt - 1) / tpt, x = (long long)c.KVH * c.splits;
    if (tiles > 65535 || c.n_seqs > 65535 || x > 0x7fffffffLL) return OE_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)x, c.n_seqs, (unsigned)tiles);
    const CUtensorMap none = {};
    int rc = OE_ERR_UNSUPPORTED;
    if (c.kind == OE_KV_INT8) rc = launch_tiles<OE_KV_INT8, false>(c.mt, none, a, grid, c.stream);
    else if (c.kind == OE_KV_E4M3) rc = launch_tiles<OE_KV_E4M3, false>(c.mt, none, a, grid, c.stream);
    if (rc || c.splits == 1) return rc;
    return oe_join_parts(call);
}

// The parts of the groups' prefixes, `splits` a row (oe_attn_kv8 with seq_pages adds them).
int oe_attn_rows_prefix(const Kv8Call* call) {
    const Kv8Call& c = *call;
    if (c.bytes != (int)sizeof(Kv8Call)) return OE_ERR_UNSUPPORTED;
    if (c.n_groups <= 0 || c.n_members <= 0) return 0;
    const Args a = arguments(c);
    if (!operands_ok(a, c.cache) || (c.mt != 1 && c.mt != 2) || c.part_o == nullptr || c.part_ml == nullptr) return OE_ERR_UNSUPPORTED;
    const int tpt = BM / (c.H / c.KVH) * c.mt;
    const long long tiles = ((long long)c.n_members + tpt - 1) / tpt, x = (long long)c.KVH * c.splits;
    if (tiles > 65535 || c.n_groups > 65535 || x > 0x7fffffffLL) return OE_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)x, c.n_groups, (unsigned)tiles);
    CUtensorMap map = {};
    if (c.kind == OE_KV_BF16) {
        // the cache entry as rows of HD: [pages * 2 * KVH * 64][HD]; a box is 64 rows x 64 dims
        if (c.n_pages * 2 * c.KVH * BN > 0x7fffffffLL - BN) return OE_ERR_UNSUPPORTED;
        int rc = get_encode();
        if (rc) return rc;
        cuuint64_t dims[2] = {(cuuint64_t)HD, (cuuint64_t)c.n_pages * 2 * c.KVH * BN};
        cuuint64_t strides[1] = {(cuuint64_t)HD * 2};
        cuuint32_t box[2] = {64, (cuuint32_t)BN};
        cuuint32_t es[2] = {1, 1};
        CUresult r = g_encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, c.cache, dims, strides, box, es,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return 2000 + (int)r;
        return launch_tiles<OE_KV_BF16, true>(c.mt, map, a, grid, c.stream);
    }
    if (c.kind == OE_KV_INT8) return launch_tiles<OE_KV_INT8, true>(c.mt, map, a, grid, c.stream);
    if (c.kind == OE_KV_E4M3) return launch_tiles<OE_KV_E4M3, true>(c.mt, map, a, grid, c.stream);
    return OE_ERR_UNSUPPORTED;
}

int oe_attn_rows_error() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_error, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_error, &zero, sizeof(int));
    return v;
}

}  // extern "C"
