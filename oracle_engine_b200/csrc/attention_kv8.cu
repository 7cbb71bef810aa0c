// Attention of a few rows at a time over the paged cache in its 8-bit forms (kv8.cuh) or in bfloat16, and the write of the
// 8-bit forms; compiled for one head size: -DOE_HD=64 or 128.
//
// A row is a (token, query head of the group) pair.  A CTA (or a cluster of CTAs) has up to 8 NT rows of one KV head and a range of
// keys; its warps split the keys in tiles of 32, each with a ring of tiles of its own that cp.async fills and a running
// softmax of its own, and the results are added up in warp order, then in rank order, through shared memory.
//   S^T = K Q^T, O^T += V^T P^T     mma.sync m16n8k16 with float32 sums: keys, then dimensions, are the 16 rows of a product and the
//                           query rows its 8 columns, so that a group of up to 8 heads leaves nothing of it empty.
//     8-bit forms           float16: a code is a float16 exactly, so K and V enter as codes.  The turned queries are rounded to float16
//                           (2^-12 of themselves; a row is scaled by a power of two first), the key's scale multiplies the score's
//                           sum, and the weight p times the value's scale is rounded to float16: relative to R, the largest power of
//                           two above a value's scale so far, and times 2^8, so that what float16 cannot hold is below 2^-33 of the
//                           row's largest weight.
//     bfloat16              K and V as they are.  Turned queries and weights enter as the sum of two bfloat16 (2^-17 of themselves), which
//                           costs a second product each in a kernel that waits for memory.
//   Reference maximum       moves only when a row's maximum has grown by more than 2^7 since it was set; with it, or when R grows, O is
//                           rescaled, which the factor in the sum cancels.
//   Fragments               the dimensions of a product's inner axis and its rows may be in any order that both operands keep, so a
//                           lane takes 4 dimensions of a row that lie together: K needs one 32-bit load of codes a k-step, V one for 4
//                           dimensions of each of 4 keys, whose bytes are paired by permutes.  P^T comes from S^T by movmatrix.
// Masks: key <= the row's position; window > 0 the last `window` keys, window < 0 the keys of the row's chunk.  A masked key's weight is
// set to zero whatever its score and scale are, so rows behind the last token of a page may hold anything.
// A page number outside the cache counts as a page without keys; a row at a position without an angle comes out undefined, and its token's key and
// value are not written.
// Measured (us; B200, 8 KV heads; with the write of the new tokens' rows):  64 sequences of 144 to 4,019 keys, 24 heads of 128, int8, 290 MB:
// 69, 4.2 TB/s, 65 % of the measured copy; one of 32,000, 32 heads of 128, e4m3: 23 with the kernel that joins 37 parts, 2.9 TB/s; 16 with a
// window of 1,024, 32 heads of 64: 9.3, 1.9 TB/s; one of 137 keys: 6.4.  Where there are few keys the chain of loads bounds it: the sequence's
// numbers, its pages, queries and rows, then the join.  Where there are many, no unit is full (64 sequences in int8 / e4m3: issue slots
// 48 / 46 %, logic pipe 46 / 53 %, DRAM 47 / 55 %): the codes' conversion and the products are chains of dependent instructions, and an SM has
// eight warps for them.  A third CTA of four warps does not help (see `len`).
#include "kv8.cuh"

#ifndef OE_HD
#define OE_HD 128
#endif

namespace {

constexpr int HD = OE_HD;
static_assert(HD == 64 || HD == 128, "built for head_dim 64 or 128");
constexpr int KS = HD / 16;
constexpr int TB = 32;                           // keys per tile: half a page
constexpr int PARTS = OE_PAGE / TB;
constexpr int MAX_ORDERED = 256;
constexpr int MAX_JOINED = 160;                  // parts that a result is joined from: a cluster's CTAs and a prefix's splits
constexpr float LOG2E = 1.4426950408889634f;

// ------------------------------------------------------------------------------------------------ the write
// Keys and values of a step's tokens into the 8-bit cache.  HD / 16 lanes have a token's key and value of one KV head: 8 dimensions of
// the lower half and the 8 that they are turned with, so that a row's lanes read 16 bytes each of both halves and only its maximum
// crosses lanes.  Both rows are asked for at once and share the look-ups of the token's place.
// Measured (B200): 7,440 tokens of 24 heads over 8 KV heads of 128 in int8, 46 MB, 16 us: 2.8 TB/s (a lane group a row: 21 us), bound by the
// loads' latency, at 32 warps an SM, and by the instructions of the exact roundings; one token 1.9 us, 64 tokens 3.8: the start of a
// kernel and two rounds of loads.
template <int KIND>
__global__ void __launch_bounds__(256)
kv8_write_kernel(const bf16* qkv, long long stride, const float* __restrict__ cos_tab, const float* __restrict__ sin_tab,
                 uint8_t* codes, float* scales, long long n_pages, const int* __restrict__ tables, int max_pages,
                 const int* __restrict__ tok_seq, const int* __restrict__ tok_pos, int n_tokens, int H, int KVH, int n_positions, int n_tables) {
    constexpr int LANES = HD / 16;
    pdl_launch_dependents();
    pdl_wait();
    const unsigned item = blockIdx.x * 256u + threadIdx.x, r = item / LANES, t = r / (unsigned)KVH;       // (token, KV head)
    const int i = (int)(item % LANES) * 8, kvh = (int)(r - t * (unsigned)KVH);
    // (two rounds of loads: the rows and the token's place, then the page's number and the angle)
    const bool here = t < (unsigned)n_tokens;
    const bf16* row = qkv + (long long)(here ? t : 0) * stride + (long long)(H + kvh) * HD + i;
    const uint4 k0 = *(const uint4*)row, k1 = *(const uint4*)(row + HD / 2);
    const uint4 v0 = *(const uint4*)(row + KVH * HD), v1 = *(const uint4*)(row + KVH * HD + HD / 2);
    const int b = here ? tok_seq[t] : -1, pos = here ? tok_pos[t] : 0;
    const bool placed = b >= 0 && b < n_tables && pos >= 0 && pos < n_positions;
    const bool turns = cos_tab != nullptr && placed;
    float cs[8], sn[8];
    if (turns) {
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            *(float4*)&cs[j] = *(const float4*)(cos_tab + (long long)pos * (HD / 2) + i + j);
            *(float4*)&sn[j] = *(const float4*)(sin_tab + (long long)pos * (HD / 2) + i + j);
        }
    }
    const int page = placed && pos / OE_PAGE < max_pages ? tables[(long long)b * max_pages + pos / OE_PAGE] : -1;
    const bool ok = page >= 0 && page < n_pages;
    const long long at = ((long long)page * 2 * KVH + kvh) * OE_PAGE + pos % OE_PAGE;
    auto quantise = [&](const uint32_t (&lo)[4], const uint32_t (&hi)[4], long long to) {      // dimensions i .. i + 7, and those they are turned with
        uint32_t w[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) most = kv8_most(most, w[j]);
        most = kv8_most(most);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        float scale;
        const float by = kv8_row<KIND>(most, w, &scale);
        if (!ok) return;
        *(uint2*)(codes + to * HD + i) = make_uint2(kv8_codes4<KIND>(by, w[0], w[1]), kv8_codes4<KIND>(by, w[2], w[3]));
        *(uint2*)(codes + to * HD + i + HD / 2) = make_uint2(kv8_codes4<KIND>(by, w[4], w[5]), kv8_codes4<KIND>(by, w[6], w[7]));
        if (i == 0) scales[to] = scale;
    };
    const uint32_t vl[4] = {v0.x, v0.y, v0.z, v0.w}, vh[4] = {v1.x, v1.y, v1.z, v1.w};
    quantise(vl, vh, at + (long long)KVH * OE_PAGE);       // (the value first: it needs no angle)
    uint32_t lo[4] = {k0.x, k0.y, k0.z, k0.w}, hi[4] = {k1.x, k1.y, k1.z, k1.w};
    if (turns) kv8_turn<8>(lo, hi, cs, sn);
    quantise(lo, hi, at);
}

// ------------------------------------------------------------------------------------------------ the attention
struct Args {
    bf16* out;                 // [T, H*HD]
    const bf16* q;             // rows of q_stride elements: the projections, queries first, not yet turned
    long long q_stride;
    const float* cos_tab;      // [max_pos, HD/2] or null
    const float* sin_tab;
    const void* cache;         // one cache entry's codes, or its bfloat16 rows
    const float* scales;       // of the 8-bit forms
    void* cache_w;             // the same two, where this kernel writes the step's new keys and values (one token a sequence); else null
    float* scales_w;
    long long n_pages;
    const int* tables;         // [B, max_pages]
    int max_pages;
    const int* cu_q;           // [B+1] first packed row of each sequence
    const int* seq_start;      // [B] cache length before the step
    const int* seq_qlen;       // [B]
    int H, KVH, window;
    int n_positions;           // that the angles are there for
    float scale_log2;
    int cluster;               // CTAs that share a tile of rows
    int ahead;                 // rows of earlier tokens may be read before the wait
    int late;                  // the kernel before this one is that of the prefixes, which lets this one start when what it waits for is
                               // done: only its parts have to be waited for
    int ordered;               // n: blockIdx.z counts the n sequences by their lengths, the longest first
    // sequences that begin with the same pages: what attention_rows.cu has left of those pages
    const int* seq_pages;      // [B] pages of the sequence's prefix (0: none); null: no prefixes
    int splits;
    const float* part_o;       // [B * H, splits, HD]
    const float* part_ml;      // [B * H, splits, 2]
    // 1, or how many CTAs that are no cluster share a tile of rows: each leaves a part for the kernel that joins them
    int shares;
    float* own_o;              // [T * H, shares, HD]
    float* own_ml;             // [T * H, shares, 2]
};

template <int S, int G>
__device__ __forceinline__ void cp_async16(uint32_t smem, const uint8_t* gmem) {
    asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%3], 16;" ::"r"(smem), "l"(gmem), "n"(S), "n"(G) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *(uint32_t*)&h;
}
// What pack_bf16(lo, hi) = h leaves of the two, again as bfloat16.
__device__ __forceinline__ uint32_t rest_bf16(float lo, float hi, uint32_t h) {
    return pack_bf16(lo - __uint_as_float(h << 16), hi - __uint_as_float(h & 0xffff0000u));
}
__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Every thread of every CTA of the cluster calls it.
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_address(const void* p, uint32_t rank) {
    uint32_t addr;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return addr;
}
__device__ __forceinline__ float4 ld_peer4(const float* p, uint32_t rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer_address(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_peer2(const float* p, uint32_t rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(peer_address(p, rank)) : "memory");
    return v;
}

// A tile of 32 keys in shared memory: rows padded so that the loads of a fragment fall into different banks.
template <int KIND>
struct Tile {
    static constexpr int ELEM = KIND == OE_KV_BF16 ? 2 : 1;
    static constexpr int K_ROW = HD * ELEM + (KIND == OE_KV_BF16 ? 32 : 16), V_ROW = HD * ELEM + 16;
    static constexpr int V_AT = TB * K_ROW, S_AT = V_AT + TB * V_ROW;         // S: 32 scales of keys, 32 of values
    static constexpr int BYTES = S_AT + (KIND == OE_KV_BF16 ? 0 : 2 * TB * 4);
};

template <int KIND, int I>
__device__ __forceinline__ void load_rows(uint32_t st, const uint8_t* kg, const uint8_t* vg) {
    using L = Tile<KIND>;
    constexpr int AT_ONCE = 512 / (HD * L::ELEM);             // rows that a warp asks for with one instruction
    cp_async16<I * AT_ONCE * L::K_ROW, I * 512>(st, kg);
    cp_async16<L::V_AT + I * AT_ONCE * L::V_ROW, I * 512>(st, vg);
    if constexpr (I + 1 < TB / AT_ONCE) load_rows<KIND, I + 1>(st, kg, vg);
}
template <int I>
__device__ __forceinline__ void load_rows_apart(uint32_t ks, uint32_t vs, const uint8_t* kg, const uint8_t* vg) {
    using L = Tile<OE_KV_BF16>;
    constexpr int AT_ONCE = 512 / (HD * 2);
    cp_async16<I * AT_ONCE * L::K_ROW, I * 512>(ks, kg);
    cp_async16<L::V_AT + I * AT_ONCE * L::V_ROW, I * 512>(vs, vg);
    if constexpr (I + 1 < TB / AT_ONCE) load_rows_apart<I + 1>(ks, vs, kg, vg);
}
template <int KIND>
__device__ __forceinline__ void load_tile(uint8_t* st, const Args& a, int page, int part, int kvh, int lane) {
    using L = Tile<KIND>;
    if ((unsigned)page < (unsigned long long)a.n_pages) {
        const long long krow = (((long long)page * 2) * a.KVH + kvh) * OE_PAGE + part * TB, vrow = krow + (long long)a.KVH * OE_PAGE;
        constexpr int PER_ROW = HD * L::ELEM / 16;
        const uint8_t* kg = (const uint8_t*)a.cache + krow * (HD * L::ELEM) + lane * 16;
        const uint8_t* vg = kg + (long long)a.KVH * (OE_PAGE * HD * L::ELEM);
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(st) + (lane / PER_ROW) * L::K_ROW + (lane % PER_ROW) * 16;
        static_assert(L::K_ROW == L::V_ROW || KIND == OE_KV_BF16, "one offset for both");
        if constexpr (KIND == OE_KV_BF16) load_rows_apart<0>(to, to - (lane / PER_ROW) * (L::K_ROW - L::V_ROW), kg, vg);
        else load_rows<KIND, 0>(to, kg, vg);
        if (KIND != OE_KV_BF16 && lane < 2 * TB / 4)
            cp_async16<L::S_AT, 0>((uint32_t)__cvta_generic_to_shared(st) + lane * 16, (const uint8_t*)(a.scales + (lane < TB / 4 ? krow : vrow - TB) + lane * 4));
    }
}

__device__ __forceinline__ int page_at(const int* trow, int j, int max_pages) { return j < max_pages ? trow[j] : -1; }

// The new token's key and value, made by one warp: its cache rows' bytes.  A lane with an even number has PP pairs of words (or of
// bytes) of the key, one with an odd number of the value: dimensions d .. d + 2 PP - 1 and d + HD/2 .., d = lane / 2 * 2 PP.
template <int KIND>
struct NewToken {
    static constexpr int PP = HD / 64;                      // words a half; HD / 32 dimensions
    uint32_t w[2 * PP];                                     // bfloat16 pairs; in the 8-bit forms the codes in w[0] and w[1]
    float scale;
    __device__ __forceinline__ void make(const Args& a, const bf16* row, int pos, int kvh, int lane) {
        const int d = lane / 2 * 2 * PP;
        const bf16* src = row + (size_t)(a.H + (lane & 1) * a.KVH + kvh) * HD + d;
        uint32_t lo[PP], hi[PP], most = 0;
#pragma unroll
        for (int j = 0; j < PP; j++) { lo[j] = __ldcg((const uint32_t*)(src + 2 * j)); hi[j] = __ldcg((const uint32_t*)(src + HD / 2 + 2 * j)); }
        if (!(lane & 1) && a.cos_tab != nullptr) {
            float cs[2 * PP], sn[2 * PP];
#pragma unroll
            for (int j = 0; j < 2 * PP; j++) { cs[j] = a.cos_tab[(size_t)pos * (HD / 2) + d + j]; sn[j] = a.sin_tab[(size_t)pos * (HD / 2) + d + j]; }
            kv8_turn<2 * PP>(lo, hi, cs, sn);
        }
#pragma unroll
        for (int j = 0; j < PP; j++) { w[j] = lo[j]; w[PP + j] = hi[j]; most = kv8_most(kv8_most(most, lo[j]), hi[j]); }
        if (KIND != OE_KV_BF16) {
            most = kv8_most(most);
#pragma unroll
            for (int o = 2; o < 32; o *= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            const float by = kv8_row<KIND>(most, w, &scale);
            if (PP == 2) {
                w[0] = kv8_codes4<KIND>(by, w[0], w[1]);
                w[1] = kv8_codes4<KIND>(by, w[2], w[2 * PP - 1]);
            } else {
                const uint32_t c = kv8_codes4<KIND>(by, w[0], w[1]);
                w[0] = c & 0xffffu;
                w[1] = c >> 16;
            }
        }
    }
    // rows: where the key's row lies, and how far behind it the value's
    __device__ __forceinline__ void store(uint8_t* krow, size_t to_value, int lane) const {
        uint8_t* row = krow + (lane & 1) * to_value;
        const int d = lane / 2 * 2 * PP;
        if (KIND == OE_KV_BF16) {
#pragma unroll
            for (int j = 0; j < PP; j++) {
                *(uint32_t*)(row + (d + 2 * j) * 2) = w[j];
                *(uint32_t*)(row + (d + HD / 2 + 2 * j) * 2) = w[PP + j];
            }
        } else if (PP == 2) {
            *(uint32_t*)(row + d) = w[0];
            *(uint32_t*)(row + d + HD / 2) = w[1];
        } else {
            *(uint16_t*)(row + d) = (uint16_t)w[0];
            *(uint16_t*)(row + d + HD / 2) = (uint16_t)w[1];
        }
    }
};

// The largest value scale of a tile: lane k has key k's.
__device__ __forceinline__ float warp_most(float v) {
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(v, 0.f))));     // (an undefined one counts as none)
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
    return d;
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The rows are those of one sequence's new tokens (blockIdx.z), the keys its own, from behind its prefix on if it has one, whose
// parts are joined with the result.
template <int KIND, int NT, int NW, int ST>
__global__ void __launch_bounds__(NW * 32)
attn_kv8_kernel(const Args a) {
    using L = Tile<KIND>;
    constexpr bool EIGHT = KIND != OE_KV_BF16;
    constexpr int ROWS = 8 * NT, WARP_BYTES = ST * L::BYTES, OD = HD + 4;
    constexpr float HEADROOM = EIGHT ? 8.f : 0.f, RESCALE_STEP = 7.f;
    static_assert((NW + 1) * ROWS * OD * 4 + ROWS * (MAX_JOINED + NW + 1) * 4 <= NW * WARP_BYTES, "the parts lie where the rings were");
    extern __shared__ __align__(16) uint8_t smem[];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    const int G = a.H / a.KVH, kvh = blockIdx.y;
    const int CR = a.cluster, rank = CR > 1 ? (int)cluster_ctarank() : 0;
    const int bx = blockIdx.x / (CR * a.shares);
    int b = blockIdx.z;
    if (a.ordered) {
        // more CTAs than there is room for: the long sequences' start first, so that the short ones' fill the end
        // With heads of 128 the list leaves an SM room for two CTAs of four warps.  Kept where the rings are, which makes room for three (us):
        // 64 sequences of 144 to 4,019 keys 88 instead of 69, one of 32,000 in 37 parts 27 instead of 23, 32 behind 4,096 common tokens 27.8
        // instead of 25.4; only many short ones gain, 200 of 100 to 900 keys 43 instead of 52.
        __shared__ int len[MAX_ORDERED], which;
        for (int t = threadIdx.x; t < a.ordered; t += NW * 32)
            len[t] = a.seq_qlen[t] > 0 ? a.seq_start[t] + 1 - (a.seq_pages != nullptr ? a.seq_pages[t] * OE_PAGE : 0) : 0;
        __syncthreads();
        for (int t = threadIdx.x; t < a.ordered; t += NW * 32) {
            int before = 0;
            for (int j = 0; j < a.ordered; j++) before += len[j] > len[t] || (len[j] == len[t] && j < t);
            if (before == b) which = t;
        }
        __syncthreads();
        b = which;
    }
    // (the step's integers, asked for together; they were written before its first kernel)
    const int qlen = a.seq_qlen[b], start = a.seq_start[b], common = a.seq_pages != nullptr ? a.seq_pages[b] : 0;
    const long long packed0 = a.cu_q[b];
    const int row0 = bx * ROWS, n_rows = qlen > 0 ? qlen * G : 0;
    if (row0 >= n_rows) {                                            // the whole cluster
        pdl_wait();
        return;
    }
    const int rows = min(ROWS, n_rows - row0);
    int key_lo = oe_first_key(start + row0 / G, a.window);
    const int key_hi = start + (row0 + rows - 1) / G;
    key_lo = max(key_lo, common * OE_PAGE);
    const int* trow = a.tables + (size_t)b * a.max_pages;
    uint8_t* mine = smem + (size_t)warp * WARP_BYTES;
    const int share = a.shares > 1 ? (int)blockIdx.x % a.shares : rank, gw = share * NW + warp, stride = NW * CR * a.shares;
    const int t_lo = key_lo / TB, t_hi = key_hi >= key_lo ? key_hi / TB : t_lo - 1;
    const int n_my = t_lo + gw <= t_hi ? (t_hi - t_lo - gw) / stride + 1 : 0;
    const bool own_kv = a.cache_w != nullptr;
    // where the caller says so, keys and values of earlier steps are asked for before the wait: only the new token's q, k and v
    // come from the kernel before this one
    const bool ahead = a.ahead && own_kv && !a.late;
    if (!ahead && !a.late) pdl_wait();
    // The queries of the rows nt * 8 + gid, 4 dimensions that lie together a k-step, and their angles: asked for before the tiles where
    // the kernel before this one has been waited for, since a score needs both.
    uint2 qw[NT][KS];
    float4 qc[NT][KS / 2], qs[NT][KS / 2];
    auto ask_for_queries = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = nt * 8 + gid, rr = row0 + (r < rows ? r : 0);
            const bf16* src = a.q + (packed0 + rr / G) * a.q_stride + (size_t)(kvh * G + rr % G) * HD + tig * 4;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) qw[nt][ks] = r < rows ? __ldcg((const uint2*)(src + ks * 16)) : make_uint2(0u, 0u);
            if (a.cos_tab != nullptr) {
                const size_t at = (size_t)min((unsigned)(start + rr / G), (unsigned)a.n_positions - 1u) * (HD / 2) + tig * 4;
#pragma unroll
                for (int ks = 0; ks < KS / 2; ks++) {
                    qc[nt][ks] = *(const float4*)(a.cos_tab + at + ks * 16);
                    qs[nt][ks] = *(const float4*)(a.sin_tab + at + ks * 16);
                }
            }
        }
    };
    if (!ahead) ask_for_queries();
    // the page numbers of this warp's next 32 tiles, one a lane, and of the 32 behind them
    auto pages_from = [&](int it) { return it + lane < n_my ? page_at(trow, (t_lo + gw + (it + lane) * stride) / PARTS, a.max_pages) : -1; };
    int pages = pages_from(0), pages_next = pages_from(32);
#pragma unroll
    for (int pre = 0; pre < ST; pre++) {
        const int page = __shfl_sync(0xffffffffu, pages, pre);
        if (pre < n_my) load_tile<KIND>(mine + pre * L::BYTES, a, page, (t_lo + gw + pre * stride) % PARTS, kvh, lane);
        cp_async_commit();
    }
    if (ahead) {
        pdl_wait();
        ask_for_queries();
    }
    // Q fragments, turned: qf, and for a 16-bit cache what its rounding leaves; a row's power of two
    constexpr int KL = EIGHT ? 1 : KS;
    uint32_t qf[NT][KS][2], ql[NT][KL][2];
    float up[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float qv[KS][4];
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const uint2 w = qw[nt][ks];
            qv[ks][0] = kv8_from_bits(w.x); qv[ks][1] = __uint_as_float(w.x & 0xffff0000u);
            qv[ks][2] = kv8_from_bits(w.y); qv[ks][3] = __uint_as_float(w.y & 0xffff0000u);
        }
        if (a.cos_tab != nullptr) {
#pragma unroll
            for (int ks = 0; ks < KS / 2; ks++) {
                const float cc[4] = {qc[nt][ks].x, qc[nt][ks].y, qc[nt][ks].z, qc[nt][ks].w}, nn[4] = {qs[nt][ks].x, qs[nt][ks].y, qs[nt][ks].z, qs[nt][ks].w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = qv[ks][e], y = qv[ks + KS / 2][e];
                    qv[ks][e] = x * cc[e] - y * nn[e];
                    qv[ks + KS / 2][e] = x * nn[e] + y * cc[e];
                }
            }
        }
        float down = 1.f;
        up[nt] = 1.f;
        if (EIGHT) {
            float most = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
#pragma unroll
                for (int e = 0; e < 4; e++) most = fmaxf(most, fabsf(qv[ks][e]));
            }
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            down = kv8_row_factor(most, &up[nt]);
        }
        const int at = start + (row0 + (nt * 8 + gid < rows ? nt * 8 + gid : 0)) / G;
        if ((unsigned)at >= (unsigned)a.n_positions) up[nt] = __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                // (a pair of the keys' codes: kv8_first and kv8_second)
                const float q0 = qv[ks][KIND == OE_KV_INT8 ? x : 2 * x] * down, q1 = qv[ks][KIND == OE_KV_INT8 ? x + 2 : 2 * x + 1] * down;
                if (EIGHT) {
                    qf[nt][ks][x] = pack_f16(q0, q1);
                } else {
                    qf[nt][ks][x] = pack_bf16(q0, q1);
                    ql[nt][EIGHT ? 0 : ks][x] = rest_bf16(q0, q1, qf[nt][ks][x]);
                }
            }
        }
    }
    // this lane's columns of S^T and O^T: rows nt * 8 + tig * 2 + e
    float row_scale[NT][2], m_run[NT][2], l_run[NT][2];
    int pos[NT][2], low[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = nt * 8 + tig * 2 + e, rr = row0 + (r < rows ? r : 0);
            pos[nt][e] = start + rr / G;
            low[nt][e] = oe_first_key(pos[nt][e], a.window);
            row_scale[nt][e] = a.scale_log2 * __shfl_sync(0xffffffffu, up[nt], (tig * 2 + e) * 4);
            m_run[nt][e] = -INFINITY;
            l_run[nt][e] = 0.f;
        }
    }
    // the warp that meets the new token's tile makes that token's rows and stores them in the cache
    // (without an angle it is not made, and the row's result, the only one that its key is for, is undefined)
    const bool owner = own_kv && n_my > 0 && (t_hi - t_lo - gw) % stride == 0 && (unsigned)start < (unsigned)a.n_positions;
    NewToken<KIND> fresh;
    if (owner) {
        fresh.make(a, a.q + packed0 * a.q_stride, start, kvh, lane);
        const int page = page_at(trow, start / OE_PAGE, a.max_pages);
        if ((unsigned)page < (unsigned long long)a.n_pages) {
            const long long krow = (((long long)page * 2) * a.KVH + kvh) * OE_PAGE + start % OE_PAGE, vrow = krow + (long long)a.KVH * OE_PAGE;
            fresh.store((uint8_t*)a.cache_w + krow * (HD * L::ELEM), (size_t)a.KVH * OE_PAGE * HD * L::ELEM, lane);
            if (EIGHT && lane < 2) a.scales_w[lane ? vrow : krow] = fresh.scale;
        }
    }

    float oacc[NT][HD / 16][4];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int n = 0; n < HD / 16; n++) { oacc[nt][n][0] = oacc[nt][n][1] = oacc[nt][n][2] = oacc[nt][n][3] = 0.f; }
    }
    float ref = kv8_above(0.f);                             // R: what O is relative to
    int stage = 0;
    for (int it = 0; it < n_my; it++) {
        const int tile = t_lo + gw + it * stride;
        uint8_t* cur = mine + (size_t)stage * L::BYTES;
        const int page = __shfl_sync(0xffffffffu, pages, it & 31);
        const int page_ahead = __shfl_sync(0xffffffffu, (it & 31) + ST < 32 ? pages : pages_next, (it + ST) & 31);
        if ((it & 31) == 31) {
            pages = pages_next;
            pages_next = pages_from(it + 33);
        }
        cp_async_wait<ST - 1>();
        __syncwarp();
        if (own_kv && tile == t_hi) {
            const int r = start % TB;
            fresh.store(cur + r * L::K_ROW, L::V_AT + r * (L::V_ROW - L::K_ROW), lane);
            if (EIGHT && lane < 2) ((float*)(cur + L::S_AT))[lane * TB + r] = fresh.scale;
            __syncwarp();
        }
        if ((unsigned)page < (unsigned long long)a.n_pages) {
            float s[NT][TB / 16][4];
#pragma unroll
            for (int mt = 0; mt < TB / 16; mt++) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) s[nt][mt][0] = s[nt][mt][1] = s[nt][mt][2] = s[nt][mt][3] = 0.f;
                const uint8_t* kr = cur + (mt * 16 + gid) * L::K_ROW + tig * 4 * L::ELEM;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    uint32_t f[4];
                    if (EIGHT) {
                        const uint32_t w0 = *(const uint32_t*)(kr + ks * 16), w1 = *(const uint32_t*)(kr + 8 * L::K_ROW + ks * 16);
                        f[0] = kv8_first<KIND>(w0); f[2] = kv8_second<KIND>(w0);
                        f[1] = kv8_first<KIND>(w1); f[3] = kv8_second<KIND>(w1);
                    } else {
                        const uint2 w0 = *(const uint2*)(kr + ks * 32), w1 = *(const uint2*)(kr + 8 * L::K_ROW + ks * 32);
                        f[0] = w0.x; f[2] = w0.y; f[1] = w1.x; f[3] = w1.y;
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        if (EIGHT) {
                            mma_f16(s[nt][mt], f, qf[nt][ks][0], qf[nt][ks][1]);
                        } else {
                            mma_bf16(s[nt][mt], f, qf[nt][ks][0], qf[nt][ks][1]);
                            mma_bf16(s[nt][mt], f, ql[nt][EIGHT ? 0 : ks][0], ql[nt][EIGHT ? 0 : ks][1]);
                        }
                    }
                }
            }
            const float* sc = (const float*)(cur + L::S_AT);
            const int k0 = tile * TB;
            bool whole = k0 >= key_lo;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) whole = whole && k0 + TB - 1 <= min(pos[nt][0], pos[nt][1]) && k0 >= max(low[nt][0], low[nt][1]);
            const bool mask = !__all_sync(0xffffffffu, whole);
            float ksc[TB / 8], vsc[TB / 8], grown = 1.f;
            if (EIGHT) {
                float sv = sc[TB + lane];
                if (mask && (k0 + lane < key_lo || k0 + lane > key_hi)) sv = 0.f;
                const float next = fmaxf(ref, kv8_above(warp_most(sv))), inv = kv8_inverse(next);
                grown = ref * inv;
                ref = next;
#pragma unroll
                for (int o = 0; o < TB / 8; o++) { ksc[o] = sc[o * 8 + gid]; vsc[o] = sc[TB + o * 8 + gid] * inv; }
            }
            float m_new[NT][2];
            bool move = EIGHT && grown != 1.f;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float most = -INFINITY;
#pragma unroll
                    for (int o = 0; o < TB / 8; o++) {
                        float& v = s[nt][o / 2][(o & 1) * 2 + e];
                        if (EIGHT) v *= ksc[o];
                        if (mask) {
                            const int key = k0 + o * 8 + gid;
                            v = key >= key_lo && key <= pos[nt][e] && key >= low[nt][e] ? v : -INFINITY;
                        }
                        most = fmaxf(most, v);
                    }
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
                    m_new[nt][e] = fmaxf(m_run[nt][e], most * row_scale[nt][e]);
                    move = move || m_new[nt][e] > m_run[nt][e] + RESCALE_STEP;
                }
            }
            if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float alpha[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        alpha[e] = fast_exp2(m_run[nt][e] - (m_new[nt][e] == -INFINITY ? 0.f : m_new[nt][e]));
                        l_run[nt][e] *= alpha[e];
                        alpha[e] *= grown;
                        m_run[nt][e] = m_new[nt][e];
                    }
#pragma unroll
                    for (int n = 0; n < HD / 16; n++) {
                        oacc[nt][n][0] *= alpha[0]; oacc[nt][n][1] *= alpha[1];
                        oacc[nt][n][2] *= alpha[0]; oacc[nt][n][3] *= alpha[1];
                    }
                }
            }
            // weights, as the columns' fragments
            uint32_t pf[NT][TB / 8], pl[NT][EIGHT ? 1 : TB / 8];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const float n0 = (m_run[nt][0] == -INFINITY ? 0.f : -m_run[nt][0]) + HEADROOM;
                const float n1 = (m_run[nt][1] == -INFINITY ? 0.f : -m_run[nt][1]) + HEADROOM;
#pragma unroll
                for (int o = 0; o < TB / 8; o++) {
                    const float v0 = s[nt][o / 2][(o & 1) * 2], v1 = s[nt][o / 2][(o & 1) * 2 + 1];
                    float p0 = fast_exp2(fmaf(v0, row_scale[nt][0], n0)), p1 = fast_exp2(fmaf(v1, row_scale[nt][1], n1));
                    l_run[nt][0] += p0;
                    l_run[nt][1] += p1;
                    if (EIGHT) {
                        p0 = mask && v0 == -INFINITY ? 0.f : p0 * vsc[o];
                        p1 = mask && v1 == -INFINITY ? 0.f : p1 * vsc[o];
                        pf[nt][o] = transposed(pack_f16(p0, p1));
                    } else {
                        const uint32_t h = pack_bf16(p0, p1);
                        pf[nt][o] = transposed(h);
                        pl[nt][EIGHT ? 0 : o] = transposed(rest_bf16(p0, p1, h));
                    }
                }
            }
#pragma unroll
            for (int kk = 0; kk < TB / 16; kk++) {
                const uint8_t* vr = cur + L::V_AT + (kk * 16 + tig * 2) * L::V_ROW + gid * 4 * L::ELEM;
#pragma unroll
                for (int c = 0; c < HD / 32; c++) {
                    uint32_t f[2][4];                       // dims c * 32 + gid * 4 + {0, 1} and + {2, 3}
                    if (EIGHT) {
                        uint32_t w0 = *(const uint32_t*)(vr + c * 32), w1 = *(const uint32_t*)(vr + L::V_ROW + c * 32);
                        uint32_t w2 = *(const uint32_t*)(vr + 8 * L::V_ROW + c * 32), w3 = *(const uint32_t*)(vr + 9 * L::V_ROW + c * 32);
                        if (KIND == OE_KV_E4M3 && mask) {      // (as below; every int8 code is a number)
                            const int key = k0 + kk * 16 + tig * 2;
                            if (key < key_lo || key > key_hi) w0 = 0u;
                            if (key + 1 < key_lo || key + 1 > key_hi) w1 = 0u;
                            if (key + 8 < key_lo || key + 8 > key_hi) w2 = 0u;
                            if (key + 9 < key_lo || key + 9 > key_hi) w3 = 0u;
                        }
                        constexpr uint32_t LOWER = KIND == OE_KV_INT8 ? 0x5410u : 0x5140u, UPPER = KIND == OE_KV_INT8 ? 0x7632u : 0x7362u;
                        const uint32_t x0 = kv8_prmt(w0, w1, LOWER), x1 = kv8_prmt(w0, w1, UPPER);
                        const uint32_t y0 = kv8_prmt(w2, w3, LOWER), y1 = kv8_prmt(w2, w3, UPPER);
                        f[0][0] = kv8_first<KIND>(x0); f[0][1] = kv8_second<KIND>(x0); f[0][2] = kv8_first<KIND>(y0); f[0][3] = kv8_second<KIND>(y0);
                        f[1][0] = kv8_first<KIND>(x1); f[1][1] = kv8_second<KIND>(x1); f[1][2] = kv8_first<KIND>(y1); f[1][3] = kv8_second<KIND>(y1);
                    } else {
                        uint2 w0 = *(const uint2*)(vr + c * 64), w1 = *(const uint2*)(vr + L::V_ROW + c * 64);
                        uint2 w2 = *(const uint2*)(vr + 8 * L::V_ROW + c * 64), w3 = *(const uint2*)(vr + 9 * L::V_ROW + c * 64);
                        if (mask) {            // a row behind the last token may hold anything, and 0 times that need not be 0
                            const int key = k0 + kk * 16 + tig * 2;
                            if (key < key_lo || key > key_hi) w0 = make_uint2(0u, 0u);
                            if (key + 1 < key_lo || key + 1 > key_hi) w1 = make_uint2(0u, 0u);
                            if (key + 8 < key_lo || key + 8 > key_hi) w2 = make_uint2(0u, 0u);
                            if (key + 9 < key_lo || key + 9 > key_hi) w3 = make_uint2(0u, 0u);
                        }
                        f[0][0] = kv8_prmt(w0.x, w1.x, 0x5410u); f[0][1] = kv8_prmt(w0.x, w1.x, 0x7632u);
                        f[0][2] = kv8_prmt(w2.x, w3.x, 0x5410u); f[0][3] = kv8_prmt(w2.x, w3.x, 0x7632u);
                        f[1][0] = kv8_prmt(w0.y, w1.y, 0x5410u); f[1][1] = kv8_prmt(w0.y, w1.y, 0x7632u);
                        f[1][2] = kv8_prmt(w2.y, w3.y, 0x5410u); f[1][3] = kv8_prmt(w2.y, w3.y, 0x7632u);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            if (EIGHT) {
                                mma_f16(oacc[nt][c * 2 + j], f[j], pf[nt][2 * kk], pf[nt][2 * kk + 1]);
                            } else {
                                mma_bf16(oacc[nt][c * 2 + j], f[j], pf[nt][2 * kk], pf[nt][2 * kk + 1]);
                                mma_bf16(oacc[nt][c * 2 + j], f[j], pl[nt][EIGHT ? 0 : 2 * kk], pl[nt][EIGHT ? 0 : 2 * kk + 1]);
                            }
                        }
                    }
                }
            }
        }
        __syncwarp();                                       // every lane has read the stage: refill it
        if (it + ST < n_my) {
            load_tile<KIND>(cur, a, page_ahead, (tile + ST * stride) % PARTS, kvh, lane);
        }
        cp_async_commit();
        stage = stage + 1 == ST ? 0 : stage + 1;
    }
    cp_async_wait<0>();
    // the warps' parts, added in warp order
    __syncthreads();                                        // every warp has left its ring
    float* part = (float*)smem;                             // [NW][ROWS][OD]: O, m, l
    float* cpart = part + (size_t)NW * ROWS * OD;           // [ROWS][OD]: this CTA's sum
    float* wts = cpart + ROWS * OD;                         // [ROWS][MAX_JOINED + NW + 1]
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
            for (int d = 4; d < 32; d *= 2) l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], d);
            const int r = nt * 8 + tig * 2 + e;
            if (r >= rows) continue;
            float* p = part + ((size_t)warp * ROWS + r) * OD;
            const float f = EIGHT ? ref : 1.f;
#pragma unroll
            for (int c = 0; c < HD / 32; c++)
                *(float4*)(p + c * 32 + gid * 4) = make_float4(oacc[nt][c * 2][e] * f, oacc[nt][c * 2][2 + e] * f, oacc[nt][c * 2 + 1][e] * f, oacc[nt][c * 2 + 1][2 + e] * f);
            if (gid == 0) *(float2*)(p + HD) = make_float2(m_run[nt][e], l_run[nt][e]);
        }
    }
    __syncthreads();
    // weights of n parts, whose (m, l) lane q < n of this warp has, once or in rounds: into w[0..n), the joined m and l behind it
    constexpr int WT = MAX_JOINED + NW + 1;
    for (int r = warp; r < rows; r += NW) {
        const float2 ml = lane < NW ? *(const float2*)(part + ((size_t)lane * ROWS + r) * OD + HD) : make_float2(-INFINITY, 0.f);
        const float m = warp_max(ml.x), mu = m == -INFINITY ? 0.f : m;
        const float w = ml.x == -INFINITY && ml.y == 0.f ? 0.f : exp2f(ml.x - mu);
        const float l = warp_sum(w == 0.f && ml.y == 0.f ? 0.f : ml.y * w);
        if (lane < NW) wts[r * WT + lane] = w;
        if (lane == 0) {
            *(float2*)(cpart + r * OD + HD) = make_float2(m, l);
            wts[r * WT + MAX_JOINED] = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
        }
    }
    __syncthreads();
    if (a.late) pdl_wait();
    const int n_pre = common > 0 ? a.splits : 0;
    const bool alone = CR == 1 && a.shares == 1 && n_pre == 0;           // nothing to join: the sum is the result
    for (int idx = threadIdx.x; idx < rows * (HD / 4); idx += NW * 32) {
        const int r = idx / (HD / 4), d = idx % (HD / 4) * 4;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float e = wts[r * WT + w];
            const float4 p = *(const float4*)(part + ((size_t)w * ROWS + r) * OD + d);
            o.x = fmaf(p.x, e, o.x); o.y = fmaf(p.y, e, o.y); o.z = fmaf(p.z, e, o.z); o.w = fmaf(p.w, e, o.w);
        }
        if (alone) {
            const float inv = wts[r * WT + MAX_JOINED];
            *(uint2*)(a.out + (packed0 + (row0 + r) / G) * (long long)(a.H * HD) + (long long)(kvh * G + (row0 + r) % G) * HD + d) =
                make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
        } else {
            *(float4*)(cpart + r * OD + d) = o;
        }
    }
    if (alone) return;
    if (a.shares > 1) {                                      // (each thread stores what it has added up)
        for (int idx = threadIdx.x; idx < rows * (HD / 4); idx += NW * 32) {
            const int r = idx / (HD / 4), d = idx % (HD / 4) * 4;
            const long long at = ((packed0 + (row0 + r) / G) * a.H + kvh * G + (row0 + r) % G) * a.shares + share;
            *(float4*)(a.own_o + at * HD + d) = *(const float4*)(cpart + r * OD + d);
            if (d == 0) *(float2*)(a.own_ml + at * 2) = *(const float2*)(cpart + r * OD + HD);
        }
        return;
    }
    if (CR > 1) cluster_sync_all();
    else __syncthreads();
    // this CTA's share of the rows' results: the cluster's sums in rank order, then the prefix's parts
    for (int r = warp; r < rows; r += NW) {
        const int h = kvh * G + (row0 + r) % G;
        const float2* pre_ml = (const float2*)a.part_ml + ((long long)b * a.H + h) * a.splits;
        float2 ml[MAX_JOINED / 32];
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int j = 0; j < MAX_JOINED / 32; j++) {
            const int q = j * 32 + lane;
            ml[j] = make_float2(-INFINITY, 0.f);
            if (q < CR) ml[j] = CR > 1 ? ld_peer2(cpart + r * OD + HD, q) : *(const float2*)(cpart + r * OD + HD);
            else if (q < CR + n_pre) ml[j] = pre_ml[q - CR];
            m = fmaxf(m, ml[j].x);
        }
        m = warp_max(m);
        const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int j = 0; j < MAX_JOINED / 32; j++) {
            const int q = j * 32 + lane;
            const bool none = ml[j].x == -INFINITY && ml[j].y == 0.f;           // no key of this row: its O is not there
            const float w = none ? 0.f : exp2f(ml[j].x - mu);
            if (!none) l += ml[j].y * w;
            if (q < CR + n_pre) wts[r * WT + q] = none ? -1.f : w;
        }
        l = warp_sum(l);
        if (lane == 0) wts[r * WT + MAX_JOINED] = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    }
    __syncthreads();
    for (int idx = threadIdx.x + rank * NW * 32; idx < rows * (HD / 4); idx += NW * 32 * CR) {
        const int r = idx / (HD / 4), d = idx % (HD / 4) * 4, h = kvh * G + (row0 + r) % G;
        const float* w = wts + r * WT;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int q = 0; q < CR; q++) {
            if (w[q] < 0.f) continue;
            const float4 p = CR > 1 ? ld_peer4(cpart + r * OD + d, q) : *(const float4*)(cpart + r * OD + d);
            o.x = fmaf(p.x, w[q], o.x); o.y = fmaf(p.y, w[q], o.y); o.z = fmaf(p.z, w[q], o.z); o.w = fmaf(p.w, w[q], o.w);
        }
        const float* pre = a.part_o + (((long long)b * a.H + h) * a.splits) * HD + d;
        for (int q = 0; q < n_pre; q += 8) {                // (eight at a time, whether they count or not: their loads overlap)
            float4 v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = *(const float4*)(pre + min(q + k, n_pre - 1) * HD);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float e = q + k < n_pre ? w[CR + q + k] : -1.f;
                if (e < 0.f) continue;
                o.x = fmaf(v[k].x, e, o.x); o.y = fmaf(v[k].y, e, o.y); o.z = fmaf(v[k].z, e, o.z); o.w = fmaf(v[k].w, e, o.w);
            }
        }
        const float inv = w[MAX_JOINED];
        *(uint2*)(a.out + (packed0 + (row0 + r) / G) * (long long)(a.H * HD) + (long long)h * HD + d) =
            make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
    }
    if (CR > 1) cluster_sync_all();                         // nobody leaves while its shared memory is read
}

template <int KIND, int NT, int NW, int ST>
int launch(const Args& a, long long rows, int n_seqs, cudaStream_t st) {
    auto kernel = attn_kv8_kernel<KIND, NT, NW, ST>;
    constexpr size_t smem = (size_t)NW * ST * Tile<KIND>::BYTES;
    static_assert(NW != 4 || HD != 128 || 3 * (smem + (MAX_ORDERED + 1) * 4 + 1024) > 228 * 1024, "two CTAs of four warps an SM, as measured");
    const long long x = (rows + 8 * NT - 1) / (8 * NT) * a.cluster * a.shares;
    if (x > 0x7fffffffLL || a.KVH > 65535 || n_seqs > 65535) return OE_ERR_UNSUPPORTED;
    static Kv8Devices set;
    if (set.first()) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        set.done();
    }
    const dim3 grid((unsigned)x, a.KVH, n_seqs);
    if (a.cluster > 1) return oe_launch_cluster(kernel, (unsigned)a.cluster, grid, dim3(NW * 32), smem, st, a);
    return oe_launch(kernel, grid, dim3(NW * 32), smem, st, a);
}
// warps: 12 (a CTA has an SM to itself) or 4 (two an SM with heads of 128, five with 64); of a 16-bit cache, whose tiles are twice as
// large, 6 or 3 (two, three).
template <int KIND, int NT>
int launch_form(int warps, const Args& a, long long rows, int n_seqs, cudaStream_t st) {
    constexpr int MANY = KIND == OE_KV_BF16 ? 6 : 12, FEW = KIND == OE_KV_BF16 ? 3 : 4;
    if (warps == MANY) return launch<KIND, NT, MANY, 2>(a, rows, n_seqs, st);
    if (warps == FEW) return launch<KIND, NT, FEW, 2>(a, rows, n_seqs, st);
    return OE_ERR_UNSUPPORTED;
}
template <int KIND>
int launch_rows(int warps, const Args& a, long long rows, int n_seqs, cudaStream_t st) {
    return rows <= 8 ? launch_form<KIND, 1>(warps, a, rows, n_seqs, st) : launch_form<KIND, 2>(warps, a, rows, n_seqs, st);
}

}  // namespace

extern "C" {

// Keys and values of n_tokens tokens into the 8-bit cache.
int oe_kv8_write(const Kv8Call* call) {
    const Kv8Call& c = *call;
    if (c.bytes != (int)sizeof(Kv8Call)) return OE_ERR_UNSUPPORTED;
    if (c.n_tokens <= 0) return 0;
    if (c.stride % 8 || ((uintptr_t)c.qkv & 15) || ((uintptr_t)c.cache & 15) || ((uintptr_t)c.scales & 15)) return OE_ERR_UNSUPPORTED;
    const long long blocks = ((long long)c.n_tokens * c.KVH * (HD / 16) + 255) / 256;
    if (blocks > 0x00ffffffLL || ((uintptr_t)c.cos_tab & 15) || ((uintptr_t)c.sin_tab & 15)) return OE_ERR_UNSUPPORTED;   // (lanes are counted in 32 bits)
    if (c.kind != OE_KV_INT8 && c.kind != OE_KV_E4M3) return OE_ERR_UNSUPPORTED;
    return oe_launch(c.kind == OE_KV_INT8 ? kv8_write_kernel<OE_KV_INT8> : kv8_write_kernel<OE_KV_E4M3>, dim3((unsigned)blocks), dim3(256), 0, c.stream, c.qkv,
                     c.stride, c.cos_tab, c.sin_tab, (uint8_t*)c.cache, c.scales, c.n_pages, c.tables, c.max_pages, c.tok_seq, c.tok_pos,
                     c.n_tokens, c.H, c.KVH, c.n_positions, c.n_tables);
}

// Attention of the step's tokens over their sequences' caches (kind: OE_KV_*).  write != 0: every sequence brings one token, whose
// key and value this kernel writes.  With seq_pages the pages before a sequence's own are left out and the parts that
// oe_attn_rows_prefix, launched right before with the same argument, left (`splits` a row) are added.  shares > 1: as many CTAs share a tile's keys and leave their parts (oe_join_parts).
int oe_attn_kv8(const Kv8Call* call) {
    const Kv8Call& c = *call;
    if (c.bytes != (int)sizeof(Kv8Call)) return OE_ERR_UNSUPPORTED;
    if (c.n_seqs <= 0 || c.max_qlen <= 0) return 0;
    if (c.KVH <= 0 || c.H % c.KVH || c.stride % 8 || ((uintptr_t)c.qkv & 15) || ((uintptr_t)c.cache & 15) || ((uintptr_t)c.scales & 15) ||
        ((uintptr_t)c.cos_tab & 15) || ((uintptr_t)c.sin_tab & 15) || ((uintptr_t)c.out & 15)) return OE_ERR_UNSUPPORTED;
    if (c.n_positions < 1) return OE_ERR_UNSUPPORTED;
    if (c.cluster < 1 || c.cluster > 8 || (c.cluster & (c.cluster - 1)) || (c.write && c.max_qlen != 1)) return OE_ERR_UNSUPPORTED;
    const bool no_parts = c.part_o == nullptr || c.part_ml == nullptr;
    if (c.seq_pages != nullptr && (c.window != 0 || c.max_qlen != 1 || c.splits < 1 || c.splits + c.cluster > MAX_JOINED || no_parts)) return OE_ERR_UNSUPPORTED;
    if (c.shares < 1 || (c.shares > 1 && (c.cluster != 1 || c.seq_pages != nullptr || no_parts))) return OE_ERR_UNSUPPORTED;
    Args a = {};
    a.out = c.out; a.q = c.qkv; a.q_stride = c.stride; a.cos_tab = c.cos_tab; a.sin_tab = c.sin_tab;
    a.cache = c.cache; a.scales = c.scales;
    if (c.write) { a.cache_w = c.cache; a.scales_w = c.scales; }
    a.n_pages = c.n_pages; a.tables = c.tables; a.max_pages = c.max_pages; a.cu_q = c.cu_q; a.seq_start = c.seq_start; a.seq_qlen = c.seq_qlen;
    a.H = c.H; a.KVH = c.KVH; a.window = c.window; a.n_positions = c.n_positions; a.scale_log2 = c.scale * LOG2E; a.cluster = c.cluster;
    a.seq_pages = c.seq_pages; a.splits = c.splits; a.ahead = c.ahead; a.shares = c.shares;
    a.late = c.seq_pages != nullptr && c.n_groups > 0 && c.n_members > 0;
    if (c.seq_pages != nullptr) { a.part_o = c.part_o; a.part_ml = c.part_ml; }
    else { a.own_o = c.part_o; a.own_ml = c.part_ml; }
    a.ordered = c.ordered && c.window == 0 && c.n_seqs > 1 && c.n_seqs <= MAX_ORDERED ? c.n_seqs : 0;
    const long long rows = (long long)c.max_qlen * (c.H / c.KVH);
    if (c.kind == OE_KV_BF16) return launch_rows<OE_KV_BF16>(c.warps, a, rows, c.n_seqs, c.stream);
    if (c.kind == OE_KV_INT8) return launch_rows<OE_KV_INT8>(c.warps, a, rows, c.n_seqs, c.stream);
    if (c.kind == OE_KV_E4M3) return launch_rows<OE_KV_E4M3>(c.warps, a, rows, c.n_seqs, c.stream);
    return OE_ERR_UNSUPPORTED;
}

}  // extern "C"
