// The 8-bit product for many rows (prompts): tiles of 64 to 256 tokens by 256 rows of w, on the schedule of the bfloat16 tiles (gemm_tiles.h).  Four
// waves, one a SIMD, each with 64 rows of w (one packed block) straight from memory into registers, the activations through LDS; a ring of
// four stages of 128 values of k, one block of each side.
//  * The bytes are those of the bfloat16 tiles: a row of a stage is 128 bytes, a wave's weights 8 KB, and v_mfma_scale_f32_16x16x128_f8f6f4 makes of
//    them in the same time twice the products.
//  * The activations' powers: a lane holds those of its TM tokens of a stage, one load of TM bytes, because row i of token tile t is token
//    i TM + t of the tile and scales hold a block's bytes of neighbouring tokens beside one another; the product picks its byte.  The weights':
//    the four strips' bytes of a stage are one word.
#include "gemm_blocks.h"
#include "gemm_tiles.h"

constexpr int kStageBytes = 128;
static_assert(kTileBlocks == kTileRowBlocks, "rows of w a tile");

// acc += w . a of the blocks' powers 2^(byte STRIP of w_powers - 127) and 2^(byte AT of a_powers - 127).  (Written as an instruction, because the compiler
// otherwise keeps some of the 256 accumulators of the largest tile outside the accumulation registers and moves them in the loop, 72 to 320 moves
// each way a round of 256 products.  The operands come from loads, which the compiler waits for.  FIRST: one of them may have been written by the vector
// unit just before, which needs the wait of the s_nop; where both have been operands before there is none: with it before every product
// the largest tile's loop took 4.4 % more cycles.)
template <int AT, int STRIP, bool FIRST> __device__ __forceinline__ void blocks_mfma(f32x4_t& acc, i32x8_8 w, i32x8_8 a, int w_powers, int a_powers) {
#ifdef __HIP_DEVICE_COMPILE__
#define BLOCKS_MFMA "v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0]"
#define BLOCKS_OPERANDS : "+a"(acc) : "v"(w), "v"(a), "v"(w_powers), "v"(a_powers), "n"(STRIP & 1), "n"(AT & 1), "n"(STRIP >> 1), "n"(AT >> 1)
    if constexpr (FIRST) asm volatile("s_nop 1\n\t" BLOCKS_MFMA BLOCKS_OPERANDS);
    else asm volatile(BLOCKS_MFMA BLOCKS_OPERANDS);
#undef BLOCKS_MFMA
#undef BLOCKS_OPERANDS
#endif
}
template <bool FIRST> __device__ __forceinline__ void blocks_mfma_at(f32x4_t& acc, i32x8_8 w, i32x8_8 a, int strip, int at, int w_powers, int a_powers) {
    switch (4 * at + strip) {                                // (a constant once unrolled)
#define CASE(A, S) case 4 * A + S: return blocks_mfma<A, S, FIRST>(acc, w, a, w_powers, a_powers)
        CASE(0, 0); CASE(0, 1); CASE(0, 2); CASE(0, 3);
        CASE(1, 0); CASE(1, 1); CASE(1, 2); CASE(1, 3);
        CASE(2, 0); CASE(2, 1); CASE(2, 2); CASE(2, 3);
        CASE(3, 0); CASE(3, 1); CASE(3, 2); CASE(3, 3);
#undef CASE
    }
}

// bfloat16; silu(gate) * up in bfloat16; float32 sums of a part of k; silu(gate) * up in 8 bits
enum { END_PLAIN = 0, END_GATED = 1, END_PARTS = 2, END_ROWS8 = 3 };

// A row of a result of any width may begin at any even address; the vector unit stores there in one instruction too.  Whole pieces at multiples of 16 go past
// the L2, others through it, where the two tiles' shares of a line meet (us, 4,806 x 5,534 x 656: 46.1, past it 49.7, value by value 79.6; 4,806 x 5,536 x 656
// past it 38.9, through it 41.7).
typedef u32x4_8 u32x4_any __attribute__((aligned(2)));
typedef u32x2_t u32x2_any __attribute__((aligned(2)));
constexpr int kStoreBytes = 8192;                            // of LDS, a wave, through which results go

// A wave's results: 16 TM tokens from m0 on by the 64 rows of w of packed block nb.  They go through the wave's own piece of LDS, a row of 64 (gated: 32)
// values for each token, and out in 16-byte pieces.
template <int TM, int END>
__device__ __forceinline__ void blocks_store(unsigned char* mine, const BlocksCall& c, f32x4_t (&acc)[TM][4], int m0, int nb, int part) {
#ifdef __HIP_DEVICE_COMPILE__
    const int lane = threadIdx.x & (kWave - 1), i16 = lane & 15, g = lane >> 4, M = c.M, n_row_blocks = (c.N + 63) / 64;
    if constexpr (END == END_PARTS) {                        // in the packed order of the rows of w, 64 n_row_blocks a token
        float* to = c.sums + (size_t)part * M * (64 * n_row_blocks) + 64 * nb + 4 * g;
#pragma unroll
        for (int tt = 0; tt < TM; ++tt) {
            const int token = m0 + i16 * TM + tt;
            float one = 1.0f;
            asm volatile("" : "+s"(one));
            if (token < M) {
#pragma unroll
                for (int rt = 0; rt < 4; ++rt) *reinterpret_cast<f32x4_t*>(to + (size_t)token * (64 * n_row_blocks) + 16 * rt) = acc[tt][rt] * one;
            }
        }
        return;
    }
    constexpr bool GATED = END == END_GATED;
    constexpr int kVals = GATED ? 32 : 64, kPieces = kVals / 8, kRowBytes = kPieces * 16, kTokens = kWave / kPieces;
    constexpr int kFit = kStoreBytes / kRowBytes / 16, kPass = TM % kFit == 0 ? kFit : 4;             // token tiles a pass
    static_assert(TM % kPass == 0, "whole passes");
    const int width = GATED ? c.N / 2 : c.N, col0 = kVals * nb;
    const bool wide = (c.ldo % 8) == 0 && (reinterpret_cast<uintptr_t>(c.out) & 15) == 0;
    float bias[4][4];
#pragma unroll
    for (int rt = 0; rt < 4; ++rt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int n = 64 * nb + 16 * rt + 4 * g + e;
            bias[rt][e] = !GATED && c.bias && n < c.N ? c.bias[n] : 0.f;
        }
    auto put = [&](int t, int value, f32x4_t y) {
        unsigned char* at = mine + t * kRowBytes + (((value / 8) ^ (t & (kPieces - 1))) * 16);
        *reinterpret_cast<uint2*>(at + (value & 4) * 2) = make_uint2(tiles_pack_bf16(y[0], y[1]), tiles_pack_bf16(y[2], y[3]));
    };
    const int piece = lane % kPieces, col = col0 + 8 * piece;
#pragma unroll
    for (int t0 = 0; t0 < TM; t0 += kPass) {
#pragma unroll
        for (int tt = t0; tt < t0 + kPass; ++tt) {
            const int t = 16 * (tt - t0) + i16;
            float one = 1.0f;                                // (hidden and made anew: the sums leave the accumulation registers here)
            asm volatile("" : "+s"(one));
            if (GATED) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    f32x4_t y = acc[tt][2 * i] * one, up = acc[tt][2 * i + 1] * one;
                    asm volatile("" : "+v"(y), "+v"(up));
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = y[e] * sigmoid8(y[e]) * up[e];
                    SB();
                    put(t, 16 * i + 4 * g, y);
                }
            } else {
#pragma unroll
                for (int rt = 0; rt < 4; ++rt) {
                    f32x4_t y = acc[tt][rt] * one;
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] += bias[rt][e];
                    put(t, 16 * rt + 4 * g, y);
                }
            }
            SB();
        }
        asm volatile("" ::: "memory");
#pragma unroll 4
        for (int it = 0; it < kPass * 16 / kTokens; ++it) {
            const int t = kTokens * it + lane / kPieces, token = m0 + (t & 15) * TM + t0 + (t >> 4);
            const u32x4_8 v = *reinterpret_cast<const u32x4_8*>(mine + t * kRowBytes + ((piece ^ (t & (kPieces - 1))) * 16));
            if (token >= M) continue;
            bf16_t* o = c.out + (size_t)token * c.ldo + col;
            if (wide && col + 8 <= width) {
                __builtin_nontemporal_store(v, reinterpret_cast<u32x4_8*>(o));
            } else if (col + 8 <= width) {
                *reinterpret_cast<u32x4_any*>(o) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (col + e < width) o[e] = (bf16_t)(v[e / 2] >> (16 * (e & 1)));
            }
        }
        asm volatile("" ::: "memory");
    }
#endif
}

// silu(gate) * up of a tile in 8 bits: its 256 rows of w are 128 columns of the result, one block of every token.  The four waves exchange each token's
// largest value through LDS, then the codes, which leave as whole lines.  (2,048 tokens of 14,336 columns: the bfloat16 result's way
// through memory and the kernel that brings it to 8 bits 207 us, this 196; 8,192 tokens 754 and 711.)
template <int TM>
__device__ __forceinline__ void blocks_store_rows8(unsigned char* lds, const BlocksCall& c, f32x4_t (&acc)[TM][4], int m0, int n_tile, int nb) {
#ifdef __HIP_DEVICE_COMPILE__
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), i16 = lane & 15, g = lane >> 4;
    uint32_t* tops = reinterpret_cast<uint32_t*>(lds);       // [4][16 TM]
    unsigned char* codes = lds + 4 * 16 * TM * 4;            // [16 TM][128], the pieces of 16 bytes swizzled
    f32x4_t y[TM][2];
#pragma unroll
    for (int tt = 0; tt < TM; ++tt) {
        float one = 1.0f;
        asm volatile("" : "+s"(one));
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f32x4_t v = acc[tt][2 * i] * one, up = acc[tt][2 * i + 1] * one;
            asm volatile("" : "+v"(v), "+v"(up));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = 64 * nb + 32 * i < c.N ? v[e] * sigmoid8(v[e]) * up[e] : 0.f;      // (columns behind the last one: 0)
                top = max(top, finite_bits(v[e]));
            }
            y[tt][i] = v;
        }
        const u32x2_t a = __builtin_amdgcn_permlane16_swap(top, top, false, false);      // over the four lanes that hold the token's columns
        top = max(a[0], a[1]);
        const u32x2_t b = __builtin_amdgcn_permlane32_swap(top, top, false, false);
        top = max(b[0], b[1]);
        if (g == 0) tops[(wave * TM + tt) * 16 + i16] = top;
        SB();
    }
    __syncthreads();
    const int b = n_tile;
#pragma unroll
    for (int tt = 0; tt < TM; ++tt) {
        uint32_t top = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) top = max(top, tops[(q * TM + tt) * 16 + i16]);
        const int power = block_power(top), token = i16 * TM + tt, t = 16 * tt + i16;
        const float inv = block_inverse(power);
#pragma unroll
        for (int i = 0; i < 2; ++i)                          // columns 32 wave + 16 i + 4 g ..
            *reinterpret_cast<uint32_t*>(codes + t * 128 + (((2 * wave + i) ^ (t & 7)) * 16) + 4 * g) =
                four_codes(y[tt][i][0] * inv, y[tt][i][1] * inv, y[tt][i][2] * inv, y[tt][i][3] * inv);
        if (wave == 0 && g == 0 && m0 + token < c.M) c.rows8_scales[(size_t)b * c.scale_stride + m0 + token] = (unsigned char)power;
    }
    __syncthreads();
    const size_t row_bytes = (size_t)((c.N / 2 + kBlock8 - 1) / kBlock8) * kBlock8;
#pragma unroll 4
    for (int it = 0; it < TM / 2; ++it) {                    // 32 tokens a round: a wave eight lines of 128 bytes
        const int t = 32 * it + (int)threadIdx.x / 8, piece = threadIdx.x & 7, token = m0 + (t & 15) * TM + (t >> 4);
        const u32x4_8 v = *reinterpret_cast<const u32x4_8*>(codes + t * 128 + ((piece ^ (t & 7)) * 16));
        if (token < c.M) *reinterpret_cast<u32x4_8*>(c.rows8 + (size_t)token * row_bytes + (size_t)b * kBlock8 + 16 * piece) = v;
    }
#endif
}

// KS: K groups of a block.  Its waves are KS groups of 4 / KS, a group takes its share of the block's stages for 256 / KS rows of w, with a ring of
// its own in LDS, and the groups' sums are added in ascending order at the end.  ONCE: w goes past the L2 (launch_tiles_end).
constexpr int kNonTemporal = 2;                              // (the bit of a load's cache policy)
template <int TM, int KS, int END, bool ONCE>
__device__ __forceinline__ void blocks_tile(unsigned char* block_lds, const BlocksCall& c, int m_tile, int n_tile, int part, int parts) {
#ifdef __HIP_DEVICE_COMPILE__
    constexpr int kBuf = TM * 16 * kStageBytes;
    constexpr int kRowWaves = kTileWaves / KS;               // waves of a group, each with 64 rows of w
    constexpr int kCopies = 2 * TM / kRowWaves;              // copies of 8 rows of activations, a wave and stage
    constexpr int kShift = kCopies < 4 ? kCopies : 4;        // copies that differ in the instruction's own offset alone
    constexpr int kLoads = 8 + kCopies + 2;                  // and 8 pieces of w and the two sides' powers
    constexpr int kUnits = TM;                               // of a stage: 16 tokens against the wave's 64 rows, four products
    constexpr int kFrags = 4, kAhead = 3, kLag = 1, kMeet = kUnits - kAhead + kLag;
    constexpr int kBefore = kLoads * kMeet / kUnits;         // loads of a stage that are asked for before the barrier ...
    constexpr int kWait = kLoads + kBefore;                  // ... and the whole stage before: what may still be on its way then
    static_assert(TM % 4 == 0 && kWait < 64, "a tile's schedule");
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int i16 = lane & 15, g = lane >> 4;
    const int row_wave = wave % kRowWaves, group = wave / kRowWaves;
    const int M = c.M, n_row_blocks = (c.N + 63) / 64;
    const size_t a_row = (size_t)c.blocks * kStageBytes;
    unsigned char* lds = block_lds + group * (kRing * kBuf);
    const unsigned as_off = i16 * TM;
    const int as_step = (int)c.scale_stride;
    int a_read[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) a_read[h] = i16 * 128 + (((4 * h + g) ^ ((i16 >> 1) & 7)) * 16);

    const int m0 = m_tile * TM * 16, nb = n_tile * kRowWaves + row_wave, nb_in = min(nb, n_row_blocks - 1);
    // the parts, and in them the groups, divide the stages evenly; all waves of a block make as many rounds as its longest group
    const int share = parts * KS, mine_at = part * KS + group;
    const int s_begin = (int)((long long)c.blocks * mine_at / share), stages = (int)((long long)c.blocks * (mine_at + 1) / share) - s_begin;
    const int longest = KS == 1 ? stages : (c.blocks + share - 1) / share;
    const unsigned char* w_base = c.wp + ((size_t)nb_in * c.blocks + s_begin) * 8192;
    asm volatile("" : "+s"(w_base));                         // (hidden: else loads move past the barriers, see tile_products)
    const __amdgpu_buffer_rsrc_t w_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)w_base, 0, 0x7fffffff, 0x00020000);
    const __amdgpu_buffer_rsrc_t a_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(c.a + (size_t)m0 * a_row - (kShift - 1) * 1024), 0, 0x7fffffff, 0x00020000);
    const __amdgpu_buffer_rsrc_t ws_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(c.w_scales + ((size_t)nb_in * c.blocks + s_begin) * 4), 0, 0x7fffffff, 0x00020000);
    // (ends with the array: the last token tile's bytes behind the last row are not read beyond it)
    const __amdgpu_buffer_rsrc_t as_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(c.a_scales + m0), 0, (int)((size_t)c.blocks * c.scale_stride - m0), 0x00020000);
    unsigned a_off[kCopies];
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {                      // LDS row `row` holds token (row & 15) TM + (row >> 4)
        const int row = 8 * (row_wave * kCopies + i) + (lane >> 3), token = (row & 15) * TM + (row >> 4);
        a_off[i] = (unsigned)min(token, M - 1 - m0) * (unsigned)a_row + 16 * ((lane & 7) ^ ((row >> 1) & 7)) + (kShift - 1 - i % kShift) * 1024;
    }

    f32x4_t acc[TM][4];
    u32x4_8 w[kRing][4][2], f[kFrags][2];
    int ap[kRing][TM / 4], wpow[kRing];
    // load l of a stage into a place of the ring.  Beyond the last stage the offset of w lies past the buffer's end: such loads bring zeros and read
    // nothing; the activations' last block is read again (times zero: a row with a NaN there is one anyway).
    struct Stage { unsigned w_off, past; int w, a, a_scales; };
    auto stage_at = [&](int stage) {
        Stage at;
        at.past = stage < stages ? 0u : 0x80000000u;
        at.w_off = lane * 16 | at.past;
        asm volatile("" : "+v"(at.w_off));                   // (one register for all pieces, which differ in the instructions' own offsets)
        const int block = min(s_begin + stage, c.blocks - 1);
        at.w = stage, at.a = block * kStageBytes, at.a_scales = block * as_step;
        return at;
    };
    auto load = [&](int slot, int l, const Stage& at) {
        if (l == 0) {
            wpow[slot] = __builtin_amdgcn_raw_buffer_load_b32(ws_rsrc, at.past, at.w * 4, 0);
        } else if (l == 1) {
            if constexpr (TM == 4) {
                ap[slot][0] = __builtin_amdgcn_raw_buffer_load_b32(as_rsrc, as_off, at.a_scales, 0);
            } else if constexpr (TM == 8) {
                const auto v = __builtin_amdgcn_raw_buffer_load_b64(as_rsrc, as_off, at.a_scales, 0);
                ap[slot][0] = v[0], ap[slot][1] = v[1];
            } else if constexpr (TM == 12) {
                const auto v = __builtin_amdgcn_raw_buffer_load_b96(as_rsrc, as_off, at.a_scales, 0);
                ap[slot][0] = v[0], ap[slot][1] = v[1], ap[slot][2] = v[2];
            } else {
                const auto v = __builtin_amdgcn_raw_buffer_load_b128(as_rsrc, as_off, at.a_scales, 0);
                ap[slot][0] = v[0], ap[slot][1] = v[1], ap[slot][2] = v[2], ap[slot][3] = v[3];
            }
        } else {
            const int k = l - 2, na = kCopies * (k + 1) / (kLoads - 2);
            if (na > kCopies * k / (kLoads - 2)) {
                switch ((na - 1) % kShift) {                 // (the offset is one of memory and of LDS)
#define CASE(I) case I: __builtin_amdgcn_raw_ptr_buffer_load_lds(a_rsrc, (__attribute__((address_space(3))) void*)(lds + slot * kBuf + (row_wave * kCopies + na - 1 - I) * 1024), \
                                                                 16, a_off[na - 1], at.a, I * 1024, 0); break
                    CASE(0); CASE(1); CASE(2); CASE(3);
#undef CASE
                }
            } else {
                const int i = k - na;
                w[slot][i & 3][i >> 2] = __builtin_amdgcn_raw_buffer_load_b128(w_rsrc, at.w_off + (i & 3) * 1024, at.w * 8192 + (i >> 2) * 4096, ONCE ? kNonTemporal : 0);
            }
        }
    };
    auto read_a = [&](int slot, int unit, int h) { f[unit % kFrags][h] = *reinterpret_cast<const u32x4_8*>(lds + slot * kBuf + a_read[h] + unit * 2048); };
    auto meet = [&]() {
        SB();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        SB();
    };
    auto stage_body = [&](auto place, int s) {
        constexpr int b = decltype(place)::value;
        const Stage next = stage_at(s + 3);
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            if (u == kMeet) {
                // this stage's fragments are all here (its buffer is the next to be written), and this wave's copies of the next stage too: loads
                // come back in the order in which they were asked for, so all but the kWait youngest are here
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                tiles_wait_loads<kWait>();
                meet();
            }
#pragma unroll
            for (int rt = 0; rt < 4; ++rt) {
                if (rt & 1) {                                // (one read or load between two products, so that none of them waits for the next's issue)
                    if (u + kAhead < kUnits) read_a(b, u + kAhead, rt / 2);
                    else if (u >= kMeet) {
#pragma unroll
                        for (int r = 0; r < kAhead; ++r)     // two a unit until they are kAhead ahead again
                            if ((r < 2 * kLag ? r / 2 : r - kLag) == u - kMeet) read_a((b + 1) & 3, r, rt / 2);
                    }
                    SB();
                }
                const i32x8_8 wv = two_pieces(w[b][rt][0], w[b][rt][1]), av = two_pieces(f[u % kFrags][0], f[u % kFrags][1]);
                if (u == 0 || rt == 0) blocks_mfma_at<true>(acc[u][rt], wv, av, rt, u % 4, wpow[b], ap[b][u / 4]);
                else blocks_mfma_at<false>(acc[u][rt], wv, av, rt, u % 4, wpow[b], ap[b][u / 4]);
                SB();
                if (rt == 1) {
#pragma unroll
                    for (int l = kLoads * u / kUnits; l < kLoads * (u + 1) / kUnits; ++l) load((b + 3) & 3, l, next);
                    SB();
                }
            }
        }
    };

#pragma unroll
    for (int tt = 0; tt < TM; ++tt)
#pragma unroll
        for (int rt = 0; rt < 4; ++rt) acc[tt][rt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        const Stage at = stage_at(p);
#pragma unroll
        for (int l = 0; l < kLoads; ++l) {
            load(p, l, at);
            SB();                                            // (in this order: the compiler's waits in the loop count what is behind a load on every way into it)
        }
    }
    tiles_wait_loads<2 * kLoads>();
    meet();
#pragma unroll
    for (int u = 0; u < kAhead; ++u) read_a(0, u, 0), read_a(0, u, 1);
    SB();
    int s = 0;
    do {                                                 // (whole rounds of the ring: the stages past the last add zeros)
        stage_body(std::integral_constant<int, 0>{}, s);
        stage_body(std::integral_constant<int, 1>{}, s + 1);
        stage_body(std::integral_constant<int, 2>{}, s + 2);
        stage_body(std::integral_constant<int, 3>{}, s + 3);
        s += 4;
    } while (s < longest);
#pragma unroll
    for (int tt = 0; tt < TM; ++tt)
#pragma unroll
        for (int rt = 0; rt < 4; ++rt) asm volatile("" : "+a"(acc[tt][rt]));      // (in accumulation registers up to here)
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");   // (the last products' results, before anything reads them)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    tiles_wait_loads<0>();                               // copies still on their way into LDS
    __syncthreads();
    if constexpr (KS > 1) {                              // (behind the first group's ring, which the epilogue uses)
        f32x4_t* sums = reinterpret_cast<f32x4_t*>(block_lds + kRing * kBuf) + row_wave * (TM * 4 * kWave) + lane;
        if (group > 0) {
#pragma unroll
            for (int tt = 0; tt < TM; ++tt)
#pragma unroll
                for (int rt = 0; rt < 4; ++rt) sums[((group - 1) * kRowWaves * TM * 4 + tt * 4 + rt) * kWave] = acc[tt][rt];
        }
        __syncthreads();
        if (group > 0) return;
#pragma unroll
        for (int tt = 0; tt < TM; ++tt)
#pragma unroll
            for (int rt = 0; rt < 4; ++rt)
#pragma unroll
                for (int q = 0; q < KS - 1; ++q) acc[tt][rt] += sums[(q * kRowWaves * TM * 4 + tt * 4 + rt) * kWave];
    }
    if constexpr (END == END_ROWS8) {
        static_assert(KS == 1, "all of a tile's columns");
        blocks_store_rows8<TM>(block_lds, c, acc, m0, n_tile, nb);
        return;
    }
    if (nb < n_row_blocks) blocks_store<TM, END>(block_lds + row_wave * kStoreBytes, c, acc, m0, nb, part);
#endif
}

// Blocks 0 .. blocks_full - 1 take tiles of 16 TM tokens over the first n_full row tiles, the blocks after them tiles of 16 TS tokens over the remaining
// ones (TS = 0: there are none).
template <int TM, int TS, int KS, int END, bool ONCE>
__global__ __launch_bounds__(kTileWaves * kWave, 1) void gemm_blocks_tiles_kernel(const BlocksCall c, int n_tiles, int n_full, int blocks_full, int parts) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char blocks_lds[];
    const bool full = TS == 0 || (int)blockIdx.x < blocks_full;
    const int b = full ? blockIdx.x : blockIdx.x - blocks_full, rows = 16 * (full ? TM : TS);          // (blocks_full is a multiple of 8)
    const int m_tiles = (c.M + rows - 1) / rows, across = full ? n_full : n_tiles - n_full;
    int m_tile, at;
    if (!tiles_place(m_tiles * across * parts, m_tiles, across * parts, b & 7, b >> 3, m_tile, at)) return;
    const int part = at / across, n_tile = (full ? 0 : n_full) + at % across;
    if (full) blocks_tile<TM, KS, END, ONCE>(blocks_lds, c, m_tile, n_tile, part, parts);
    else if constexpr (TS > 0) blocks_tile<TS, KS, END, ONCE>(blocks_lds, c, m_tile, n_tile, part, parts);
}

// out = the sum of the parts, in ascending order, with the bias or as silu(gate) * up of alternating strips.  Four values a thread.
template <bool GATED>
__global__ __launch_bounds__(256) void blocks_parts_kernel(const BlocksCall c, int parts, int fours) {
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
    const size_t m = id / fours;
    if (m >= (size_t)c.M) return;
    const int col = (int)(id - m * fours) * 4, wide = (c.N + 63) / 64 * 64, width = GATED ? c.N / 2 : c.N;
    const size_t step = (size_t)c.M * wide;
    const float* at = c.sums + m * wide + (GATED ? col / 16 * 32 + col % 16 : col);
    f32x4_t v = *reinterpret_cast<const f32x4_t*>(at), u = {0.f, 0.f, 0.f, 0.f};
    if (GATED) u = *reinterpret_cast<const f32x4_t*>(at + 16);
    for (int p = 1; p < parts; p += 3) {                     // (three parts' loads on their way at once: 128 x 512 x 16,384 in eight parts 12.9 us one by one, 12.3)
        f32x4_t y[3], z[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            if (p + i >= parts) break;
            const float* from = at + (p + i) * step;
            y[i] = *reinterpret_cast<const f32x4_t*>(from);
            if (GATED) z[i] = *reinterpret_cast<const f32x4_t*>(from + 16);
        }
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (p + i < parts) {
                v += y[i];
                if (GATED) u += z[i];
            }
    }
    bf16_t* o = c.out + m * c.ldo + col;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (GATED) v[e] = v[e] * sigmoid8(v[e]) * u[e];
        else if (c.bias && col + e < width) v[e] += c.bias[col + e];
    }
    if (col + 4 <= width) {
        *reinterpret_cast<u32x2_any*>(o) = u32x2_any{tiles_pack_bf16(v[0], v[1]), tiles_pack_bf16(v[2], v[3])};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < width) o[e] = f32_to_bf16(v[e]);
    }
}

template <int TM, int TS, int KS, int END, bool ONCE = false>
static int launch_tiles_kernel(const BlocksCall& c, int n_full, int parts, hipStream_t stream) {
    constexpr int kBlocks = kTileWaves / KS;
    const int n_tiles = ((c.N + 63) / 64 + kBlocks - 1) / kBlocks;
    if (TS == 0 || n_full > n_tiles) n_full = n_tiles;
    const long long full = ((long long)((c.M + 16 * TM - 1) / (16 * TM)) * n_full * parts + 7) / 8 * 8;
    const long long last = TS > 0 ? ((long long)((c.M + 16 * TS - 1) / (16 * (TS > 0 ? TS : 1))) * (n_tiles - n_full) * parts + 7) / 8 * 8 : 0;
    if (full + last > 1 << 26) return LLOGOS_UNSUPPORTED;
    constexpr int smem = KS * kRing * TM * 16 * kStageBytes;
    static std::atomic<uint64_t> asked{0};
    const int code = allow_dynamic_lds((const void*)gemm_blocks_tiles_kernel<TM, TS, KS, END, ONCE>, smem, asked);
    if (code != 0) return code;
    gemm_blocks_tiles_kernel<TM, TS, KS, END, ONCE><<<(unsigned)(full + last), kTileWaves * kWave, smem, stream>>>(c, n_tiles, n_full, (int)full, parts);
    return LLOGOS_LAUNCH_CHECK();
}

template <int TM, int TS, int KS>
static int launch_tiles_end(const BlocksCall& c, bool gated, int n_full, int parts, hipStream_t stream) {
    if (c.rows8 != nullptr) {
        if constexpr (KS == 1) return gated && parts == 1 ? launch_tiles_kernel<TM, TS, KS, END_ROWS8>(c, n_full, 1, stream) : LLOGOS_BAD_ARGUMENT;
        else return LLOGOS_BAD_ARGUMENT;
    }
    // w goes past the L2 where one tile covers the tokens, in four K groups where four do, if the caller says that it comes from memory: that its program reads more
    // than the 256 MB last-level cache holds before it reads w again (us: 64 x 14,336 x 4,096 gated in two groups 25.5 / past it 23.3, 61 x 4,096 x 14,336 in four groups and
    // parts 21.3 / 20.7 from memory, but 16.8 / 20.1 from that cache; a step of 64 tokens of the 8B sizes, 8.0 GB, 3,240 / 3,110, of one such layer and a small head,
    // 222 MB, 163 / 163.  Where more tiles take the same rows of w at different times they are read again: 512 x
    // 14,336 x 4,096 in two groups 94 / 102)
    const int m_tiles = (c.M + 16 * TM - 1) / (16 * TM);
    const bool once = KS > 1 && c.once && (m_tiles == 1 || (KS == 4 && m_tiles <= 4));
#define TILES(TS_, END, PARTS) (KS > 1 && once ? launch_tiles_kernel<TM, TS_, KS, END, (KS > 1)>(c, n_full, PARTS, stream) : launch_tiles_kernel<TM, TS_, KS, END>(c, n_full, PARTS, stream))
    if (parts == 1 && c.out != nullptr) return gated ? TILES(TS, END_GATED, 1) : TILES(TS, END_PLAIN, 1);
    if (TS > 0) return LLOGOS_BAD_ARGUMENT;                  // (half tiles have no parts)
    const int code = TILES(0, END_PARTS, parts);
#undef TILES
    if (code != 0 || c.out == nullptr) return code;          // (without out the caller's next kernel takes the sums)
    const int fours = ((gated ? c.N / 2 : c.N) + 3) / 4;
    const unsigned grid = (unsigned)(((size_t)c.M * fours + 255) / 256);
    if (gated) blocks_parts_kernel<true><<<grid, 256, 0, stream>>>(c, parts, fours);
    else blocks_parts_kernel<false><<<grid, 256, 0, stream>>>(c, parts, fours);
    return LLOGOS_LAUNCH_CHECK();
}

int launch_blocks_tiles(const BlocksCall& c, bool gated, int token_tiles, int groups, int n_full, int parts, hipStream_t stream) {
    // (a wave's loads count bytes from its tile's first row, its block of w, or the first byte of the tile's powers in 31 bits)
    if (c.blocks > 1 << 14 || c.scale_stride * c.blocks >= (size_t)1 << 31 || c.scale_stride % 4) return LLOGOS_UNSUPPORTED;
    if (parts < 1 || (parts > 1 && !c.sums)) return LLOGOS_BAD_ARGUMENT;
#define BT(TM, KS) if (token_tiles == TM && groups == KS) return launch_tiles_end<TM, 0, KS>(c, gated, 0, parts, stream)
    BT(4, 1);
    BT(4, 2);
    BT(4, 4);
    BT(8, 1);
    BT(8, 2);
    BT(12, 1);
    if (token_tiles == 16 && groups == 1 && n_full > 0) return launch_tiles_end<16, 8, 1>(c, gated, n_full, parts, stream);
    BT(16, 1);
#undef BT
    return LLOGOS_BAD_ARGUMENT;
}
