// Block-scaled ("microscaled") tensors: quantisation, restoration, the 4-bit product, and the two backward
// operations that read 8-bit checkpoints.  The storage form is described in program.hpp.
#include "kernels.hpp"
#include "activation.cuh"
#include "lowp.cuh"
#include "tensor_core.cuh"

#include <atomic>
#include <cstdlib>
#include <type_traits>

namespace syn {
namespace kern {

namespace {

constexpr int MX_THREADS = 256;
constexpr int MX_WARPS = MX_THREADS / 32;

// Programmatic dependent launch: a kernel launched with mx_launch_dependent may start while the one before it still runs,
// and does what does not depend on it; `wait` returns when that one has finished.  `release` in the earlier kernel lets
// the later one's blocks in as soon as there is room.  Both do nothing without such a launch.
__device__ __forceinline__ void mx_dependent_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void mx_dependent_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Storage type of a floating tensor: 0 FLOAT32, 1 BFLOAT16, 2 FLOAT16 (the KIND of lowp.cuh).
template <int KIND> struct MxElement { using type = uint16_t; };
template <> struct MxElement<0> { using type = float; };
template <int KIND> __device__ __forceinline__ float mx_load(const typename MxElement<KIND>::type *p) {
    if constexpr (KIND == 0) return *p; else return low_decode<KIND>(*p);
}
template <int KIND> __device__ __forceinline__ typename MxElement<KIND>::type mx_narrow(float x) {
    if constexpr (KIND == 0) return x; else return low_encode<KIND>(x);
}

// ------------------------------------------------------------------------------------------------
// Element-wise passes, bound by HBM.  A thread owns a group of 8 consecutive elements (16 where the quantiser reads
// 16-bit types), so 2 or 4 lanes own a block of 32: 16 or 32 bytes of the wide tensor per thread and access, the
// block's largest magnitude by one or two shuffles.  A row has `per_row` groups, counted over the padded scales (a
// multiple of 8 or 16), so a block never straddles two warps.  65536 x 4096 FLOAT32, 8 bits: quantisation 220 us (6.1 TB/s),
// restoration 240 us (5.6 TB/s), activation gradients 381 (ReLU) to 408 us (SiLU; 5.9 to 6.4 TB/s).  16-bit types are bound by their instructions:
// BFLOAT16 to 4 bits 146 us (4.7 TB/s), ReLU gradient 312 us (4.3 TB/s).
// ------------------------------------------------------------------------------------------------
// I: int64_t, or uint32_t where the groups of the whole tensor, and a step beyond them, can be counted with it.
template <typename I> struct MxRows {
    I rows, per_row, total;         // groups per row and in all
    I whole, rest;                  // whole groups of a row, columns of the one that is left
    I blocks;                       // blocks of a row that exist
    I hop, hop_rows, hop_groups;    // groups from one step of a thread to its next: in all, in whole rows, and the rest
    uint32_t code_pitch, scale_pitch;
};

inline int mx_grid(int64_t total) {
    const int64_t blocks = (total + MX_THREADS - 1) / MX_THREADS;
    return (int)(blocks < 148 * 8 ? (blocks < 1 ? 1 : blocks) : 148 * 8);
}
template <typename I> inline MxRows<I> mx_rows(int64_t rows, int64_t cols, int format, int group = 8) {
    const int64_t per_row = mx_scale_bytes(cols) * (MX_BLOCK / group), hop = (int64_t)mx_grid(rows * per_row) * MX_THREADS;
    MxRows<I> r;
    r.rows = (I)rows; r.per_row = (I)per_row; r.total = (I)(rows * per_row);
    r.whole = (I)(cols / group); r.rest = (I)(cols % group); r.blocks = (I)mx_blocks(cols);
    r.hop = (I)hop; r.hop_rows = (I)(hop / per_row); r.hop_groups = (I)(hop % per_row);
    // a single row never multiplies by its pitch
    r.code_pitch = rows > 1 ? (uint32_t)mx_code_bytes(format, cols) : 0u; r.scale_pitch = rows > 1 ? (uint32_t)mx_scale_bytes(cols) : 0u;
    return r;
}
inline bool mx_narrow_rows(int64_t rows, int64_t cols) { return rows * mx_scale_bytes(cols) * 4 < (1ll << 31); }

// The groups of a thread, `hop` apart: one division at the start, additions afterwards.  Past the last group `count` is
// 0; threads of a warp leave the loop together, since shuffles need all of them.
template <typename I> struct MxSpot {
    I g, row, group;                // the group's number, its row, its number in the row
    __device__ __forceinline__ void start(const MxRows<I> &r) {
        g = (I)blockIdx.x * MX_THREADS + threadIdx.x;
        row = r.rows == 1 ? 0 : g / r.per_row;
        group = g - row * r.per_row;
    }
    __device__ __forceinline__ void next(const MxRows<I> &r) {
        g += r.hop;
        row += r.hop_rows; group += r.hop_groups;
        if (group >= r.per_row) { group -= r.per_row; row++; }
    }
    __device__ __forceinline__ bool in(const MxRows<I> &r) const { return (g & ~(I)31) < r.total; }
    template <int E = 8> __device__ __forceinline__ int count(const MxRows<I> &r) const { return g >= r.total ? 0 : group < r.whole ? E : group == r.whole ? (int)r.rest : 0; }
    // of this group's first element in rows `pitch` elements apart
    template <int E = 8> __device__ __forceinline__ int64_t offset(int64_t pitch) const { return (int64_t)row * pitch + (int64_t)group * E; }
};

// Eight elements from memory aligned to their size (32 or 16 bytes).
template <int KIND> __device__ __forceinline__ void mx_load8(const typename MxElement<KIND>::type *p, float (&v)[8]) {
    if constexpr (KIND == 0) {
        asm volatile("ld.global.nc.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(p));
    } else {
        const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p));
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { v[2 * i] = low_decode<KIND>((uint16_t)(u[i] & 0xffffu)); v[2 * i + 1] = low_decode<KIND>((uint16_t)(u[i] >> 16)); }
    }
}
template <int KIND> __device__ __forceinline__ void mx_store8(typename MxElement<KIND>::type *p, const float (&v)[8]) {
    if constexpr (KIND == 0) {
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                     ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
    } else {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) u[i] = low_pack2<KIND>(v[2 * i], v[2 * i + 1]);
        float largest = 0.0f;           // NaN if any is
#pragma unroll
        for (int i = 0; i < 8; i++) asm("max.NaN.f32 %0, %0, %1;" : "+f"(largest) : "f"(fabsf(v[i])));
        if (largest != largest) {
#pragma unroll
            for (int i = 0; i < 4; i++) u[i] = low_canonical_nan2<KIND>(u[i]);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    }
}

// Sixteen elements of a 16-bit type from memory aligned to 32 bytes.
template <int KIND> __device__ __forceinline__ void mx_load16(const uint16_t *p, float (&v)[16]) {
    uint32_t u[8];
    asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]) : "l"(p));
#pragma unroll
    for (int i = 0; i < 8; i++) { v[2 * i] = low_decode<KIND>((uint16_t)(u[i] & 0xffffu)); v[2 * i + 1] = low_decode<KIND>((uint16_t)(u[i] >> 16)); }
}

// Rows that do not start on such an address: the warp reads (writes) its 256 elements 32 consecutive ones at a time and
// hands them over through its part of shared memory; a thread per group would touch every line eight times.
// `offset`: element offset of this lane's group, `step`: distance of consecutive columns.  Where the warp's groups
// follow one another in memory (one row, or dense rows without a gap between them) the first one's offset serves all.
// mx_gather8 only starts the loads (element i * 32 + lane of the warp's 256), mx_exchange8 hands them over, so that the
// work on one group can lie between the two of the next.
template <int KIND> __device__ __forceinline__ void mx_gather8(const typename MxElement<KIND>::type *p, int64_t offset, int64_t step, int count, int lane, float (&raw)[8]) {
    const int64_t base = __shfl_sync(0xffffffffu, offset, 0);
    if (__all_sync(0xffffffffu, offset == base + lane * 8 * step && count == 8)) {
#pragma unroll
        for (int i = 0; i < 8; i++) raw[i] = mx_load<KIND>(p + base + (i * 32 + lane) * step);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int owner = i * 4 + (lane >> 3);
            const int64_t at = __shfl_sync(0xffffffffu, offset, owner);
            const int have = __shfl_sync(0xffffffffu, count, owner);
            raw[i] = (lane & 7) < have ? mx_load<KIND>(p + at + (lane & 7) * step) : 0.0f;
        }
    }
}
__device__ __forceinline__ void mx_exchange8(const float (&raw)[8], float *box, int lane, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) box[i * 32 + lane] = raw[i];
    __syncwarp();
    const float4 a = *reinterpret_cast<const float4 *>(box + lane * 8), b = *reinterpret_cast<const float4 *>(box + lane * 8 + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    __syncwarp();
}
template <int KIND> __device__ __forceinline__ void mx_scatter8(typename MxElement<KIND>::type *p, int64_t offset, int count, float *box, int lane, const float (&v)[8]) {
    *reinterpret_cast<float4 *>(box + lane * 8) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(box + lane * 8 + 4) = make_float4(v[4], v[5], v[6], v[7]);
    __syncwarp();
    const int64_t base = __shfl_sync(0xffffffffu, offset, 0);
    if (__all_sync(0xffffffffu, offset == base + lane * 8 && count == 8)) {
#pragma unroll
        for (int i = 0; i < 8; i++) p[base + i * 32 + lane] = mx_narrow<KIND>(box[i * 32 + lane]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int owner = i * 4 + (lane >> 3);
            const int64_t at = __shfl_sync(0xffffffffu, offset, owner);
            const int have = __shfl_sync(0xffffffffu, count, owner);
            if ((lane & 7) < have) p[at + (lane & 7)] = mx_narrow<KIND>(box[i * 32 + lane]);
        }
    }
    __syncwarp();
}

// The byte of the least scale 2^(byte - 127) under which `largest` (the bit pattern of a finite magnitude) fits:
// with largest = 1.f * 2^(E - 127), 6 = 1.5 * 2^2 and 448 = 1.75 * 2^8, that is E - 2 or E - 8, one more when the
// mantissa exceeds the element type's, and at least 0.  255 for an infinity or a NaN.
template <int FORMAT> __device__ __forceinline__ uint32_t mx_scale_byte(uint32_t largest) {
    if (largest >= 0x7f800000u) return 255u;
    const int e = (int)(largest >> 23);
    const int b = FORMAT == 4 ? e - 2 + ((largest & 0x7fffffu) > 0x400000u) : e - 8 + ((largest & 0x7fffffu) > 0x600000u);
    return (uint32_t)(b < 0 ? 0 : b);
}
// 2^(byte - 127), NaN for 255.
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7fffffffu) : byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
__device__ __forceinline__ void low_unpack_half2(uint32_t h, float &a, float &b) {
    a = low_decode<2>((uint16_t)(h & 0xffffu)); b = low_decode<2>((uint16_t)(h >> 16));
}
// Two values, already under their scale, as one byte of E2M1 or two of E4M3; the first in the low part.
__device__ __forceinline__ uint32_t mx_encode4x2(float a, float b) {
    uint32_t r;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint32_t mx_encode8x2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void mx_decode4x2(uint32_t byte, float &a, float &b) {
    uint32_t h;
    asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(byte));
    low_unpack_half2(h, a, b);
}
__device__ __forceinline__ void mx_decode8x2(uint32_t bytes, float &a, float &b) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)bytes));
    low_unpack_half2(h, a, b);
}

// Scales of a 4-bit operand in the order tensor memory takes them: atoms of 512 bytes hold 128 rows x 4 blocks, row r
// of an atom at 16 (r mod 32) + 4 (r / 32); atoms of one band of rows in a row, an even number of them (a k-block of
// the product takes two).
constexpr int MX_ATOM = 512;
__host__ __device__ constexpr int64_t mx_tile_atoms(int64_t k) { return (k + 255) / 256 * 2; }
__device__ __forceinline__ int64_t mx_tile_offset(int64_t row, int64_t block, int64_t atoms) {
    return ((row >> 7) * atoms + (block >> 2)) * MX_ATOM + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}
// The same from scales that exist already: a thread moves one word of four rows.  Bytes past the last block are not
// taken over: against codes of zero a scale of NaN would still make NaN.  Launched behind the quantisation of the other
// operand it works beside it, and ends after it, so that the product only has to wait for this launch.  Quantisation,
// tiling and product so overlapped, 4096 x 4096 BFLOAT16 weights: 1024 rows 34.0 -> 28.9 us, 8192 rows 106 -> 102 us.
__global__ void __launch_bounds__(MX_THREADS) mx_tile_scales_kernel(const uint8_t *__restrict__ scales, int64_t rows, int64_t blocks, uint8_t *__restrict__ tiles) {
    mx_dependent_release();
    const int64_t words = (blocks + 3) / 4, atoms = mx_tile_atoms(blocks * MX_BLOCK), total = (rows + 127) / 128 * 32 * words;
    for (int64_t i = blockIdx.x * (int64_t)MX_THREADS + threadIdx.x; i < total; i += (int64_t)gridDim.x * MX_THREADS) {
        const int64_t line = i / words, word = i - line * words, band = line >> 5, r = band * 128 + (line & 31);
        const int left = blocks - word * 4 < 4 ? (int)(blocks - word * 4) : 4;
        const uint32_t keep = left == 4 ? 0xffffffffu : (1u << (8 * left)) - 1u;
        uint32_t v[4];
#pragma unroll
        for (int q = 0; q < 4; q++) v[q] = r + 32 * q < rows ? *reinterpret_cast<const uint32_t *>(scales + (r + 32 * q) * words * 4 + word * 4) & keep : 0u;
        *reinterpret_cast<uint4 *>(tiles + (band * atoms + word) * MX_ATOM + (line & 31) * 16) = make_uint4(v[0], v[1], v[2], v[3]);
    }
    mx_dependent_wait();
}

// x -> codes, scales.  Bound by HBM: the wide tensor once, an eighth to a half of it written.  A thread takes 32 aligned
// bytes (8 FLOAT32 or 16 16-bit elements) where rows allow, 8 elements through shared memory elsewhere.  Positions in 32
// bits where they fit: with 64-bit ones and 8 elements the 16-bit types were bound by the instructions around them.
// KEEP_NONZERO is a kernel of its own for the same reason: as a flag it cost the 16-bit types 2 %.
template <int FORMAT, int KIND, bool VEC, bool KEEP_NONZERO, typename I>
__global__ void __launch_bounds__(MX_THREADS) mx_quantize_kernel(const typename MxElement<KIND>::type *__restrict__ x, Index4 ix, MxRows<I> r, int64_t row_step, int even,
                                                                 uint8_t *__restrict__ codes, uint8_t *__restrict__ scales, uint8_t *__restrict__ tiles, uint32_t atoms) {
    constexpr int E = VEC && KIND != 0 ? 16 : 8, LANES = MX_BLOCK / E;      // lanes per block
    __shared__ float boxes[VEC ? 1 : MX_WARPS][VEC ? 1 : 256];
    const int lane = threadIdx.x & 31;
    mx_dependent_release();             // the product that reads the codes
    MxSpot<I> at;
    auto fetch = [&](float (&v)[E]) {
        const int count = at.template count<E>(r);
        if constexpr (VEC) {
            const auto *p = x + at.template offset<E>(row_step);
            if (count == E) {
                if constexpr (E == 16) mx_load16<KIND>(p, v); else mx_load8<KIND>(p, v);
            } else {
#pragma unroll
                for (int i = 0; i < E; i++) v[i] = i < count ? mx_load<KIND>(p + i) : 0.0f;
            }
        } else {
            int64_t base = (int64_t)at.row * row_step;
            if (!even) {
                const int64_t row = count ? (int64_t)at.row : 0, r2 = row % ix.shape[2], rest = row / ix.shape[2];
                base = r2 * ix.sa[2] + rest % ix.shape[1] * ix.sa[1] + rest / ix.shape[1] * ix.sa[0];
            }
            mx_gather8<KIND>(x, base + (int64_t)at.group * 8 * ix.sa[3], ix.sa[3], count, lane, v);
        }
    };
    float ahead[E];
    at.start(r);
    if (at.in(r)) fetch(ahead);
    while (at.in(r)) {
        float v[E];
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < E; i++) v[i] = ahead[i];
        } else mx_exchange8(ahead, boxes[threadIdx.x >> 5], lane, v);
        const I row = at.row, group = at.group;
        const bool mine = at.g < r.total;
        at.next(r);
        if (at.in(r)) fetch(ahead);         // in flight while this group is worked on
        float most = 0.0f;                  // NaN if any is
#pragma unroll
        for (int i = 0; i < E; i++) asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(fabsf(v[i])));
        uint32_t largest = __float_as_uint(most);       // bit patterns of magnitudes order like the magnitudes, NaN above infinity
#pragma unroll
        for (int d = 1; d < LANES; d *= 2) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, d));
        if (!mine) continue;
        const I block = group / LANES;
        const bool exists = block < r.blocks;       // else: padding of the scales
        const uint32_t byte = exists ? mx_scale_byte<FORMAT>(largest) : 0u;
        if (lane % LANES == 0) {
            scales[(int64_t)row * r.scale_pitch + block] = (uint8_t)byte;
            if (tiles) tiles[mx_tile_offset(row, block, atoms)] = (uint8_t)byte;
        }
        if (!exists) continue;
        if (byte == 255u) {
#pragma unroll
            for (int i = 0; i < E; i++) v[i] = 0.0f;
        }
        if constexpr (KEEP_NONZERO) {
            const float least = (FORMAT == 4 ? 0.5f : 0.001953125f) * mx_scale_value(byte);     // the smallest element, 2^-136 or more: exact; no block of NaN is below it
#pragma unroll
            for (int i = 0; i < E; i++) v[i] = v[i] != 0.0f && fabsf(v[i]) < least ? copysignf(least, v[i]) : v[i];
        }
        // the inverse scale 2^(127 - byte) is a normal number for every other byte that occurs; a product with it is
        // exact, or below half the smallest element
        const float inverse = byte == 255u ? 0.0f : __uint_as_float((254u - byte) << 23);
#pragma unroll
        for (int i = 0; i < E; i++) v[i] *= inverse;
        uint32_t words[E * FORMAT / 32];
#pragma unroll
        for (int w = 0; w < E * FORMAT / 32; w++) {
            if constexpr (FORMAT == 4) words[w] = mx_encode4x2(v[8 * w], v[8 * w + 1]) | mx_encode4x2(v[8 * w + 2], v[8 * w + 3]) << 8 | mx_encode4x2(v[8 * w + 4], v[8 * w + 5]) << 16 | mx_encode4x2(v[8 * w + 6], v[8 * w + 7]) << 24;
            else words[w] = mx_encode8x2(v[4 * w], v[4 * w + 1]) | mx_encode8x2(v[4 * w + 2], v[4 * w + 3]) << 16;
        }
        uint8_t *dst = codes + (int64_t)row * r.code_pitch + (int64_t)group * (E * FORMAT / 8);
        if constexpr (E * FORMAT == 32) *reinterpret_cast<uint32_t *>(dst) = words[0];
        else if constexpr (E * FORMAT == 64) *reinterpret_cast<uint2 *>(dst) = make_uint2(words[0], words[1]);
        else *reinterpret_cast<uint4 *>(dst) = make_uint4(words[0], words[1], words[2], words[3]);
    }
}

// The eight values of a group; the caller has checked that its block exists.
template <int FORMAT> struct MxHeld { uint32_t w[FORMAT / 4]; uint32_t byte; };
template <int FORMAT, typename I> __device__ __forceinline__ void mx_fetch_held(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, const MxRows<I> &r,
                                                                                const MxSpot<I> &at, MxHeld<FORMAT> &h) {
    h.byte = __ldg(scales + (int64_t)at.row * r.scale_pitch + (at.group >> 2));
    const uint8_t *src = codes + (int64_t)at.row * r.code_pitch + (int64_t)at.group * FORMAT;
    if constexpr (FORMAT == 4) h.w[0] = __ldg(reinterpret_cast<const uint32_t *>(src));
    else { const uint2 w = __ldg(reinterpret_cast<const uint2 *>(src)); h.w[0] = w.x; h.w[1] = w.y; }
}
template <int FORMAT> __device__ __forceinline__ void mx_values8(const MxHeld<FORMAT> &h, float (&v)[8]) {
    const float scale = mx_scale_value(h.byte);
    if constexpr (FORMAT == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) mx_decode4x2(h.w[0] >> (8 * i) & 0xffu, v[2 * i], v[2 * i + 1]);
    } else {
        mx_decode8x2(h.w[0] & 0xffffu, v[0], v[1]); mx_decode8x2(h.w[0] >> 16, v[2], v[3]);
        mx_decode8x2(h.w[1] & 0xffffu, v[4], v[5]); mx_decode8x2(h.w[1] >> 16, v[6], v[7]);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] *= scale;
}

template <int FORMAT, int KIND, bool VEC, typename I>
__global__ void __launch_bounds__(MX_THREADS) mx_restore_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, MxRows<I> r, int64_t cols,
                                                                typename MxElement<KIND>::type *__restrict__ out) {
    __shared__ float boxes[VEC ? 1 : MX_WARPS][VEC ? 1 : 256];
    MxSpot<I> at;
    MxHeld<FORMAT> ahead = {};
    at.start(r);
    if (at.count(r)) mx_fetch_held<FORMAT>(codes, scales, r, at, ahead);
    while (at.in(r)) {
        const MxHeld<FORMAT> held = ahead;
        const int count = at.count(r);
        const int64_t offset = at.offset(cols);
        at.next(r);
        if (at.count(r)) mx_fetch_held<FORMAT>(codes, scales, r, at, ahead);
        float v[8];
        mx_values8<FORMAT>(held, v);
        if constexpr (VEC) { if (count) mx_store8<KIND>(out + offset, v); }      // rows are whole groups here
        else mx_scatter8<KIND>(out, offset, count, boxes[threadIdx.x >> 5], threadIdx.x & 31, v);
    }
}

// exp(-x) for x >= 0, within 4 + 2.35 x units of 2^-24 of itself (the documented bound of the intrinsic), which is less
// than 6 units of 1 everywhere.
__device__ __forceinline__ float mx_exp_minus(float x) { return __expf(-x); }

// act'(z) in FLOAT32.  exp(-|z|) keeps every form free of overflow and of cancellation against 1.  Beyond 120 the
// exponentials are below the smallest number and the slope is 0 or 1, so z (an infinity too, which a scale near the end
// of its range can make of a finite value) is brought to that range first; NaN stays NaN.  Over every value that 8 bits can
// hold the slopes are within 4 units of 2^-24 of 1 and, but for GELU's next to their zero, within 2^-18 of themselves; the framework's
// activations evaluate in binary64, which here would bind the pass to its instructions rather than to HBM.
template <Op ACT> __device__ __forceinline__ float mx_slope(float z) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(-120.0f));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(120.0f));
    if constexpr (ACT == Op::TANH) {
        const float e = mx_exp_minus(2.0f * fabsf(z)), d = 1.0f + e;
        return __fdividef(4.0f * e, d * d);
    } else if constexpr (ACT == Op::SIGMOID) {
        const float e = mx_exp_minus(fabsf(z)), d = 1.0f + e;
        return __fdividef(e, d * d);
    } else if constexpr (ACT == Op::SILU) {
        const float e = mx_exp_minus(fabsf(z)), near = __fdividef(1.0f, 1.0f + e), far = e * near;
        const float s = z >= 0.0f ? near : far, t = z >= 0.0f ? far : near;      // sigmoid(z) and 1 - sigmoid(z)
        return s * fmaf(z, t, 1.0f);
    } else if constexpr (ACT == Op::GELU_TANH) {    // z sigmoid(2u), u = sqrt(2 / pi) (z + 0.044715 z^3)
        const float c = 1.5957691216057308f, zz = z * z;
        const float u = c * z * fmaf(0.044715f, zz, 1.0f);
        const float e = mx_exp_minus(fabsf(u)), near = __fdividef(1.0f, 1.0f + e), far = e * near;
        return fmaf(z * (near * far), c * fmaf(0.134145f, zz, 1.0f), u >= 0.0f ? near : far);
    } else {                                        // GELU: Phi(z) + z phi(z)
        // Phi(-|z|) = exp(-z^2 / 2) t p(t), t = 1 / (1 + 0.305 |z|): p of degree 7 fitted for the least relative error on
        // 0 <= |z| <= 13.5, where the exponential leaves the normal numbers (2^-23.3; 6 units of 2^-24 with FLOAT32 arithmetic),
        // so the tail is as exact as its exponential, which it shares with the density
        const float e = mx_exp_minus(0.5f * z * z), t = __fdividef(1.0f, fmaf(0.305f, fabsf(z), 1.0f));
        float p = fmaf(t, 0.0366990678f, -0.152987808f);
        p = fmaf(t, p, 0.185716048f); p = fmaf(t, p, -0.0379760452f); p = fmaf(t, p, 0.121021271f);
        p = fmaf(t, p, 0.103420988f); p = fmaf(t, p, 0.122466795f); p = fmaf(t, p, 0.121639736f);
        const float tail = e * (t * p);
        return fmaf(0.3989422804014327f * z, e, z >= 0.0f ? 1.0f - tail : tail);
    }
}
template <Op ACT> __device__ __forceinline__ void mx_slopes(float (&z)[8], const float (&up)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (ACT == Op::RELU) z[i] = z[i] > 0.0f ? up[i] : z[i] != z[i] ? z[i] : 0.0f;
        else z[i] = up[i] * mx_slope<ACT>(z[i]);
    }
}

// dz = g * act'(z).  A closed ReLU gate gives 0 whatever g holds, like the WHERE of the ordinary gradient rule; a
// block of NaN gives NaN, so that a step over it is refused rather than taken without its gradient.
template <int KIND, bool VEC, typename I>
__global__ void __launch_bounds__(MX_THREADS) mx_activation_gradient_kernel(int act, const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                                                                            const typename MxElement<KIND>::type *__restrict__ g_in, MxRows<I> r, int64_t cols,
                                                                            typename MxElement<KIND>::type *__restrict__ out) {
    __shared__ float boxes[VEC ? 1 : MX_WARPS][VEC ? 1 : 256];
    const int lane = threadIdx.x & 31;
    MxSpot<I> at;
    MxHeld<8> held_ahead = {};
    float up_ahead[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    auto fetch = [&]() {
        const int count = at.count(r);
        if (count) mx_fetch_held<8>(codes, scales, r, at, held_ahead);
        if constexpr (VEC) { if (count) mx_load8<KIND>(g_in + at.offset(cols), up_ahead); }
        else mx_gather8<KIND>(g_in, at.offset(cols), 1, count, lane, up_ahead);
    };
    at.start(r);
    if (at.in(r)) fetch();
    while (at.in(r)) {
        const MxHeld<8> held = held_ahead;
        float up[8], z[8];
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < 8; i++) up[i] = up_ahead[i];
        } else mx_exchange8(up_ahead, boxes[threadIdx.x >> 5], lane, up);
        const int count = at.count(r);
        const int64_t offset = at.offset(cols);
        at.next(r);
        if (at.in(r)) fetch();
        mx_values8<8>(held, z);
        switch ((Op)act) {
            case Op::RELU: mx_slopes<Op::RELU>(z, up); break;
            case Op::TANH: mx_slopes<Op::TANH>(z, up); break;
            case Op::SIGMOID: mx_slopes<Op::SIGMOID>(z, up); break;
            case Op::SILU: mx_slopes<Op::SILU>(z, up); break;
            case Op::GELU_TANH: mx_slopes<Op::GELU_TANH>(z, up); break;
            default: mx_slopes<Op::GELU>(z, up); break;
        }
        if constexpr (VEC) { if (count) mx_store8<KIND>(out + offset, z); }
        else mx_scatter8<KIND>(out, offset, count, boxes[threadIdx.x >> 5], lane, z);
    }
}

// Activations of a FLOAT32 sum before its one rounding, from exp(-|z|) like the slopes above; below -120 SILU and
// both GELUs are below the smallest number (-0, also for -infinity).
__device__ __forceinline__ float mx_activate(int act, float z) {
    switch ((Op)act) {
        case Op::RELU: return relu_value(z);
        case Op::TANH: return tanhf(z);
        case Op::SIGMOID: { const float e = expf(-fabsf(z)), near = __fdividef(1.0f, 1.0f + e); return z >= 0.0f ? near : e * near; }
        case Op::SILU: case Op::GELU_TANH: {
            if (z < -120.0f) return -0.0f;
            if (z > 120.0f) return z;
            const float u = act == (int)Op::SILU ? z : 1.5957691216057308f * z * fmaf(0.044715f * z, z, 1.0f);
            const float e = expf(-fabsf(u)), near = __fdividef(1.0f, 1.0f + e);
            return z * (u >= 0.0f ? near : e * near);
        }
        case Op::GELU: return z < -120.0f ? -0.0f : 0.5f * z * erfcf(-0.7071067811865476f * z);
        default: return z;
    }
}
__device__ __noinline__ float4 mx_activate4(int act, float4 z) {
    return make_float4(mx_activate(act, z.x), mx_activate(act, z.y), mx_activate(act, z.z), mx_activate(act, z.w));
}

// ------------------------------------------------------------------------------------------------
// 4-bit products on the tensor cores: tcgen05.mma kind::mxf4 multiplies E2M1 codes under one E8M0 scale per 32
// contraction steps, exactly, and adds in FP32 in tensor memory.  Codes go from the tensors to shared memory by TMA
// (a k-block is 256 elements = one 128-byte swizzle row); their scales have to lie in tensor memory in the
// order [lane = row mod 32][column = row / 32], four contraction blocks per 32-bit word.
// ------------------------------------------------------------------------------------------------
constexpr int MX_BK = 256;                      // contraction steps per k-block
// k-blocks per partial sum in tensor memory, by the type of the result: 64 MMAs for FLOAT32, 256 for 16 bits.  Tensor
// memory adds with truncation: two-SM sums of positive terms fell short by 0.1 units of 2^-23 per MMA and more as they grow (6 units
// after 64 MMAs, 2600 after 16384).  Longer contractions add their partial sums in FP32 registers (8 units), each
// at the price of a stop of the MMAs: 8192 x 16384 x 4096 in FLOAT32 takes 6 % longer than with one sum (237 against 224 us).
template <int KIND> constexpr int mx_chunk() { return KIND == 0 ? 16 : 64; }

// Instruction descriptor of kind::mxf4: E2M1 x E2M1 (format 1), UE8M0 scales (bit 23), K-major, M rows, N columns;
// sf: which two of the four scale bytes per word the 64 contraction steps use (0 or 2).
__device__ __forceinline__ uint32_t mx_idesc(int rows, int cols, int sf) {
    return ((uint32_t)sf << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(cols >> 3) << 17) | (1u << 23) | ((uint32_t)(rows >> 4) << 24) | ((uint32_t)sf << 29);
}
__device__ __forceinline__ uint64_t mx_operand_desc(uint32_t smem_addr) {       // K-major, 128-byte swizzle
    return (1ull << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61) | (uint64_t)((smem_addr & 0x3ffffu) >> 4);
}
__device__ __forceinline__ uint64_t mx_scale_desc(uint32_t smem_addr) {         // 32 rows of 16 bytes, 8-row groups 128 bytes apart
    return ((uint64_t)(128u >> 4) << 32) | (1ull << 46) | (uint64_t)((smem_addr & 0x3ffffu) >> 4);
}
template <int PAIR> __device__ __forceinline__ void mx_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t scale_a, uint32_t scale_b, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\ttcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\ttcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mx_copy_atom(uint32_t taddr, uint32_t smem_addr) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(mx_scale_desc(smem_addr)) : "memory");
}
// Four bytes global -> shared, the part past `bytes` (0 to 4) zero.
__device__ __forceinline__ void mx_copy_word(uint32_t dst, const uint8_t *src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// The scale words of `count` rows from row0 for the k-block that starts at contraction block b0, `threads` threads in
// turn.  dst: atoms [contraction half][row / 128].
__device__ __forceinline__ void mx_copy_scales(uint32_t dst, int atoms, const uint8_t *scales, int64_t pitch, int rows, int blocks, int row0, int count, int b0, int thread, int threads) {
    for (int i = thread; i < 2 * count; i += threads) {
        const int half = i & 1, r = i >> 1, b = b0 + half * 4;
        const int left = blocks - b;
        const int bytes = row0 + r < rows ? (left >= 4 ? 4 : left > 0 ? left : 0) : 0;
        const uint8_t *src = bytes ? scales + (int64_t)(row0 + r) * pitch + b : scales;
        mx_copy_word(dst + (uint32_t)((half * atoms + (r >> 7)) * MX_ATOM + (r & 31) * 16 + ((r >> 5) & 3) * 4), src, bytes);
    }
}

// Arrival on a barrier of the cluster's block `rank`.  Default (block) scope: what the arrival announces lies in this
// block's own shared or tensor memory and has been made visible to the tensor core by a proxy or tcgen05 fence; a
// release at cluster scope waits for every access of the thread, which cost more than a stage's work.
__device__ __forceinline__ void mx_arrive_rank(uint32_t bar, uint32_t rank) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(map_to_rank(bar, rank)) : "memory");
}
// Waits, for at most a tenth of a second and whatever the abort flag says, for copies whose barrier nothing else arrives on.
__device__ __forceinline__ void mx_wait_landed(uint32_t bar, uint32_t parity) {
    const uint64_t start = global_timer();
    while (!mbar_try_wait(bar, parity) && global_timer() - start < 100000000ull) { }
}

// 24 columns of tensor memory, this warp's 32 lanes.
__device__ __forceinline__ void tmem_store24(uint32_t taddr, const uint4 (&v)[6]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(v[0].x), "r"(v[0].y), "r"(v[0].z), "r"(v[0].w), "r"(v[1].x), "r"(v[1].y), "r"(v[1].z), "r"(v[1].w),
                   "r"(v[2].x), "r"(v[2].y), "r"(v[2].z), "r"(v[2].w), "r"(v[3].x), "r"(v[3].y), "r"(v[3].z), "r"(v[3].w) : "memory");
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(taddr + 16u), "r"(v[4].x), "r"(v[4].y), "r"(v[4].z), "r"(v[4].w), "r"(v[5].x), "r"(v[5].y), "r"(v[5].z), "r"(v[5].w) : "memory");
}

// One lane waits for the warp: 32 lanes that poll a barrier take issue slots from the rest of the block.
__device__ __forceinline__ bool mx_warp_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int lane) {
    if (lane == 0) mbar_wait_cluster(bar, parity, abort_flag);
    __syncwarp();
    return *abort_flag == 0;
}

struct MxLinear {
    int m, n, blocks, k_blocks;         // blocks: contraction blocks of 32; k_blocks: of 256
    int64_t scale_pitch;
    const uint8_t *xs, *ws;
    const void *bias; void *out;
    int act;
    int tiles_m, tiles_n, group_n;
    int staged;                         // rows of `out` can be written by TMA
    int after_x;                        // the launch before this one is the quantisation of x
    int *error_word;
};

// ---- few rows: weights on the M side ----------------------------------------------------------------
// One block multiplies 128 rows of W by BN rows of x over a slice of the contraction; the up to eight blocks of a
// cluster share a tile and add their partial sums, in ascending order, through each other's shared memory.  With
// W as the M operand a tile wastes no MMA rows on absent rows of x, and the result leaves with 32 consecutive
// columns per warp without a transposition.  Bound by latency: one row of 4096 against 4096 x 4096 takes 12.7 to 15.3 us per call
// with its quantisation, 11 of them on the host.  Two warps fetch the scales word by word, with 4-byte asynchronous
// copies, into the order of tensor memory; the issuing thread sends them there with tcgen05.cp in front of the MMAs.
template <int BN> struct MxFewConfig {
    static constexpr int kStages = BN <= 64 ? 6 : 5;
    static constexpr int kABytes = 128 * 128, kBBytes = BN * 128;
    static constexpr int kScaleBytes = 4 * MX_ATOM;             // two halves of W's atom, two of x's
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kScaleCols = 16;                       // tensor-memory columns of one stage's scales
    static constexpr int kTmemCols = BN + kStages * kScaleCols <= 128 ? 128 : 256;
    static constexpr int kSmemBytes = kStages * (kStageBytes + kScaleBytes) + 1024 + 256;
    static_assert(BN * 128 * 4 <= kStages * kStageBytes, "partial sums reuse the operand stages");
};

template <int BN, int KIND>
__global__ void __launch_bounds__(256, 1) mx_linear_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, MxLinear prm, int slices) {
    using Cfg = MxFewConfig<BN>;
    using T = typename MxElement<KIND>::type;
    constexpr int S = Cfg::kStages, CHUNK = mx_chunk<KIND>();
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S * (Cfg::kStageBytes + Cfg::kScaleBytes));
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 3 * S + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t bar_base = smem_u32(bars), smem_base = smem_u32(smem), scale_base = smem_base + S * Cfg::kStageBytes;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (S + s); };
    auto scale_bar = [&](int s) { return bar_base + 8u * (2 * S + s); };
    const uint32_t done_bar = bar_base + 8u * (3 * S), drained_bar = bar_base + 8u * (3 * S + 1);     // of a partial sum

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; s++) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); mbar_init(scale_bar(s), 2); }
        mbar_init(done_bar, 1); mbar_init(drained_bar, 4);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)Cfg::kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    // a cluster of `slices` blocks per tile; neighbouring clusters share the rows of x
    const int slice = (int)(blockIdx.x % slices), tile = (int)(blockIdx.x / slices);
    const int n0 = tile % prm.tiles_n * 128, m0 = tile / prm.tiles_n * BN;
    const int kb0 = (int)((int64_t)prm.k_blocks * slice / slices), kb1 = (int)((int64_t)prm.k_blocks * (slice + 1) / slices);

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0; uint32_t phase = 0;
            int armed = 0;
            bool ok = true;
            // W does not depend on the launch before this one: its first stages are on their way before x is waited for
            const int early = kb1 - kb0 < S ? kb1 - kb0 : S;
            for (int i = 0; i < early; i++) {
                mbar_expect_tx(full_bar(i), Cfg::kStageBytes);
                tma_load_2d(smem_base + i * Cfg::kStageBytes, &map_w, full_bar(i), (kb0 + i) * (MX_BK / 2), n0);
            }
            mx_dependent_wait();
            for (int kb = kb0; kb < kb1; kb++) {
                const uint32_t sa = smem_base + stage * Cfg::kStageBytes;
                if (kb - kb0 >= early) {
                    if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag)) { ok = false; break; }
                    mbar_expect_tx(full_bar(stage), Cfg::kStageBytes);
                    tma_load_2d(sa, &map_w, full_bar(stage), kb * (MX_BK / 2), n0);
                }
                tma_load_2d(sa + Cfg::kABytes, &map_x, full_bar(stage), kb * (MX_BK / 2), m0);
                armed++;
                if (++stage == S) { stage = 0; phase ^= 1u; }
            }
            // giving up: the copies in flight land before the block leaves
            if (!ok || *abort_flag) for (int i = armed > S ? armed - S : 0; i < armed; i++) mx_wait_landed(full_bar(i % S), (uint32_t)(i / S) & 1u);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int stage = 0; uint32_t phase = 0;
            const uint32_t id0 = mx_idesc(128, BN, 0), id2 = mx_idesc(128, BN, 2);
            bool ok = true;
            for (int kb = kb0; kb < kb1; kb++) {
                const int in_chunk = (kb - kb0) % CHUNK, chunk = (kb - kb0) / CHUNK;
                if (in_chunk == 0 && chunk > 0) {
                    umma_commit(done_bar);
                    if (!mbar_wait(drained_bar, (uint32_t)(chunk - 1) & 1u, abort_flag)) { ok = false; break; }
                }
                if (!mbar_wait(full_bar(stage), phase, abort_flag) || !mbar_wait(scale_bar(stage), phase, abort_flag)) { ok = false; break; }
                tc_fence_after();
                const uint32_t pa = smem_base + stage * Cfg::kStageBytes, pb = pa + Cfg::kABytes, ps = scale_base + stage * Cfg::kScaleBytes;
                const uint32_t ts = tmem_base + BN + (uint32_t)(stage * Cfg::kScaleCols);
#pragma unroll
                for (int i = 0; i < 4; i++) mx_copy_atom(ts + i * 4, ps + i * MX_ATOM);
#pragma unroll
                for (int k4 = 0; k4 < 4; k4++)
                    mx_mma<0>(tmem_base, mx_operand_desc(pa + k4 * 32), mx_operand_desc(pb + k4 * 32), (k4 & 1) ? id2 : id0, ts + (k4 >> 1) * 4, ts + 8 + (k4 >> 1) * 4,
                              (in_chunk != 0 || k4 != 0) ? 1u : 0u);
                umma_commit(empty_bar(stage));
                if (++stage == S) { stage = 0; phase ^= 1u; }
            }
            if (ok) umma_commit(done_bar);
        }
    } else if (warp < 4) {
        // scales: copies of up to three stages in flight per thread
        const int thread = threadIdx.x - 64;
        int stage = 0; uint32_t phase = 0;
        bool ok = true;
        mx_dependent_wait();
        auto arrive = [&](int kb) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(scale_bar((kb - kb0) % S));
        };
        for (int kb = kb0; kb < kb1; kb++) {
            ok = __all_sync(0xffffffffu, mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag));
            if (!ok) break;
            const uint32_t ps = scale_base + stage * Cfg::kScaleBytes;
            mx_copy_scales(ps, 1, prm.ws, prm.scale_pitch, prm.n, prm.blocks, n0, 128, kb * 8, thread, 64);
            mx_copy_scales(ps + 2 * MX_ATOM, 1, prm.xs, prm.scale_pitch, prm.m, prm.blocks, m0, BN < 128 ? BN : 128, kb * 8, thread, 64);
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (kb - kb0 >= 2) { asm volatile("cp.async.wait_group 2;" ::: "memory"); arrive(kb - 2); }
            if (++stage == S) { stage = 0; phase ^= 1u; }
        }
        if (ok && kb1 - kb0 >= 2) { asm volatile("cp.async.wait_group 1;" ::: "memory"); arrive(kb1 - 2); }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (ok && kb1 > kb0) arrive(kb1 - 1);
    }
    __syncwarp();
    bool ok = true;
    float *partial = reinterpret_cast<float *>(smem);       // [BN][128]
    if (warp >= 4) {
        const int row = (warp & 3) * 32 + lane;             // of W's tile
        const uint32_t taddr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
        float sum[BN];
#pragma unroll
        for (int i = 0; i < BN; i++) sum[i] = -0.0f;        // what adds up to the first partial sum as it is
        for (int kb = kb0; kb < kb1; kb += CHUNK) {
            ok = __all_sync(0xffffffffu, mbar_wait(done_bar, (uint32_t)((kb - kb0) / CHUNK) & 1u, abort_flag));
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < BN / 16; c++) {
                float t[16];
                tmem_load16(taddr + (uint32_t)(c * 16), t);
#pragma unroll
                for (int i = 0; i < 16; i++) sum[c * 16 + i] = __fadd_rn(sum[c * 16 + i], t[i]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(drained_bar);
        }
#pragma unroll
        for (int i = 0; i < BN; i++) partial[i * 128 + row] = sum[i];
    }
    tc_fence_before();
    if (slices > 1) cluster_sync_all(); else __syncthreads();
    // every block finishes its share of the tile's rows of x; two rows at a time, 128 threads each
    const int per = (BN + slices - 1) / slices;
    const int col = n0 + (int)(threadIdx.x & 127);
    const int first = slice * per, last = first + per < BN ? first + per : BN;
    const uint32_t mine = smem_u32(partial) + (threadIdx.x & 127) * 4;
    const float b = prm.bias && col < prm.n ? mx_load<KIND>((const T *)prm.bias + col) : 0.0f;
    for (int r = first + (int)(threadIdx.x >> 7); r < last; r += 2) {
        if (m0 + r >= prm.m) break;
        float sum;
        if (slices == 1) sum = partial[r * 128 + (threadIdx.x & 127)];
        else {
            float v[8];         // all on their way before the first is added
#pragma unroll
            for (int q = 0; q < 8; q++)
                if (q < slices) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[q]) : "r"(map_to_rank(mine + (uint32_t)r * 512u, (uint32_t)q)));
            sum = v[0];
#pragma unroll
            for (int q = 1; q < 8; q++) if (q < slices) sum = __fadd_rn(sum, v[q]);
        }
        if (col < prm.n) ((T *)prm.out)[(int64_t)(m0 + r) * prm.n + col] = mx_narrow<KIND>(mx_activate(prm.act, prm.bias ? __fadd_rn(sum, b) : sum));
    }
    if (slices > 1) cluster_sync_all(); else __syncthreads();      // no block leaves while another reads its sums
    if (threadIdx.x == 0 && *abort_flag) atomicOr(prm.error_word, ERR_WAIT_TIMEOUT);
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)Cfg::kTmemCols) : "memory");
    }
}

// ---- many rows: two-SM tiles of 256 x 256 -----------------------------------------------------------
// A cluster of two blocks per tile (cta_group::2, M = 256): each loads its 128 rows of x, half of the tile's 256
// rows of W; the scales of its rows of x and of all of W's go into its tensor memory.  A one-SM block would move
// (128 + 256) x 128 bytes of codes into shared memory and the tensor core read them out again within 512 clocks of
// MMA, more than shared memory delivers; the pair moves a third less.  Accumulators take 256 columns of tensor memory
// and the scales of the stages in flight most of the rest, so there is one accumulator: the epilogue warps first copy
// it to registers, hand it back, and finish the tile under the next one's main loop.  37888 x 4096 x 4096: 297 us
// in a burst (4.3 PFLOP/s), 338 us in a row under the power cap (1.64 GHz); an earlier build's MMAs alone, without any load, took 232.
// Scales: TMA fetches their tiles into a ring of their own, further ahead than the codes, and four warps move them on
// to tensor memory through registers as soon as a stage's columns are free, so they lie there before the codes land.
// tcgen05.cp from shared memory shares the tensor pipe with the MMAs: its six copies per k-block cost 60 of 334 us on
// 37888 x 4096 x 4096.  Gathering the words from rows instead of tiles cost three times the main loop.
struct MxPairConfig {
    static constexpr int BN = 256;
    static constexpr int kStages = 5;
    static constexpr int kABytes = 128 * 128, kBBytes = 128 * 128;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kScaleBytes = 6 * MX_ATOM;             // two atoms of x's rows, two of each half of W's
    static constexpr int kScaleSlots = 8;
    static constexpr int kScaleCols = 24;                       // of a stage: two atoms of x, two of each half of W
    static constexpr int kTmemCols = 512;
    static constexpr int kStagingBytes = 8 * 4096;
    static constexpr int kSmemBytes = kStages * kStageBytes + kScaleSlots * kScaleBytes + kStagingBytes + 1024 + 512;
};
constexpr int MX_PAIR_THREADS = 512;    // warp 0 TMA of codes, warp 1 MMA, warp 2 TMA of scales, warps 4-7 scales, warps 8-15 epilogue
// Registers per thread of the three groups after the split; their sum over the four warpgroups is at most the 512 of
// the launch.
constexpr int MX_PAIR_REGS_LOW = 40, MX_PAIR_REGS_SCALES = 64, MX_PAIR_REGS_EPILOGUE = 200;

// One warp's 32 rows x 128 columns: bias, activation, one rounding, then boxes of 32 rows x 128 bytes through
// shared memory (16-byte chunk j of row r at chunk j ^ (r & 7), the 128-byte swizzle) and out by TMA, which clips the
// edges; rows of `out` that TMA cannot address are copied from the box 32 columns at a time.
template <int KIND, bool GENERAL>
__device__ __forceinline__ void mx_emit(const MxLinear &prm, const CUtensorMap *map_out, uint32_t stage, int row0, int col0, float (&sum)[128], float4 bias_lane, int lane) {
    using T = typename MxElement<KIND>::type;
    constexpr int WIDTH = KIND == 0 ? 32 : 64;          // columns per box
    constexpr int PER = WIDTH / 8;                      // columns per 16-byte chunk
#pragma unroll
    for (int b = 0; b < 128 / WIDTH; b++) {
        const int c0 = col0 + b * WIDTH;
        if (c0 >= prm.n || row0 >= prm.m) break;        // warp-uniform
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // the previous box has been read
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; j++) {
            uint32_t words[4];
#pragma unroll
            for (int q = 0; q < PER / 4; q++) {
                float *v = &sum[b * WIDTH + j * PER + q * 4];
                const int src = (b * WIDTH + j * PER) / 4 + q;
                float z[4] = {v[0], v[1], v[2], v[3]};
                if (prm.bias) {
                    z[0] = __fadd_rn(z[0], __shfl_sync(0xffffffffu, bias_lane.x, src));
                    z[1] = __fadd_rn(z[1], __shfl_sync(0xffffffffu, bias_lane.y, src));
                    z[2] = __fadd_rn(z[2], __shfl_sync(0xffffffffu, bias_lane.z, src));
                    z[3] = __fadd_rn(z[3], __shfl_sync(0xffffffffu, bias_lane.w, src));
                }
                if constexpr (GENERAL) {
                    const float4 a = mx_activate4(prm.act, make_float4(z[0], z[1], z[2], z[3]));
                    z[0] = a.x; z[1] = a.y; z[2] = a.z; z[3] = a.w;
                } else if (prm.act) {
#pragma unroll
                    for (int e = 0; e < 4; e++) z[e] = relu_value(z[e]);
                }
                if constexpr (KIND == 0) {
#pragma unroll
                    for (int e = 0; e < 4; e++) words[e] = __float_as_uint(z[e]);
                } else {
                    words[2 * q] = low_canonical_nan2<KIND>(low_pack2<KIND>(z[0], z[1]));
                    words[2 * q + 1] = low_canonical_nan2<KIND>(low_pack2<KIND>(z[2], z[3]));
                }
            }
            const uint32_t dst = stage + (uint32_t)(lane * 128 + ((j ^ (lane & 7)) << 4));
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(words[0]), "r"(words[1]), "r"(words[2]), "r"(words[3]) : "memory");
        }
        if (prm.staged) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                tma_store_2d(map_out, stage, c0, row0);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
        } else {
            __syncwarp();
            const int rows = prm.m - row0 < 32 ? prm.m - row0 : 32;
            for (int r = 0; r < rows; r++) {
                T *out = (T *)prm.out + (int64_t)(row0 + r) * prm.n + c0;
                uint32_t w;
                if constexpr (KIND == 0) {
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(stage + (uint32_t)(r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4)));
                    if (c0 + lane < prm.n) out[lane] = __uint_as_float(w);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int c = h * 32 + lane;
                        uint16_t e;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(e) : "r"(stage + (uint32_t)(r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2)));
                        if (c0 + c < prm.n) out[c] = e;
                    }
                }
            }
            __syncwarp();
        }
    }
}

template <int KIND, bool GENERAL>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MX_PAIR_THREADS, 1) mx_linear_pair_kernel(
        const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_out,
        const __grid_constant__ CUtensorMap map_xs, const __grid_constant__ CUtensorMap map_ws, MxLinear prm) {
    using Cfg = MxPairConfig;
    using T = typename MxElement<KIND>::type;
    constexpr int S = Cfg::kStages, R = Cfg::kScaleSlots, BN = Cfg::BN, CHUNK = mx_chunk<KIND>();
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S * Cfg::kStageBytes + R * Cfg::kScaleBytes + Cfg::kStagingBytes);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 3 * S + 2 * R + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const uint32_t bar_base = smem_u32(bars), smem_base = smem_u32(smem);
    const uint32_t staging_base = smem_base + S * Cfg::kStageBytes, scale_base = staging_base + Cfg::kStagingBytes;
    // full (codes), scale (scales in tensor memory) and accumulator-empty barriers are those of the even block; empty,
    // fetched and taken (scales in shared memory) and accumulator-full are each block's own
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (S + s); };
    auto scale_bar = [&](int s) { return bar_base + 8u * (2 * S + s); };
    auto fetched_bar = [&](int i) { return bar_base + 8u * (3 * S + i); };
    auto taken_bar = [&](int i) { return bar_base + 8u * (3 * S + R + i); };
    const uint32_t acc_full_bar = bar_base + 8u * (3 * S + 2 * R), acc_empty_bar = bar_base + 8u * (3 * S + 2 * R + 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; s++) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); mbar_init(scale_bar(s), 8); }
        for (int i = 0; i < R; i++) { mbar_init(fetched_bar(i), 1); mbar_init(taken_bar(i), 4); }
        mbar_init(acc_full_bar, 1); mbar_init(acc_empty_bar, 512);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)Cfg::kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = prm.tiles_m * prm.tiles_n, kb_count = prm.k_blocks;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(MX_PAIR_REGS_LOW));
        if (warp == 0) {
            if (lane == 0) {
                mx_dependent_wait();        // x, and the scales in tiles
                int stage = 0; uint32_t phase = 0;
                int armed = 0;
                bool ok = true;
                for (int tile = pair; tile < total_tiles && ok; tile += pairs) {
                    int mi, ni;
                    tile_origin(tile, prm.tiles_m, prm.tiles_n, prm.group_n, mi, ni);
                    const int m0 = mi * 256 + (int)rank * 128, n0 = ni * BN + (int)rank * 128;
                    for (int kb = 0; kb < kb_count; kb++) {
                        if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag)) { ok = false; break; }
                        const uint32_t sa = smem_base + stage * Cfg::kStageBytes;
                        const uint32_t leader_full = map_to_rank(full_bar(stage), 0);
                        if (rank == 0) mbar_expect_tx(full_bar(stage), 2 * Cfg::kStageBytes);
                        tma_load_2d_pair(sa, &map_x, leader_full, kb * (MX_BK / 2), m0);
                        tma_load_2d_pair(sa + Cfg::kABytes, &map_w, leader_full, kb * (MX_BK / 2), n0);
                        armed = armed < (1 << 30) ? armed + 1 : armed;
                        if (++stage == S) { stage = 0; phase ^= 1u; }
                    }
                }
                // giving up: the even block waits for both blocks' copies in flight; the odd one cannot leave before it
                if ((!ok || *abort_flag) && rank == 0) for (int i = armed > S ? armed - S : 0; i < armed; i++) mx_wait_landed(full_bar(i % S), (uint32_t)(i / S) & 1u);
            }
        } else if (warp == 2) {
            if (lane == 0) {
                mx_dependent_wait();
                int slot = 0; uint32_t phase = 0;
                int armed = 0;
                bool ok = true;
                for (int tile = pair; tile < total_tiles && ok; tile += pairs) {
                    int mi, ni;
                    tile_origin(tile, prm.tiles_m, prm.tiles_n, prm.group_n, mi, ni);
                    for (int kb = 0; kb < kb_count; kb++) {
                        if (!mbar_wait(taken_bar(slot), phase ^ 1u, abort_flag)) { ok = false; break; }
                        // two atoms of every band, 256 words: always a multiple of 16 bytes; bands past the matrix read as zeros
                        const uint32_t ss = scale_base + slot * Cfg::kScaleBytes;
                        mbar_expect_tx(fetched_bar(slot), Cfg::kScaleBytes);
                        tma_load_2d(ss, &map_xs, fetched_bar(slot), kb * 256, mi * 2 + (int)rank);
                        tma_load_2d(ss + 2 * MX_ATOM, &map_ws, fetched_bar(slot), kb * 256, ni * 2);
                        armed = armed < (1 << 30) ? armed + 1 : armed;
                        if (++slot == R) { slot = 0; phase ^= 1u; }
                    }
                }
                if (!ok || *abort_flag) for (int i = armed > R ? armed - R : 0; i < armed; i++) mx_wait_landed(fetched_bar(i % R), (uint32_t)(i / R) & 1u);
            }
        } else if (warp == 1) {
            if (rank == 0 && lane == 0) {
                const uint32_t id0 = mx_idesc(256, BN, 0), id2 = mx_idesc(256, BN, 2);
                int stage = 0; uint32_t phase = 0, done = 0;
                bool ok = true;
                for (int tile = pair; tile < total_tiles && ok; tile += pairs) {
                    for (int kb0 = 0; kb0 < kb_count && ok; kb0 += CHUNK, done++) {
                        if (!mbar_wait_cluster(acc_empty_bar, (done & 1u) ^ 1u, abort_flag)) { ok = false; break; }
                        tc_fence_after();
                        const int kb1 = kb0 + CHUNK < kb_count ? kb0 + CHUNK : kb_count;
                        for (int kb = kb0; kb < kb1; kb++) {
                            if (!mbar_wait(scale_bar(stage), phase, abort_flag) || !mbar_wait(full_bar(stage), phase, abort_flag)) { ok = false; break; }
                            tc_fence_after();
                            const uint32_t pa = smem_base + stage * Cfg::kStageBytes, pb = pa + Cfg::kABytes;
                            const uint32_t ts = tmem_base + BN + (uint32_t)(stage * Cfg::kScaleCols);
#pragma unroll
                            for (int k4 = 0; k4 < 4; k4++)
                                mx_mma<1>(tmem_base, mx_operand_desc(pa + k4 * 32), mx_operand_desc(pb + k4 * 32), (k4 & 1) ? id2 : id0, ts + (k4 >> 1) * 4, ts + 8 + (k4 >> 1) * 8,
                                          (kb != kb0 || k4 != 0) ? 1u : 0u);
                            umma_commit_pair(empty_bar(stage));
                            umma_commit_pair(map_to_rank(empty_bar(stage), 1));
                            if (++stage == S) { stage = 0; phase ^= 1u; }
                        }
                        if (ok) { umma_commit_pair(acc_full_bar); umma_commit_pair(map_to_rank(acc_full_bar, 1)); }
                    }
                }
            }
        }
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(MX_PAIR_REGS_SCALES));
        // this warp's 32 lanes of tensor memory get the same words as the other three warps'
        const uint32_t taddr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + BN;
        int stage = 0, slot = 0; uint32_t phase = 0, slot_phase = 0;
        bool ok = true;
        for (int tile = pair; tile < total_tiles && ok; tile += pairs) {
            for (int kb = 0; kb < kb_count; kb++) {
                ok = mx_warp_wait(fetched_bar(slot), slot_phase, abort_flag, lane);
                if (!ok) break;
                const uint32_t ps = scale_base + slot * Cfg::kScaleBytes + lane * 16;
                uint4 v[6];
                // columns: x half 0, x half 1, W half 0 (both bands), W half 1; in shared memory W's bands come one after the other
#pragma unroll
                for (int i = 0; i < 6; i++) {
                    const int atom = i < 2 ? i : 2 + ((i & 1) << 1) + ((i - 2) >> 1);
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[i].x), "=r"(v[i].y), "=r"(v[i].z), "=r"(v[i].w) : "r"(ps + (uint32_t)(atom * MX_ATOM)) : "memory");
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(taken_bar(slot));
                if (++slot == R) { slot = 0; slot_phase ^= 1u; }
                // the MMAs that read this stage's columns before have finished
                ok = mx_warp_wait(empty_bar(stage), phase ^ 1u, abort_flag, lane);
                if (!ok) break;
                tc_fence_after();
                tmem_store24(taddr + (uint32_t)(stage * Cfg::kScaleCols), v);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mx_arrive_rank(scale_bar(stage), 0);
                if (++stage == S) { stage = 0; phase ^= 1u; }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MX_PAIR_REGS_EPILOGUE));
        const int quarter = warp & 3, half = (warp - 8) >> 2;
        uint32_t done = 0;
        bool ok = true;
        for (int tile = pair; tile < total_tiles && ok; tile += pairs) {
            int mi, ni;
            tile_origin(tile, prm.tiles_m, prm.tiles_n, prm.group_n, mi, ni);
            const int row0 = mi * 256 + (int)rank * 128 + quarter * 32, col0 = ni * BN + half * 128;
            float4 bias_lane = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (prm.bias) {
                const T *b = (const T *)prm.bias;
                const int c = col0 + lane * 4;
                if (c < prm.n) bias_lane.x = mx_load<KIND>(b + c);
                if (c + 1 < prm.n) bias_lane.y = mx_load<KIND>(b + c + 1);
                if (c + 2 < prm.n) bias_lane.z = mx_load<KIND>(b + c + 2);
                if (c + 3 < prm.n) bias_lane.w = mx_load<KIND>(b + c + 3);
            }
            const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 128);
            ok = mx_warp_wait(acc_full_bar, done & 1u, abort_flag, lane);
            if (!ok) break;
            tc_fence_after();
            float sum[128];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                float t[32];
                tmem_load32(taddr + (uint32_t)(c * 32), t);
#pragma unroll
                for (int i = 0; i < 32; i++) sum[c * 32 + i] = t[i];
            }
            tc_fence_before();
            mx_arrive_rank(acc_empty_bar, 0);
            done++;
            for (int kb = CHUNK; kb < kb_count; kb += CHUNK, done++) {
                ok = mx_warp_wait(acc_full_bar, done & 1u, abort_flag, lane);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    float t[16];
                    tmem_load16(taddr + (uint32_t)(c * 16), t);
#pragma unroll
                    for (int i = 0; i < 16; i++) sum[c * 16 + i] = __fadd_rn(sum[c * 16 + i], t[i]);
                }
                tc_fence_before();
                mx_arrive_rank(acc_empty_bar, 0);
            }
            if (!ok) break;
            mx_emit<KIND, GENERAL>(prm, &map_out, staging_base + (uint32_t)((warp - 8) * 4096), row0, col0, sum, bias_lane, lane);
        }
        staged_drain(lane);
    }

    tc_fence_before();
    __syncthreads();
    __syncwarp();
    cluster_sync_all();     // neither block frees tensor memory or leaves while the partner may still signal it
    if (threadIdx.x == 0 && *abort_flag) atomicOr(prm.error_word, ERR_WAIT_TIMEOUT);
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)Cfg::kTmemCols) : "memory");
    }
}

// ------------------------------------------------------------------------------------------------
// Weight gradient from an 8-bit checkpoint: D[n, k] = sum over rows of g[row, n] x[row, k] on the tensor cores
// (tcgen05 kind::f16, BFLOAT16 operands, FP32 accumulators), two-SM tiles of 256 n x 256 k (784 columns as
// four tiles of 224 start off 128-byte lines and took 12 % longer than four of 256).
//   An E4M3 element under a power-of-two scale is a BFLOAT16 number as it stands (below 2^-133 it rounds), so the
// checkpoint costs one operand.  g is cut into BFLOAT16 pieces that add up to it exactly (apart from what lies below 2^-133):
// 8 + 8 + 8 significand bits for FLOAT32 (three products), 8 + 3 for FLOAT16 (two), one for BFLOAT16.  Every product is then exact; a FLOAT32 gradient
// takes three products at the BFLOAT16 rate where a split into TF32 numbers would take three at half of it.
//   mx_pieces_kernel writes the pieces and the checkpoint's values to scratch (10 bytes to move per element of a FLOAT32 g, 3
// per element of x; BFLOAT16 gradients whose rows TMA can address stay where they are), once each.  Converting inside the
// product, by worker warps between raw and operand tiles, repeats it for every tile and was bound by the workers'
// instructions and barriers: 1008 us on 8192 x 4096 x 4096 in FLOAT32, 523 us in BFLOAT16.
//   Both operands are contracted along their rows, that is, they are MN-major tiles (64 columns of one row = one
// 128-byte swizzle row), which TMA loads as they lie.  Tensor memory adds with truncation, so it only holds partial sums
// of kChunk stages, which the epilogue warps add into FP32 registers: two accumulators in turn.
//   Tiles that do not fill a wave of block pairs are cut into slices of the rows; their sums go to scratch and are
// added in ascending order by a last launch.
//   8192 x 4096 x 4096, whole calls in a row: FLOAT32 645 to 671 us (1.25 PFLOP/s of BFLOAT16 products with the conversion; the sustained rate
// under the power cap is 1.39), BFLOAT16 254 us (1.08: the operand loads of one product per stage do not keep up).
//   Sums of 65536 positive terms fall short by 17 units of 2^-23 (20 at most), of 1024 in BFLOAT16 or 512 in FLOAT16, one partial
// sum without a break, by 31 at most; half as many MMAs per partial sum cost 5 % (416 -> 437 us on 65536 x 784 x 4096, one call at a time).
// ------------------------------------------------------------------------------------------------
constexpr int MX_ROWS = 64;             // rows per stage
constexpr int MX_GRAD_THREADS = 384;    // warp 0 TMA, warp 1 MMA, warps 4-11 epilogue

template <int PIECES> struct MxGradConfig {
    static constexpr int kTileBytes = MX_ROWS * 128 * 2;                // one operand piece of 128 columns
    static constexpr int kStageBytes = (PIECES + 1) * kTileBytes;
    static constexpr int kStages = PIECES == 3 ? 3 : PIECES == 2 ? 4 : 6;
    static constexpr int kChunk = PIECES == 3 ? 4 : PIECES == 2 ? 8 : 16;      // stages per partial sum in tensor memory: at most 64 MMAs
    static constexpr int kStagingBytes = 8 * 4096;                      // a box of 32 rows x 32 columns per epilogue warp
    static constexpr int kSmemBytes = kStages * kStageBytes + kStagingBytes + 1024 + 256;
};

struct MxGrad {
    int n, k;
    int staged;                         // rows of `out` can be written by TMA
    int tiles_n, whole_tiles, units;    // units: the whole tiles, then `slices` per tile that is left
    int slices, stages, stages_per_slice;       // of MX_ROWS rows
    float *out, *partial;               // partial: [tile that is left][slice][256][256]
    int *error_word;
};

// Two floats as the next piece: the upper 16 bits of each (truncation keeps the remainder exact), which are taken off.
// At the first piece an infinity leaves no remainder (infinity - infinity would be NaN); a NaN leaves a NaN.
template <bool FIRST> __device__ __forceinline__ uint32_t mx_piece(float &a, float &b) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    const uint32_t word = __byte_perm(ua, ub, 0x7632);
    const float ra = __fsub_rn(a, __uint_as_float(ua & 0xffff0000u)), rb = __fsub_rn(b, __uint_as_float(ub & 0xffff0000u));
    a = FIRST && fabsf(a) == __uint_as_float(0x7f800000u) ? 0.0f : ra;
    b = FIRST && fabsf(b) == __uint_as_float(0x7f800000u) ? 0.0f : rb;
    return word;
}

// The first g_blocks blocks cut g [rows, n] into pieces, planes [PIECES][rows][g_pitch]; the others restore x into [rows, x_pitch].
// Padding columns are written as zeros.  A thread takes groups of eight columns.
template <int KIND, bool VEC>
__global__ void __launch_bounds__(MX_THREADS) mx_pieces_kernel(const typename MxElement<KIND>::type *__restrict__ g, int64_t rows, int64_t n, int64_t g_pitch, uint16_t *__restrict__ g_planes, int g_blocks,
                                                               const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, int64_t x_pitch, int64_t scale_pitch, uint16_t *__restrict__ x_plane) {
    constexpr int PIECES = KIND == 0 ? 3 : KIND == 1 ? 1 : 2;
    mx_dependent_release();
    if ((int)blockIdx.x < g_blocks) {
        __shared__ float boxes[VEC ? 1 : MX_WARPS][VEC ? 1 : 256];
        const int64_t per_row = g_pitch / 8, total = rows * per_row, hop = (int64_t)g_blocks * MX_THREADS;
        int64_t i = blockIdx.x * (int64_t)MX_THREADS + threadIdx.x, row = i / per_row, group = i - row * per_row;
        const int64_t hop_rows = hop / per_row, hop_groups = hop - hop_rows * per_row;
        for (; (i & ~(int64_t)31) < total; i += hop) {
            const int64_t left = i < total ? n - group * 8 : 0;
            const int count = left >= 8 ? 8 : left > 0 ? (int)left : 0;
            float f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (VEC) { if (count) mx_load8<KIND>(g + row * n + group * 8, f); }
            else {
                float raw[8];
                mx_gather8<KIND>(g, row * n + group * 8, 1, count, threadIdx.x & 31, raw);
                mx_exchange8(raw, boxes[threadIdx.x >> 5], threadIdx.x & 31, f);
            }
            if (i < total) {
#pragma unroll
                for (int piece = 0; piece < PIECES; piece++) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) w[e] = piece == 0 ? mx_piece<true>(f[2 * e], f[2 * e + 1]) : mx_piece<false>(f[2 * e], f[2 * e + 1]);
                    *reinterpret_cast<uint4 *>(g_planes + ((int64_t)piece * rows + row) * g_pitch + group * 8) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            row += hop_rows; group += hop_groups;
            if (group >= per_row) { group -= per_row; row++; }
        }
    } else {
        const int64_t per_row = x_pitch / 8, total = rows * per_row, hop = (int64_t)(gridDim.x - g_blocks) * MX_THREADS;
        int64_t i = (int64_t)(blockIdx.x - g_blocks) * MX_THREADS + threadIdx.x, row = i / per_row, group = i - row * per_row;
        const int64_t hop_rows = hop / per_row, hop_groups = hop - hop_rows * per_row;
        for (; i < total; i += hop) {
            const uint2 c = __ldg(reinterpret_cast<const uint2 *>(codes + row * x_pitch + group * 8));
            const float scale = mx_scale_value(__ldg(scales + row * scale_pitch + (group >> 2)));
            float v[8];
            mx_decode8x2(c.x & 0xffffu, v[0], v[1]); mx_decode8x2(c.x >> 16, v[2], v[3]);
            mx_decode8x2(c.y & 0xffffu, v[4], v[5]); mx_decode8x2(c.y >> 16, v[6], v[7]);
            *reinterpret_cast<uint4 *>(x_plane + row * x_pitch + group * 8) = make_uint4(low_pack2<1>(v[0] * scale, v[1] * scale), low_pack2<1>(v[2] * scale, v[3] * scale),
                                                                                         low_pack2<1>(v[4] * scale, v[5] * scale), low_pack2<1>(v[6] * scale, v[7] * scale));
            row += hop_rows; group += hop_groups;
            if (group >= per_row) { group -= per_row; row++; }
        }
    }
}

template <int PIECES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MX_GRAD_THREADS, 1) mx_weight_gradient_kernel(
        const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_out,
        const __grid_constant__ CUtensorMap map_partial, MxGrad prm) {
    using Cfg = MxGradConfig<PIECES>;
    constexpr int S = Cfg::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S * Cfg::kStageBytes + Cfg::kStagingBytes);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * S + 4);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const uint32_t bar_base = smem_u32(bars), smem_base = smem_u32(smem);
    // full and accumulator-empty barriers are those of the even block; empty and accumulator-full are each block's own
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (S + s); };
    auto acc_full_bar = [&](int a) { return bar_base + 8u * (2 * S + a); };
    auto acc_empty_bar = [&](int a) { return bar_base + 8u * (2 * S + 2 + a); };

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; s++) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int a = 0; a < 2; a++) { mbar_init(acc_full_bar(a), 1); mbar_init(acc_empty_bar(a), 16); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    mx_dependent_release();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    // a unit's tile and stages; every slice has at least one
    auto unit_of = [&](int unit, int &n0, int &k0, int &first, int &count) {
        int tile = unit;
        first = 0; count = prm.stages;
        if (unit >= prm.whole_tiles) {
            const int u = unit - prm.whole_tiles;
            tile = prm.whole_tiles + u / prm.slices;
            first = u % prm.slices * prm.stages_per_slice;
            count = prm.stages - first < prm.stages_per_slice ? prm.stages - first : prm.stages_per_slice;
        }
        n0 = tile % prm.tiles_n * 256; k0 = tile / prm.tiles_n * 256;
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 0) {
            if (lane == 0) {
                mx_dependent_wait();        // the operands
                int stage = 0; uint32_t phase = 0;
                int armed = 0;
                bool ok = true;
                for (int unit = pair; unit < prm.units && ok; unit += pairs) {
                    int n0, k0, first, count;
                    unit_of(unit, n0, k0, first, count);
                    n0 += (int)rank * 128; k0 += (int)rank * 128;
                    for (int i = 0; i < count; i++) {
                        if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag)) { ok = false; break; }
                        const uint32_t leader_full = map_to_rank(full_bar(stage), 0), pa = smem_base + stage * Cfg::kStageBytes, pb = pa + PIECES * Cfg::kTileBytes;
                        if (rank == 0) mbar_expect_tx(full_bar(stage), 2 * Cfg::kStageBytes);
                        const int r0 = (first + i) * MX_ROWS;
                        // boxes of 64 columns (128 bytes) x 64 rows; columns and rows past the matrix read as zeros
#pragma unroll
                        for (int half = 0; half < 2; half++) {
#pragma unroll
                            for (int piece = 0; piece < PIECES; piece++)
                                tma_load_3d_pair(pa + piece * Cfg::kTileBytes + half * (MX_ROWS * 128), &map_g, leader_full, n0 + half * 64, r0, piece);
                            tma_load_2d_pair(pb + half * (MX_ROWS * 128), &map_x, leader_full, k0 + half * 64, r0);
                        }
                        armed = armed < (1 << 30) ? armed + 1 : armed;
                        if (++stage == S) { stage = 0; phase ^= 1u; }
                    }
                }
                // giving up: the even block waits for both blocks' copies in flight; the odd one cannot leave before it
                if ((!ok || *abort_flag) && rank == 0) for (int i = armed > S ? armed - S : 0; i < armed; i++) mx_wait_landed(full_bar(i % S), (uint32_t)(i / S) & 1u);
            }
        } else if (warp == 1) {
            if (rank == 0 && lane == 0) {
                // BFLOAT16 operands, FP32 accumulators, both MN-major, 256 x 256
                const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | ((256u >> 3) << 17) | ((256u >> 4) << 24);
                // groups of 64 columns 8 KB apart (leading offset), groups of 8 rows 1 KB (stride offset), 128-byte swizzle
                const uint64_t fixed = ((uint64_t)((MX_ROWS * 128u) >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
                auto desc = [&](uint32_t addr) { return fixed | (uint64_t)((addr & 0x3ffffu) >> 4); };
                int stage = 0; uint32_t phase = 0, chunk = 0;
                bool ok = true;
                for (int unit = pair; unit < prm.units && ok; unit += pairs) {
                    int n0, k0, first, count;
                    unit_of(unit, n0, k0, first, count);
                    for (int i0 = 0; i0 < count && ok; i0 += Cfg::kChunk, chunk++) {
                        const int buf = chunk & 1;
                        if (!mbar_wait_cluster(acc_empty_bar(buf), ((chunk >> 1) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
                        tc_fence_after();
                        const uint32_t d = tmem_base + (uint32_t)(buf * 256);
                        const int i1 = i0 + Cfg::kChunk < count ? i0 + Cfg::kChunk : count;
                        for (int i = i0; i < i1; i++) {
                            if (!mbar_wait_cluster(full_bar(stage), phase, abort_flag)) { ok = false; break; }
                            tc_fence_after();
                            const uint32_t pa = smem_base + stage * Cfg::kStageBytes, pb = pa + PIECES * Cfg::kTileBytes;
#pragma unroll
                            for (int piece = PIECES - 1; piece >= 0; piece--)         // small terms first
#pragma unroll
                                for (int r16 = 0; r16 < MX_ROWS / 16; r16++)
                                    umma_f16_pair(d, desc(pa + piece * Cfg::kTileBytes + r16 * 2048), desc(pb + r16 * 2048), idesc,
                                                  (i != i0 || piece != PIECES - 1 || r16 != 0) ? 1u : 0u);
                            umma_commit_pair(empty_bar(stage));
                            umma_commit_pair(map_to_rank(empty_bar(stage), 1));
                            if (++stage == S) { stage = 0; phase ^= 1u; }
                        }
                        if (ok) { umma_commit_pair(acc_full_bar(buf)); umma_commit_pair(map_to_rank(acc_full_bar(buf), 1)); }
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        uint32_t chunk = 0;
        bool ok = true;
        for (int unit = pair; unit < prm.units && ok; unit += pairs) {
            int n0, k0, first, count;
            unit_of(unit, n0, k0, first, count);
            float sum[128];
#pragma unroll
            for (int q = 0; q < 128; q++) sum[q] = 0.0f;
            for (int i0 = 0; i0 < count; i0 += Cfg::kChunk, chunk++) {
                const int buf = chunk & 1;
                ok = mx_warp_wait(acc_full_bar(buf), (chunk >> 1) & 1u, abort_flag, lane);
                if (!ok) break;
                tc_fence_after();
                const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * 256 + half * 128);
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    float t[16];
                    tmem_load16(taddr + (uint32_t)(q * 16), t);
#pragma unroll
                    for (int e = 0; e < 16; e++) sum[q * 16 + e] = __fadd_rn(sum[q * 16 + e], t[e]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mx_arrive_rank(acc_empty_bar(buf), 0);
            }
            if (!ok) break;
            // out through boxes of 32 x 32 in shared memory (16-byte chunk j of row r at chunk j ^ (r & 7)) and TMA, which clips
            // the edges; rows of `out` that TMA cannot address are copied from the box, a row per instruction
            const bool partial = unit >= prm.whole_tiles;
            const int row0 = (int)rank * 128 + quarter * 32, row_limit = partial ? 32 : prm.n - n0 - row0;
            const uint32_t box = smem_base + (uint32_t)(S * Cfg::kStageBytes + (warp - 4) * 4096);
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const int col = half * 128 + b * 32;        // in the tile
                if (row_limit <= 0 || (!partial && k0 + col >= prm.k)) break;      // warp-uniform
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");       // the previous box has been read
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; j++)
                    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(box + (uint32_t)(lane * 128 + ((j ^ (lane & 7)) << 4))),
                                 "f"(sum[b * 32 + j * 4]), "f"(sum[b * 32 + j * 4 + 1]), "f"(sum[b * 32 + j * 4 + 2]), "f"(sum[b * 32 + j * 4 + 3]) : "memory");
                if (partial || prm.staged) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        if (partial) tma_store_2d(&map_partial, box, col, (unit - prm.whole_tiles) * 256 + row0);
                        else tma_store_2d(&map_out, box, k0 + col, n0 + row0);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                } else {
                    __syncwarp();
                    float *out = prm.out + (int64_t)(n0 + row0) * prm.k + k0 + col;
                    for (int r = 0; r < 32 && r < row_limit; r++) {
                        float v;
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(box + (uint32_t)(r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4)));
                        if (k0 + col + lane < prm.k) out[(int64_t)r * prm.k + lane] = v;
                    }
                    __syncwarp();
                }
            }
        }
        staged_drain(lane);
    }

    tc_fence_before();
    __syncthreads();
    __syncwarp();
    cluster_sync_all();     // neither block frees tensor memory or leaves while the partner may still signal it
    if (threadIdx.x == 0 && *abort_flag) atomicOr(prm.error_word, ERR_WAIT_TIMEOUT);
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    }
}

// Small products (mx_gradient_small): three launches and two-SM tiles would cost more than the work.  A block of 32 warps
// makes partial sums of 8 n x 32 k results over its share of the rows: a lane per column of x (one block of the
// checkpoint), the warps take rows in turn, eight at a time in flight.  The warps' FP32 sums are added in a fixed order
// through shared memory, those of a cluster's blocks, also in order, through the first one's view of theirs.
constexpr int MX_SMALL_N = 8, MX_SMALL_THREADS = 1024, MX_SMALL_FLIGHT = 8;
template <int KIND>
__global__ void __launch_bounds__(MX_SMALL_THREADS) mx_weight_gradient_small_kernel(int64_t rows, int n, int k, const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                                                                                    int64_t code_pitch, int64_t scale_pitch, const typename MxElement<KIND>::type *__restrict__ g, float *__restrict__ out, int slices) {
    __shared__ float sums[32][MX_SMALL_N][32];
    __shared__ float totals[MX_SMALL_N][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int slice = blockIdx.x % slices, block = blockIdx.x / slices, n0 = blockIdx.y * MX_SMALL_N;
    const int64_t begin = rows * slice / slices, end = rows * (slice + 1) / slices;
    float sum[MX_SMALL_N] = {};
    for (int64_t r0 = begin + warp; r0 < end; r0 += MX_SMALL_FLIGHT * 32) {
        uint32_t code[MX_SMALL_FLIGHT], byte[MX_SMALL_FLIGHT];
        float up[MX_SMALL_FLIGHT];
#pragma unroll
        for (int q = 0; q < MX_SMALL_FLIGHT; q++) {
            const int64_t row = r0 + q * 32;
            const bool here = row < end;
            code[q] = here ? __ldg(codes + row * code_pitch + block * MX_BLOCK + lane) : 0u;
            byte[q] = here ? __ldg(scales + row * scale_pitch + block) : 0u;
            up[q] = here && lane < MX_SMALL_N && n0 + lane < n ? mx_load<KIND>(g + row * n + n0 + lane) : 0.0f;
        }
#pragma unroll
        for (int q = 0; q < MX_SMALL_FLIGHT; q++) {
            float x, unused;
            mx_decode8x2(code[q], x, unused);
            x *= mx_scale_value(byte[q]);
#pragma unroll
            for (int e = 0; e < MX_SMALL_N; e++) sum[e] = fmaf(__shfl_sync(0xffffffffu, up[q], e), x, sum[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < MX_SMALL_N; e++) sums[warp][e][lane] = sum[e];
    __syncthreads();
    if (warp < MX_SMALL_N) {
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < 32; w++) total += sums[w][warp][lane];
        totals[warp][lane] = total;
    }
    __syncwarp();
    cluster_sync_all();
    if (slice == 0 && warp < MX_SMALL_N) {
        float total = totals[warp][lane];
        for (int q = 1; q < slices; q++) {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_rank(smem_u32(&totals[warp][lane]), (uint32_t)q)) : "memory");
            total += v;
        }
        const int col = block * MX_BLOCK + lane;
        if (n0 + warp < n && col < k) out[(int64_t)(n0 + warp) * k + col] = total;
    }
    __syncwarp();
    cluster_sync_all();         // no block leaves while another reads its sums
}

// The tiles that were cut into slices: their sums in ascending order.  blockIdx.y: the tile; a thread adds four columns.
// Loads from L2: the launch in front may still write the sums when this one starts, and the read-only path (ld.global.nc)
// is only defined for memory that nothing writes while the kernel runs.
__global__ void __launch_bounds__(MX_THREADS) mx_add_slices_kernel(MxGrad prm) {
    mx_dependent_wait();
    const int tile = prm.whole_tiles + blockIdx.y, n0 = tile % prm.tiles_n * 256, k0 = tile / prm.tiles_n * 256;
    const int i = blockIdx.x * MX_THREADS + threadIdx.x, row = i >> 6, col = (i & 63) * 4;
    if (n0 + row >= prm.n || k0 + col >= prm.k) return;
    const float *p = prm.partial + (int64_t)blockIdx.y * prm.slices * 65536 + row * 256 + col;
    float4 a = __ldcg(reinterpret_cast<const float4 *>(p));
    for (int q = 1; q < prm.slices; q++) {
        const float4 b = __ldcg(reinterpret_cast<const float4 *>(p + (int64_t)q * 65536));
        a.x = __fadd_rn(a.x, b.x); a.y = __fadd_rn(a.y, b.y); a.z = __fadd_rn(a.z, b.z); a.w = __fadd_rn(a.w, b.w);
    }
    float *out = prm.out + (int64_t)(n0 + row) * prm.k + k0 + col;
    if ((prm.k & 3) == 0 && ((uintptr_t)prm.out & 15) == 0) *reinterpret_cast<float4 *>(out) = a;
    else {
        const float v[4] = {a.x, a.y, a.z, a.w};
        for (int e = 0; e < 4; e++) if (k0 + col + e < prm.k) out[e] = v[e];
    }
}

}  // namespace

// What a kernel needs once per device before its first launch: leave to use `smem` bytes of shared memory, and a look
// at its registers per thread (those a register split at run time draws on).
template <typename Kernel>
static cudaError_t mx_prepare_kernel(Kernel kernel, int smem, int least_regs, std::atomic<uint64_t> &done) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (device & 63);
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    cudaFuncAttributes attr;
    e = cudaFuncGetAttributes(&attr, kernel);
    if (e != cudaSuccess) return e;
    if (attr.numRegs < least_regs) return cudaErrorLaunchOutOfResources;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && device < 64) done.fetch_or(bit, std::memory_order_release);
    return e;
}

// A launch that may overlap the end of the one before it (see mx_dependent_wait).
template <typename... Args>
static cudaError_t mx_launch_dependent(void (*kernel)(Args...), dim3 grid, int threads, int smem, cudaStream_t s, std::common_type_t<Args>... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3((unsigned)threads); cfg.dynamicSmemBytes = (size_t)smem; cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

#define MX_KINDS(dtype, CALL) ((dtype) == DType::F32 ? CALL(0) : (dtype) == DType::BF16 ? CALL(1) : (dtype) == DType::F16 ? CALL(2) : cudaErrorInvalidValue)

template <int FORMAT, int KIND, bool KEEP>
static cudaError_t launch_mx_quantize(cudaStream_t s, const void *x, const Index4 &ix, uint8_t *codes, uint8_t *scales, uint8_t *tiles) {
    using T = typename MxElement<KIND>::type;
    const int64_t rows = ix.shape[0] * ix.shape[1] * ix.shape[2], cols = ix.shape[3];
    if (rows == 0 || cols == 0) return cudaSuccess;
    // the rows lie at one distance when each leading axis continues the next
    bool even = true;
    int64_t row_step = 0, extent = 1;
    for (int d = 2; d >= 0; d--) {
        if (ix.shape[d] == 1) continue;
        if (extent == 1) row_step = ix.sa[d];
        else even &= ix.sa[d] == row_step * extent;
        extent *= ix.shape[d];
    }
    constexpr int E = KIND == 0 ? 8 : 16;       // elements of 32 bytes
    const bool vec = even && (ix.sa[3] == 1 || cols == 1) && (uintptr_t)x % 32 == 0 && (rows == 1 || row_step % E == 0);
    // dense rows of whole scale words are one long row
    const bool flat = vec && !tiles && row_step == cols && cols % (4 * MX_BLOCK) == 0;
    const int64_t r = flat ? 1 : rows, c = flat ? rows * cols : cols;
    const int grid = mx_grid(r * mx_scale_bytes(c) * (vec ? MX_BLOCK / E : 4));
    const uint32_t atoms = (uint32_t)mx_tile_atoms(cols);
    const auto launch = [&](auto kernel, auto shape) { kernel<<<grid, MX_THREADS, 0, s>>>((const T *)x, ix, shape, row_step, even ? 1 : 0, codes, scales, tiles, atoms); };
    if (mx_narrow_rows(r, c)) {
        if (vec) launch(mx_quantize_kernel<FORMAT, KIND, true, KEEP, uint32_t>, mx_rows<uint32_t>(r, c, FORMAT, E));
        else launch(mx_quantize_kernel<FORMAT, KIND, false, KEEP, uint32_t>, mx_rows<uint32_t>(r, c, FORMAT));
    } else {
        if (vec) launch(mx_quantize_kernel<FORMAT, KIND, true, KEEP, int64_t>, mx_rows<int64_t>(r, c, FORMAT, E));
        else launch(mx_quantize_kernel<FORMAT, KIND, false, KEEP, int64_t>, mx_rows<int64_t>(r, c, FORMAT));
    }
    return cudaGetLastError();
}

cudaError_t mx_quantize(cudaStream_t s, int format, bool keep_nonzero, DType dtype, const void *x, const Index4 &ix, uint8_t *codes, uint8_t *scales, uint8_t *tiles) {
#define CALL4(KIND) (keep_nonzero ? launch_mx_quantize<4, KIND, true>(s, x, ix, codes, scales, tiles) : launch_mx_quantize<4, KIND, false>(s, x, ix, codes, scales, tiles))
#define CALL8(KIND) (keep_nonzero ? launch_mx_quantize<8, KIND, true>(s, x, ix, codes, scales, tiles) : launch_mx_quantize<8, KIND, false>(s, x, ix, codes, scales, tiles))
    return format == 4 ? MX_KINDS(dtype, CALL4) : format == 8 ? MX_KINDS(dtype, CALL8) : cudaErrorInvalidValue;
#undef CALL4
#undef CALL8
}

// A dense [rows, cols] tensor beside a block-scaled one of the same shape: whether all its groups are whole and aligned,
// and the shape to count in (dense rows of whole scale words are one long row).
template <typename T> static bool mx_dense_shape(int64_t &rows, int64_t &cols, const void *a, const void *b) {
    const bool vec = cols % 8 == 0 && (uintptr_t)a % (8 * sizeof(T)) == 0 && (uintptr_t)b % (8 * sizeof(T)) == 0;
    if (vec && cols % (4 * MX_BLOCK) == 0) { cols *= rows; rows = 1; }
    return vec;
}

template <int FORMAT, int KIND>
static cudaError_t launch_mx_restore(cudaStream_t s, const uint8_t *codes, const uint8_t *scales, int64_t rows, int64_t cols, void *out) {
    using T = typename MxElement<KIND>::type;
    if (rows == 0 || cols == 0) return cudaSuccess;
    const bool vec = mx_dense_shape<T>(rows, cols, out, out);
    const auto launch = [&](auto kernel, auto shape) { kernel<<<mx_grid(rows * mx_scale_bytes(cols) * 4), MX_THREADS, 0, s>>>(codes, scales, shape, cols, (T *)out); };
    if (mx_narrow_rows(rows, cols)) {
        if (vec) launch(mx_restore_kernel<FORMAT, KIND, true, uint32_t>, mx_rows<uint32_t>(rows, cols, FORMAT));
        else launch(mx_restore_kernel<FORMAT, KIND, false, uint32_t>, mx_rows<uint32_t>(rows, cols, FORMAT));
    } else {
        if (vec) launch(mx_restore_kernel<FORMAT, KIND, true, int64_t>, mx_rows<int64_t>(rows, cols, FORMAT));
        else launch(mx_restore_kernel<FORMAT, KIND, false, int64_t>, mx_rows<int64_t>(rows, cols, FORMAT));
    }
    return cudaGetLastError();
}

cudaError_t mx_restore(cudaStream_t s, int format, DType dtype, const uint8_t *codes, const uint8_t *scales, int64_t rows, int64_t cols, void *out) {
#define CALL4(KIND) launch_mx_restore<4, KIND>(s, codes, scales, rows, cols, out)
#define CALL8(KIND) launch_mx_restore<8, KIND>(s, codes, scales, rows, cols, out)
    return format == 4 ? MX_KINDS(dtype, CALL4) : format == 8 ? MX_KINDS(dtype, CALL8) : cudaErrorInvalidValue;
#undef CALL4
#undef CALL8
}

template <int KIND>
static cudaError_t launch_mx_activation_gradient(cudaStream_t s, int act, const uint8_t *codes, const uint8_t *scales, const void *g, int64_t rows, int64_t cols, void *out) {
    using T = typename MxElement<KIND>::type;
    if (rows == 0 || cols == 0) return cudaSuccess;
    const bool vec = mx_dense_shape<T>(rows, cols, g, out);
    const auto launch = [&](auto kernel, auto shape) { kernel<<<mx_grid(rows * mx_scale_bytes(cols) * 4), MX_THREADS, 0, s>>>(act, codes, scales, (const T *)g, shape, cols, (T *)out); };
    if (mx_narrow_rows(rows, cols)) {
        if (vec) launch(mx_activation_gradient_kernel<KIND, true, uint32_t>, mx_rows<uint32_t>(rows, cols, 8));
        else launch(mx_activation_gradient_kernel<KIND, false, uint32_t>, mx_rows<uint32_t>(rows, cols, 8));
    } else {
        if (vec) launch(mx_activation_gradient_kernel<KIND, true, int64_t>, mx_rows<int64_t>(rows, cols, 8));
        else launch(mx_activation_gradient_kernel<KIND, false, int64_t>, mx_rows<int64_t>(rows, cols, 8));
    }
    return cudaGetLastError();
}

cudaError_t mx_activation_gradient(cudaStream_t s, int act, DType dtype, const uint8_t *codes, const uint8_t *scales, const void *g,
                                   int64_t rows, int64_t cols, void *out) {
#define CALL(KIND) launch_mx_activation_gradient<KIND>(s, act, codes, scales, g, rows, cols, out)
    return MX_KINDS(dtype, CALL);
#undef CALL
}

// Tensor map over the codes of a 4-bit operand [rows, k]: boxes of 256 elements x box_rows, 128-byte swizzle.
static bool make_code_map(CUtensorMap *map, const uint8_t *codes, int64_t rows, int64_t k, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)(k / 2), (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(k / 2)};
    cuuint32_t box[2] = {MX_BK / 2, (cuuint32_t)box_rows};
    cuuint32_t elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(codes), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tensor map over tiled scales: rows are the bands of 128 rows; boxes of two atoms x `bands`.
static bool make_tile_map(CUtensorMap *map, const uint8_t *tiles, int64_t rows, int64_t k, int bands) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)(mx_tile_atoms(k) * MX_ATOM / 4), (cuuint64_t)((rows + 127) / 128)};
    cuuint64_t strides[1] = {(cuuint64_t)(mx_tile_atoms(k) * MX_ATOM)};
    cuuint32_t box[2] = {256, (cuuint32_t)bands};
    cuuint32_t elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<uint8_t *>(tiles), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, int KIND>
static cudaError_t launch_mx_few(cudaStream_t s, const uint8_t *x, const uint8_t *w, const MxLinear &prm, int slices) {
    using Cfg = MxFewConfig<BN>;
    CUtensorMap map_w, map_x;
    const int64_t k = (int64_t)prm.blocks * MX_BLOCK;
    if (!make_code_map(&map_w, w, prm.n, k, 128) || !make_code_map(&map_x, x, prm.m, k, BN)) return cudaErrorInvalidValue;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = mx_prepare_kernel(mx_linear_few_kernel<BN, KIND>, Cfg::kSmemBytes, 0, done);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((int64_t)slices * prm.tiles_n * prm.tiles_m));
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = Cfg::kSmemBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)slices, 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = prm.after_x ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, mx_linear_few_kernel<BN, KIND>, map_w, map_x, prm, slices);
}

template <int KIND, bool GENERAL>
static cudaError_t launch_mx_pair(cudaStream_t s, const uint8_t *x, const uint8_t *w, const uint8_t *x_tiles, const uint8_t *w_tiles, MxLinear prm, int sm_count) {
    using Cfg = MxPairConfig;
    using T = typename MxElement<KIND>::type;
    CUtensorMap map_x, map_w, map_out, map_xs, map_ws;
    const int64_t k = (int64_t)prm.blocks * MX_BLOCK;
    EncodeTiledFn fn = encode_fn();
    if (!fn || !make_code_map(&map_x, x, prm.m, k, 128) || !make_code_map(&map_w, w, prm.n, k, 128)
        || !make_tile_map(&map_xs, x_tiles, prm.m, k, 1) || !make_tile_map(&map_ws, w_tiles, prm.n, k, 2)) return cudaErrorInvalidValue;
    prm.staged = 0;
    map_out = map_x;            // unused unless staged
    if ((int64_t)prm.n * sizeof(T) % 16 == 0 && ((uintptr_t)prm.out & 15) == 0) {
        cuuint64_t dims[2] = {(cuuint64_t)prm.n, (cuuint64_t)prm.m};
        cuuint64_t strides[1] = {(cuuint64_t)prm.n * sizeof(T)};
        cuuint32_t box[2] = {128 / sizeof(T), 32};
        cuuint32_t elem[2] = {1, 1};
        prm.staged = fn(&map_out, KIND == 0 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, prm.out, dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    prm.tiles_m = (prm.m + 255) / 256; prm.tiles_n = (prm.n + 255) / 256;
    if ((int64_t)prm.tiles_m * prm.tiles_n >= (1ll << 30)) return cudaErrorInvalidValue;
    const int groups = (prm.tiles_n + 7) / 8;
    prm.group_n = (prm.tiles_n + groups - 1) / groups;
    const int tiles = prm.tiles_m * prm.tiles_n, pairs = sm_count / 2;
    // the register split draws on what the block was launched with
    static std::atomic<uint64_t> done{0};
    cudaError_t e = mx_prepare_kernel(mx_linear_pair_kernel<KIND, GENERAL>, Cfg::kSmemBytes, (MX_PAIR_REGS_LOW + MX_PAIR_REGS_SCALES + 2 * MX_PAIR_REGS_EPILOGUE + 3) / 4, done);
    if (e != cudaSuccess) return e;
    const unsigned grid = (unsigned)(2 * (tiles < pairs ? tiles : pairs));
    if (prm.after_x) return mx_launch_dependent(mx_linear_pair_kernel<KIND, GENERAL>, dim3(grid), MX_PAIR_THREADS, Cfg::kSmemBytes, s, map_x, map_w, map_out, map_xs, map_ws, prm);
    mx_linear_pair_kernel<KIND, GENERAL><<<grid, MX_PAIR_THREADS, Cfg::kSmemBytes, s>>>(map_x, map_w, map_out, map_xs, map_ws, prm);
    return cudaGetLastError();
}

// SYNAPTIK_CUDA_MX_PAIR=0 / 1 forces the one-SM / two-SM form of the 4-bit product (for comparisons).
static int forced_mx_pair() {
    static const int v = [] { const char *e = getenv("SYNAPTIK_CUDA_MX_PAIR"); return e && (e[0] == '0' || e[0] == '1') ? e[0] - '0' : -1; }();
    return v;
}

// Two-SM tiles where the one-SM tiles of 128 x 128 would take more than one wave: measured with the quantisation of x, K =
// 4096: 512 x 4096 (128 tiles) 34.6 us on one-SM tiles and 32.8 on two-SM ones, 4096 x 128 (32) 31.9 and 41.4, 1024 x 4096
// (256) 60.6 and 34.2, 1 x 4096 15.4 and 29.7.
bool mx_linear_tiled(int64_t m, int64_t n, int sm_count) {
    if (sm_count < 2) return false;
    if (forced_mx_pair() >= 0) return forced_mx_pair() == 1;
    return m > 128 && ((m + 127) / 128) * ((n + 127) / 128) > sm_count;
}
int64_t mx_tile_bytes(int64_t rows, int64_t k) { return (rows + 127) / 128 * mx_tile_atoms(k) * MX_ATOM; }
cudaError_t mx_tile_scales(cudaStream_t s, const uint8_t *scales, int64_t rows, int64_t k, uint8_t *tiles, bool after_x) {
    if (rows == 0) return cudaSuccess;
    const int64_t blocks = ((rows + 127) / 128 * 32 * ((mx_blocks(k) + 3) / 4) + MX_THREADS - 1) / MX_THREADS;
    const unsigned grid = (unsigned)(blocks < 148 * 8 ? blocks : 148 * 8);
    if (after_x) return mx_launch_dependent(mx_tile_scales_kernel, dim3(grid), MX_THREADS, 0, s, scales, rows, mx_blocks(k), tiles);
    mx_tile_scales_kernel<<<grid, MX_THREADS, 0, s>>>(scales, rows, mx_blocks(k), tiles);
    return cudaGetLastError();
}

template <int KIND>
static cudaError_t launch_mx_linear(cudaStream_t s, const uint8_t *x, const uint8_t *w, const uint8_t *x_tiles, const uint8_t *w_tiles, MxLinear prm, int sm_count) {
    if (x_tiles && w_tiles)
        return prm.act && prm.act != (int)Op::RELU ? launch_mx_pair<KIND, true>(s, x, w, x_tiles, w_tiles, prm, sm_count)
                                                   : launch_mx_pair<KIND, false>(s, x, w, x_tiles, w_tiles, prm, sm_count);
    const int bn = prm.m <= 16 ? 16 : prm.m <= 32 ? 32 : prm.m <= 64 ? 64 : 128;
    prm.tiles_n = (prm.n + 127) / 128; prm.tiles_m = (prm.m + bn - 1) / bn;
    const int64_t tiles = (int64_t)prm.tiles_n * prm.tiles_m;
    if (tiles >= (1ll << 28)) return cudaErrorInvalidValue;
    // Slices of the contraction while blocks are left over, each of at least `least` k-blocks: adding up the slices costs
    // time with the rows of a tile.  Measured: 203 x 4096 x 1000 in slices of 4 and 2 k-blocks 20.5 and 24.5 us, 16 x 784 x
    // 4096 in slices of 4, 2 and 1 14.3, 12.7 and 12.3 us.
    const int least = bn <= 32 ? 1 : bn == 64 ? 2 : 4;
    int slices = 1;
    while (slices < 8 && tiles * slices * 2 <= sm_count && prm.k_blocks >= slices * 2 * least) slices *= 2;
    switch (bn) {
        case 16: return launch_mx_few<16, KIND>(s, x, w, prm, slices);
        case 32: return launch_mx_few<32, KIND>(s, x, w, prm, slices);
        case 64: return launch_mx_few<64, KIND>(s, x, w, prm, slices);
        default: return launch_mx_few<128, KIND>(s, x, w, prm, slices);
    }
}

cudaError_t mx_linear(cudaStream_t s, DType dtype, int act, int64_t m, int64_t n, int64_t k, const uint8_t *x, const uint8_t *x_scales,
                      const uint8_t *w, const uint8_t *w_scales, const uint8_t *x_tiles, const uint8_t *w_tiles, const void *bias, void *out,
                      bool after_x, int sm_count, int *error_word) {
    if (m == 0 || n == 0) return cudaSuccess;
    MxLinear prm = {};
    prm.after_x = after_x ? 1 : 0;
    prm.m = (int)m; prm.n = (int)n; prm.blocks = (int)(k / MX_BLOCK); prm.k_blocks = (int)((k + MX_BK - 1) / MX_BK);
    prm.scale_pitch = mx_scale_bytes(k); prm.xs = x_scales; prm.ws = w_scales;
    prm.bias = bias; prm.out = out; prm.act = act; prm.error_word = error_word;
#define CALL(KIND) launch_mx_linear<KIND>(s, x, w, x_tiles, w_tiles, prm, sm_count)
    return MX_KINDS(dtype, CALL);
#undef CALL
}

// Slices of the rows for the plain kernel: at least one pass of all warps each.
static int mx_small_slices(int64_t rows) {
    int s = 1;
    while (s < 8 && rows >= (int64_t)s * 2 * MX_SMALL_FLIGHT * 32) s *= 2;
    return s;
}
// Where the plain kernel is the faster one: its blocks get an SM each and its warps pass over the rows once or twice.
// Measured, FLOAT32: 1024 x 32 x 128 (64 blocks) 15.4 us against 21.5 us on tiles, 1024 x 128 x 128 (256) 21.6 and 21.3,
// 65536 x 32 x 32 (32 blocks, 32 passes) 99 and 43.
static bool mx_gradient_small(int64_t rows, int64_t n, int64_t k, int sm_count) {
    const int64_t s = mx_small_slices(rows), blocks = mx_blocks(k) * ((n + MX_SMALL_N - 1) / MX_SMALL_N) * s;
    return rows > 0 && blocks <= sm_count && rows <= 2 * s * MX_SMALL_FLIGHT * 32;
}

template <int KIND>
static cudaError_t launch_mx_gradient_small(cudaStream_t s, int64_t rows, int64_t n, int64_t k, const uint8_t *codes, const uint8_t *scales, const void *g, float *out) {
    using T = typename MxElement<KIND>::type;
    const int slices = mx_small_slices(rows);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(mx_blocks(k) * slices), (unsigned)((n + MX_SMALL_N - 1) / MX_SMALL_N));
    cfg.blockDim = dim3(MX_SMALL_THREADS);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)slices, 1, 1};
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, mx_weight_gradient_small_kernel<KIND>, rows, (int)n, (int)k, codes, scales, mx_code_bytes(8, k), mx_scale_bytes(k), (const T *)g, out, slices);
}

// How the tiles are spread over the block pairs, and what scratch that takes.
struct MxGradPlan {
    int pieces, tiles_n, tiles, whole_tiles, slices, stages, stages_per_slice;
    bool direct;                        // BFLOAT16 rows that TMA can address are read where they are
    int64_t g_pitch, g_bytes, x_bytes, partial_bytes;       // of the planes and partial sums, each a multiple of 256
};
static MxGradPlan mx_gradient_plan(DType dtype, int64_t rows, int64_t n, int64_t k, bool aligned, int sm_count) {
    MxGradPlan p = {};
    p.pieces = dtype == DType::F32 ? 3 : dtype == DType::BF16 ? 1 : 2;
    const int tiles_k = (int)((k + 255) / 256);
    p.tiles_n = (int)((n + 255) / 256); p.tiles = p.tiles_n * tiles_k;
    p.stages = (int)((rows + MX_ROWS - 1) / MX_ROWS);
    const int pairs = sm_count / 2 > 0 ? sm_count / 2 : 1;
    p.whole_tiles = p.tiles / pairs * pairs;
    // Tiles left over: the number of slices with the least estimated time.  A stage takes 0.3 us per piece, a unit's start
    // and end about 1.5 us, the last launch 3 us and 0.1 us per slice of a tile (512 KB to write and read).
    const int left = p.tiles - p.whole_tiles;
    p.slices = 1;
    double best = 1e300;
    for (int s = 1; left > 0 && s <= 64 && s <= p.stages; s++) {
        const int per = (p.stages + s - 1) / s;
        if ((p.stages + per - 1) / per != s) continue;          // some slice would be empty
        const double cost = (double)(((int64_t)left * s + pairs - 1) / pairs) * (0.3 * p.pieces * per + 1.5) + (s > 1 ? 3.0 + 0.1 * left * s : 0.0);
        if (cost < best) { best = cost; p.slices = s; }
    }
    if (p.slices == 1) p.whole_tiles = p.tiles;
    p.stages_per_slice = p.stages > 0 ? (p.stages + p.slices - 1) / p.slices : 0;
    const auto rounded = [](int64_t bytes) { return (bytes + 255) / 256 * 256; };
    p.g_pitch = (n + 7) / 8 * 8;
    p.direct = dtype == DType::BF16 && n % 8 == 0 && aligned;
    p.g_bytes = p.direct ? 0 : rounded(p.pieces * rows * p.g_pitch * 2);
    p.x_bytes = rounded(rows * mx_code_bytes(8, k) * 2);
    p.partial_bytes = p.slices > 1 ? (int64_t)left * p.slices * 65536 * 4 : 0;
    return p;
}

int64_t mx_weight_gradient_workspace(DType dtype, int64_t rows, int64_t n, int64_t k, bool aligned, int sm_count) {
    if (mx_gradient_small(rows, n, k, sm_count)) return 0;
    const MxGradPlan p = mx_gradient_plan(dtype, rows, n, k, aligned, sm_count);
    return p.g_bytes + p.x_bytes + p.partial_bytes;
}
int mx_weight_gradient_launches(DType dtype, int64_t rows, int64_t n, int64_t k, int sm_count) {
    return rows == 0 || mx_gradient_small(rows, n, k, sm_count) ? 1 : mx_gradient_plan(dtype, rows, n, k, true, sm_count).slices > 1 ? 3 : 2;
}

// Tensor map over BFLOAT16 planes [planes][rows][pitch] of `cols` columns: boxes of 64 columns x 64 rows, 128-byte swizzle.
static bool make_piece_map(CUtensorMap *map, const void *base, int64_t planes, int64_t rows, int64_t cols, int64_t pitch) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    cuuint64_t strides[2] = {(cuuint64_t)pitch * 2, (cuuint64_t)(rows * pitch) * 2};
    cuuint32_t box[3] = {64, MX_ROWS, 1};
    cuuint32_t elem[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, planes > 0 ? 3 : 2, const_cast<void *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tensor map over dense FLOAT32 [rows, cols]: boxes of 32 x 32, 128-byte swizzle.
static bool make_result_map(CUtensorMap *map, const void *base, int64_t rows, int64_t cols) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)cols * 4};
    cuuint32_t box[2] = {32, 32};
    cuuint32_t elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int PIECES>
static cudaError_t launch_mx_gradient(cudaStream_t s, const CUtensorMap &map_g, const CUtensorMap &map_x, const CUtensorMap &map_out, const CUtensorMap &map_partial, const MxGrad &prm, int sm_count) {
    using Cfg = MxGradConfig<PIECES>;
    // the register split draws on what the block was launched with
    static std::atomic<uint64_t> done{0};
    cudaError_t e = mx_prepare_kernel(mx_weight_gradient_kernel<PIECES>, Cfg::kSmemBytes, (72 + 2 * 216 + 2) / 3, done);
    if (e != cudaSuccess) return e;
    const int pairs = sm_count / 2;
    return mx_launch_dependent(mx_weight_gradient_kernel<PIECES>, dim3((unsigned)(2 * (prm.units < pairs ? prm.units : pairs))), MX_GRAD_THREADS, Cfg::kSmemBytes, s, map_g, map_x, map_out, map_partial, prm);
}

template <int KIND>
static cudaError_t launch_mx_pieces(cudaStream_t s, const void *g, int64_t rows, int64_t n, const MxGradPlan &p, uint16_t *g_planes,
                                    const uint8_t *codes, const uint8_t *scales, int64_t x_pitch, int64_t scale_pitch, uint16_t *x_plane) {
    using T = typename MxElement<KIND>::type;
    // blocks in proportion to the bytes moved
    const int64_t g_work = p.direct ? 0 : rows * p.g_pitch / 8, x_work = rows * x_pitch / 8;
    const int64_t most = 148 * 8;
    const double share = (double)g_work * (sizeof(T) + 2.0 * p.pieces) / ((double)g_work * (sizeof(T) + 2.0 * p.pieces) + (double)x_work * 3.0);
    const auto blocks = [&](int64_t work, double part) {
        const int64_t want = (work + MX_THREADS - 1) / MX_THREADS, limit = (int64_t)(most * part) < 1 ? 1 : (int64_t)(most * part);
        return (int)(want < limit ? want : limit);
    };
    const int g_blocks = g_work ? blocks(g_work, share) : 0, x_blocks = blocks(x_work, 1.0 - share);
    const bool vec = n % 8 == 0 && (uintptr_t)g % (8 * sizeof(T)) == 0;
    if (vec) mx_pieces_kernel<KIND, true><<<g_blocks + x_blocks, MX_THREADS, 0, s>>>((const T *)g, rows, n, p.g_pitch, g_planes, g_blocks, codes, scales, x_pitch, scale_pitch, x_plane);
    else mx_pieces_kernel<KIND, false><<<g_blocks + x_blocks, MX_THREADS, 0, s>>>((const T *)g, rows, n, p.g_pitch, g_planes, g_blocks, codes, scales, x_pitch, scale_pitch, x_plane);
    return cudaGetLastError();
}

cudaError_t mx_weight_gradient(cudaStream_t s, DType dtype, int64_t rows, int64_t n, int64_t k, const uint8_t *codes, const uint8_t *scales,
                               const void *g, float *out, void *workspace, int sm_count, int *error_word) {
    if (n == 0 || k == 0) return cudaSuccess;
    if (rows == 0) return cudaMemsetAsync(out, 0, (size_t)n * k * 4, s);
    if (mx_gradient_small(rows, n, k, sm_count)) {
#define CALL(KIND) launch_mx_gradient_small<KIND>(s, rows, n, k, codes, scales, g, out)
        return MX_KINDS(dtype, CALL);
#undef CALL
    }
    if (sm_count < 2 || !workspace) return cudaErrorInvalidValue;
    const MxGradPlan p = mx_gradient_plan(dtype, rows, n, k, ((uintptr_t)g & 15) == 0, sm_count);
    const int64_t x_pitch = mx_code_bytes(8, k), units = p.whole_tiles + (int64_t)(p.tiles - p.whole_tiles) * p.slices;
    if (units >= (1ll << 30)) return cudaErrorInvalidValue;
    uint16_t *g_planes = (uint16_t *)workspace, *x_plane = (uint16_t *)((uint8_t *)workspace + p.g_bytes);
#define CALL(KIND) launch_mx_pieces<KIND>(s, g, rows, n, p, g_planes, codes, scales, x_pitch, mx_scale_bytes(k), x_plane)
    cudaError_t e = MX_KINDS(dtype, CALL);
#undef CALL
    if (e != cudaSuccess) return e;
    CUtensorMap map_g, map_x;
    if (!make_piece_map(&map_g, p.direct ? g : g_planes, p.pieces, rows, n, p.direct ? n : p.g_pitch) || !make_piece_map(&map_x, x_plane, 0, rows, x_pitch, x_pitch)) return cudaErrorInvalidValue;
    MxGrad prm = {};
    prm.n = (int)n; prm.k = (int)k;
    prm.tiles_n = p.tiles_n; prm.whole_tiles = p.whole_tiles; prm.units = (int)units;
    prm.slices = p.slices; prm.stages = p.stages; prm.stages_per_slice = p.stages_per_slice;
    prm.out = out; prm.partial = (float *)((uint8_t *)workspace + p.g_bytes + p.x_bytes); prm.error_word = error_word;
    CUtensorMap map_out = map_x, map_partial = map_x;           // unused where they are not made
    prm.staged = k % 4 == 0 && ((uintptr_t)out & 15) == 0 && make_result_map(&map_out, out, n, k);
    if (p.slices > 1 && !make_result_map(&map_partial, prm.partial, (units - p.whole_tiles) * 256, 256)) return cudaErrorInvalidValue;
    e = p.pieces == 3 ? launch_mx_gradient<3>(s, map_g, map_x, map_out, map_partial, prm, sm_count) : p.pieces == 2 ? launch_mx_gradient<2>(s, map_g, map_x, map_out, map_partial, prm, sm_count) : launch_mx_gradient<1>(s, map_g, map_x, map_out, map_partial, prm, sm_count);
    if (e != cudaSuccess || p.slices == 1) return e;
    return mx_launch_dependent(mx_add_slices_kernel, dim3(65536 / 4 / MX_THREADS, (unsigned)(p.tiles - p.whole_tiles)), MX_THREADS, 0, s, prm);
}

}  // namespace kern
}  // namespace syn
