// paged_rope.cuh -- the rotation of rows of heads as a device function: the
// whole of fo_rope's kernel (rope.cu) and the queries' part of the paged
// append (paged_append.cu).
#pragma once

#include "paged.cuh"

namespace fo {

constexpr int ROPE_THREADS = 256;
// Heads a thread takes with one read of its table entries: 64 or 128 bytes of
// loads in flight for each thread.
template <typename T, bool HALF>
__host__ __device__ constexpr int rope_heads() {
    return sizeof(T) == 4 && HALF ? 2 : 4;
}

// Work of one row: a slot is eight adjacent elements of a head (interleaved
// layout, and elements that pass unrotated), or eight pairs (half layout:
// two groups of eight elements rot_dim / 2 apart); without 16-byte alignment
// (VEC false) one pair or one passing element.
__host__ __device__ inline int rope_slots(const fo_rope_launch &a, bool vec, bool half) {
    const int rot = a.rope.rot_dim, pass = a.in_place ? 0 : a.head_dim - rot;
    if (!vec) return rot / 2 + pass;
    return half ? rot / 16 + pass / 8 : (rot + pass + 7) / 8;
}

// Chooses between whole 16-byte groups and single elements, and the block's
// width; returns whether groups are used.
inline bool rope_shape(fo_rope_launch *a) {
    const int64_t unit = a->x.dtype == FO_DT_F32 ? 4 : 8;  // elements in 16 bytes
    auto ok = [&](const fo_rows &r) {
        return (reinterpret_cast<uintptr_t>(r.data) & 15) == 0 && r.row_stride % unit == 0 && r.head_stride % unit == 0;
    };
    const bool half = a->rope.layout == FO_ROPE_HALF;
    const bool vec = ok(a->x) && ok(a->out) && a->head_dim % 8 == 0 && (!half || a->rope.rot_dim % 16 == 0);
    a->slots = rope_slots(*a, vec, half);
    const int heads = a->x.dtype == FO_DT_F32 && half ? rope_heads<float, true>() : rope_heads<uint16_t, false>();
    a->head_blocks = (a->x.heads + heads - 1) / heads;
    const int64_t width = (int64_t)a->slots * a->head_blocks;
    a->block_x = (int)(width < ROPE_THREADS ? (width < 1 ? 1 : width) : ROPE_THREADS);
    return vec;
}

// Block `block` of the rotation, thread t of ROPE_THREADS; `position(row, padded)` gives a row's
// position, or sets padded (the row is copied as it is).
template <typename T, bool HALF, bool VEC, typename Position>
__device__ __forceinline__ void rope_block(const fo_rope_launch &a, int64_t block, int t, Position position) {
    // block_x threads over (head block, slot), the others over rows.
    const int rows_per_block = ROPE_THREADS / a.block_x;
    const int ty = t / a.block_x, tx = t - ty * a.block_x;
    const int64_t row = block * rows_per_block + ty;
    if (ty >= rows_per_block || row >= a.rows) return;
    constexpr int HEADS = rope_heads<T, HALF>();
    const int rot = a.rope.rot_dim, h2 = rot / 2;
    const T *xr = static_cast<const T *>(a.x.data) + row * a.x.row_stride;
    T *yr = static_cast<T *>(a.out.data) + row * a.out.row_stride;
    // A row's table entries: looked up behind the first loads of its elements,
    // which do not wait for its position.
    const float2 *entries = nullptr;
    bool inside = false, padded = false;
    auto look_up = [&]() {
        if (entries) return;
        const int64_t p = position(row, padded);
        inside = p >= 0 && p < a.rope.positions;
        if (!inside && !padded && tx == 0) atomicOr(a.err, FO_DEVERR_POSITION);
        entries = reinterpret_cast<const float2 *>(a.rope.table) + (inside ? p : 0) * h2;
    };
    auto entry = [&](int pair) {
        float2 cs = load_entry(entries + pair);
        if (!inside) cs = padded ? make_float2(1.0f, 0.0f) : make_float2(NAN, NAN);
        if (a.transpose) cs.y = -cs.y;
        return cs;
    };
    const int width = a.slots * a.head_blocks;
    for (int w = tx; w < width; w += a.block_x) {
        // Heads hb, hb + head_blocks, ..: neighbouring threads take neighbouring
        // heads.
        const int hb = w / a.slots, slot = w - hb * a.slots;
        if constexpr (VEC) {
            const bool pairs = HALF && slot < rot / 16;  // eight pairs: two groups of eight elements
            const int d = !HALF || pairs ? slot * 8 : rot + (slot - rot / 16) * 8;
            Raw8<T> r0[HEADS], r1[HEADS];
#pragma unroll
            for (int k = 0; k < HEADS; k++) {
                const int h = hb + k * a.head_blocks;
                if (h < a.x.heads) {
                    r0[k] = load_raw8(xr + h * a.x.head_stride + d);
                    if (HALF && pairs) r1[k] = load_raw8(xr + h * a.x.head_stride + d + h2);
                }
            }
            float2 cs[HALF ? 8 : 4];
            if (d < rot) {
                look_up();
#pragma unroll
                for (int e = 0; e < (HALF ? 8 : 4); e++)
                    cs[e] = HALF || d + 2 * e < rot ? entry(HALF ? d + e : d / 2 + e) : make_float2(1.0f, 0.0f);
            }
#pragma unroll
            for (int k = 0; k < HEADS; k++) {
                const int h = hb + k * a.head_blocks;
                if (h >= a.x.heads) break;
                T *to = yr + h * a.out.head_stride + d;
                float x[8], y[8];
                unpack8(r0[k], x);
                if (d >= rot) {
                    store8(to, x);
                } else if constexpr (HALF) {
                    float z[8];
                    unpack8(r1[k], z);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        y[e] = rot_first(x[e], z[e], cs[e]);
                        z[e] = rot_second(x[e], z[e], cs[e]);
                    }
                    store8(to, y);
                    store8(to + h2, z);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool turn = d + 2 * e < rot;  // a passing element keeps its value
                        y[2 * e] = turn ? rot_first(x[2 * e], x[2 * e + 1], cs[e]) : x[2 * e];
                        y[2 * e + 1] = turn ? rot_second(x[2 * e], x[2 * e + 1], cs[e]) : x[2 * e + 1];
                    }
                    store8(to, y);
                }
            }
        } else {
            look_up();
            const bool pair = slot < h2;
            const int d0 = !pair ? rot + slot - h2 : HALF ? slot : 2 * slot;
            const int d1 = HALF ? slot + h2 : 2 * slot + 1;
            const float2 cs = pair ? entry(slot) : make_float2(1.0f, 0.0f);
            for (int h = hb; h < a.x.heads; h += a.head_blocks) {
                const float u = load1(xr + h * a.x.head_stride + d0);
                if (pair) {
                    const float v = load1(xr + h * a.x.head_stride + d1);
                    store1(yr + h * a.out.head_stride + d0, rot_first(u, v, cs));
                    store1(yr + h * a.out.head_stride + d1, rot_second(u, v, cs));
                } else {
                    store1(yr + h * a.out.head_stride + d0, u);
                }
            }
        }
    }
}

}  // namespace fo
