// One block of MXFP4: values in, codes and scale out (device helpers).
#pragma once

#include "iqk_common.cuh"

namespace iqk {

// Eight consecutive values as loaded, and as f32.
template <typename T> struct Raw8 {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_float<T>(e[j]);
    }
    // The largest magnitude's f32 bits (NaN above infinity above numbers):
    // 16-bit types compare two magnitudes at a time.
    __device__ __forceinline__ uint32_t peak() const {
        if constexpr (sizeof(T) == 4) {
            const uint32_t *b = reinterpret_cast<const uint32_t *>(w);
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, b[j] & 0x7fffffffu);
            return m;
        } else {
            constexpr uint32_t kSize = 0x7fff7fffu;
            const uint32_t m2 = __vmaxu2(__vmaxu2(w[0].x & kSize, w[0].y & kSize),
                                         __vmaxu2(w[0].z & kSize, w[0].w & kSize));
            const uint16_t m = (uint16_t)max(m2 & 0xffffu, m2 >> 16);
            return __float_as_uint(to_float<T>(*reinterpret_cast<const T *>(&m))) & 0x7fffffffu;
        }
    }
};

// Row and column of an item that moves on by a fixed number of items: no
// division after the first.
template <typename I> struct Walk {
    I row, col, per, rows_on, cols_on;
    __device__ __forceinline__ Walk(I at, I per_row, I step)
        : row(at / per_row), col(at % per_row), per(per_row), rows_on(step / per_row),
          cols_on(step % per_row) {}
    __device__ __forceinline__ void next() {
        row += rows_on;
        col += cols_on;
        if (col >= per) {
            col -= per;
            ++row;
        }
    }
};
template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T *p, Raw8<T> &r) {
    if constexpr (WIDE) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j) r.w[j] = reinterpret_cast<const uint4 *>(p)[j];
    } else {
        T *e = reinterpret_cast<T *>(r.w);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = p[j];
    }
}
template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
    Raw8<T> r;
    load8<T, WIDE>(p, r);
    r.get(v);
}

// Two values to two codes, `lo` in the low nibble.
__device__ __forceinline__ uint32_t codes8(const float (&v)[8], float inv) {
    uint32_t r;
    asm("{\n .reg .b8 a, b, c, d;\n"
        " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n"
        " cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
        " cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        " mov.b32 %0, {a, b, c, d};\n}\n"
        : "=r"(r)
        : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv),
          "f"(v[5] * inv), "f"(v[6] * inv), "f"(v[7] * inv));
    return r;
}

// The scale byte of a block whose magnitudes' largest bit pattern is `amax`,
// and the factor that its values are multiplied with.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax, float &inv) {
    const uint32_t field = amax >> 23;  // floor(log2) + 127; 255: NaN or infinity
    const uint32_t byte = field <= 2u ? 0u : field - 2u;
    inv = __uint_as_float((254u - byte) << 23);
    return field == 255u ? 255u : byte;
}

}  // namespace iqk
