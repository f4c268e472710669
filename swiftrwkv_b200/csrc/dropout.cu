// Dropout with a mask that is never stored (philox.cuh): y = x scale where kept, 0
// elsewhere; its gradient is the same call on dy.  One pass over memory: a thread
// takes DU blocks of 8 elements DT apart, all loads first, and draws a block's bits
// while they arrive.  16384 x 8192 bf16: 80 us (a copy: 82), 113 instructions per block of 8
// elements (28 at p = 0), 58 of them for its bits; one or two blocks a thread 87 and 90 us.
#include "ckpt8.cuh"
#include "philox.cuh"

namespace rwkv {
namespace {

constexpr int DT = 256, DU = 4;

template <typename T, int MODE>
__global__ void __launch_bounds__(DT) dropout_kernel(const T* x, T* y, int64_t n, const __grid_constant__ Dropout d) {
    // places within the thread block's part in 32 bits: its first unit is a multiple of
    // DT DU, so that no carry leaves the low word of a block's number
    const int64_t u0 = blockIdx.x * (int64_t)(DT * DU), units = n / 8;
    const int mine = (int)min((int64_t)(DT * DU), units - u0);
    x += 8 * u0;
    y += 8 * u0;
    Raw8<T> raw[DU];
#pragma unroll
    for (int j = 0; j < DU; j++) {
        const int u = j * DT + threadIdx.x;
        if (u < mine) raw[j].load(x + 8 * u);
    }
    const DropKey key = drop_key<MODE>(d);
#pragma unroll
    for (int j = 0; j < DU; j++) {
        const int u = j * DT + threadIdx.x;
        if (u >= mine) continue;
        float v[8];
        raw[j].floats(v);
        if constexpr (MODE != DROP_NONE)
            drop_block(v, philox<MODE>(d, key, (uint32_t)u0 + u, (uint32_t)(u0 >> 32)), d);
        store8(y + 8 * u, v);
    }
    // the tensor's last n % 8 elements
    const int t = threadIdx.x;
    if (u0 + DT * DU >= units && t < (int)(n % 8)) {
        const uint4 r = philox<MODE == DROP_STATE ? DROP_STATE : DROP_KEY>(d, key, (uint32_t)units, (uint32_t)(units >> 32));
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
        const int64_t at = 8 * (units - u0) + t;
        const uint32_t bits = w[t / 2] >> 16 * (t & 1) & 0xffffu;
        y[at] = from_f<T>(bits < d.threshold ? 0.f : __fmul_rn(to_f<T>(x[at]), d.scale));
    }
}

}  // namespace
}  // namespace rwkv

using namespace rwkv;

extern "C" int rwkv_dropout(int dtype, const void* x, double p, uint64_t seed, uint64_t offset, const int64_t* state,
                            void* y, int64_t n, rwkv_stream_t stream) {
    const char* fn = "rwkv_dropout";
    RWKV_REQUIRE(valid_dtype(dtype), RWKV_E_DTYPE, "%s: dtype %d", fn, dtype);
    RWKV_REQUIRE(x && y, RWKV_E_NULL, "%s: NULL argument", fn);
    RWKV_REQUIRE(n >= 1 && n <= 1ll << 40, RWKV_E_SHAPE, "%s: n=%lld (1..2^40)", fn, (long long)n);
    RWKV_REQUIRE(p >= 0.0 && p <= 1.0, RWKV_E_SHAPE, "%s: p=%g must be in 0..1", fn, p);
    RWKV_REQUIRE((((uintptr_t)x | (uintptr_t)y) & 15) == 0 && ((uintptr_t)state & 7) == 0, RWKV_E_UNSUPPORTED,
                 "%s: x and y must be 16-byte aligned, state 8-byte", fn);
    const Dropout d = make_dropout(p, 1.0, seed, offset, state);
    return dispatch_dtype(dtype, [&]<typename T>() {
        const int64_t blocks = (n / 8 + DT * DU - 1) / (DT * DU);
        return dispatch_drop(d, [&]<int MODE>() {
            dropout_kernel<T, MODE><<<(unsigned)(blocks ? blocks : 1), DT, 0, (cudaStream_t)stream>>>((const T*)x, (T*)y, n, d);
            return check_launch("dropout_kernel");
        });
    });
}
