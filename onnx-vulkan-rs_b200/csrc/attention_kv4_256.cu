// Attention over the 4-bit cache for heads of 256: see attention_kv4.cuh.
#include "attention_kv4.cuh"

int32_t ovk_kv4_launch_256(ovk_ctx *ctx, const Kv4Args &a, int32_t dtype, int tiles, int ctas)
{
    if (dtype == OVK_FLOAT)
        return tiles == 1 ? kv4::launch<float, 256, 1>(ctx, a, ctas) : kv4::launch<float, 256, 2>(ctx, a, ctas);
    return tiles == 1 ? kv4::launch<__half, 256, 1>(ctx, a, ctas) : kv4::launch<__half, 256, 2>(ctx, a, ctas);
}
