// Tree attention, float32 (tree_attention.cu says what is computed and how): products in two terms on the tensor cores.
#include "tree_attention_tiles.cuh"

namespace {

template <int DP>
int by_rows(const Args* a, long long pages, int tile_rows, int wide, int* info, cudaStream_t stream) {
    if (tile_rows == 16) {
        if constexpr (DP <= 64) {
            if (wide == 1) TREE_GO(float, 1, 8, 32, 1, 1);
            if (!wide) TREE_GO(float, 1, 4, 32, 1, 3);
        } else if constexpr (DP == 128) {
            if (wide == 1) TREE_GO(float, 1, 6, 32, 1, 1);
            if (!wide) TREE_GO(float, 1, 3, 32, 1, 2);
        } else {
            if (!wide) TREE_GO(float, 1, 3, 32, 1, 1);
        }
    }
    return mllm_fail(1, "tree_attention: no kernel takes tiles of %d rows (variant %d)", tile_rows, wide);
}

}  // namespace

int tree::f32(const Args* a, int dh, long long pages, int tile_rows, int wide, int* info, cudaStream_t stream) {
    if (dh <= 32) return by_rows<32>(a, pages, tile_rows, wide, info, stream);
    if (dh <= 64) return by_rows<64>(a, pages, tile_rows, wide, info, stream);
    if (dh <= 128) return by_rows<128>(a, pages, tile_rows, wide, info, stream);
    return by_rows<256>(a, pages, tile_rows, wide, info, stream);
}
int tree::bind_error_f32(int* word) { return tc::bind_host_error(word); }
int tree::error_f32(int* code) {
    int zero = 0;
    MLLM_CUDA(cudaMemcpyFromSymbol(code, g_tiles_error, sizeof(int)));
    if (*code) MLLM_CUDA(cudaMemcpyToSymbol(g_tiles_error, &zero, sizeof(int)));
    return 0;
}
