// token_step.cuh - what the token-step kernels share: the error word, cluster
// launches, and the checks of cache descriptors.
#pragma once

#include "common.cuh"

namespace tadma_b200 {

// The address of the error word on the current device: gather.cu has it, and
// the kernels of other units take it as a parameter, so that
// tadma_b200_error_flags has one word to copy.
cudaError_t error_word(uint32_t** word);

// launch_pdl with clusters of `cluster` CTAs along the grid's x.
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl_cluster(void (*kernel)(KArgs...), dim3 grid, int cluster, dim3 block, size_t smem,
                               cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// One half (keys or values) of a 4-bit cache as the kernels address it.
struct Kv4View {
    uint8_t* codes;
    __half2* params;
    int64_t c_page, c_head, c_tok;  // codes strides, bytes
    int64_t p_page, p_head, p_tok;  // params strides, (scale, minimum) pairs
};

// Sizes of a cache, one for keys and values.
struct Kv4Dims {
    int64_t pages = 0;
    int heads = 0, page = 0, dim = 0, groups = 0;
};

// Checks the codes / params descriptors of one half and fills its view; sets
// `d` when `first`, compares with it otherwise.  Returns TADMA_OK or fails.
int check_kv4(const tadma_tensor* codes, const tadma_tensor* params, const char* name, bool first, Kv4Dims& d,
              Kv4View& v);

// A 1-D int32 operand.
struct IntVec {
    int32_t* p;
    int64_t stride;
};

}  // namespace tadma_b200
