/* Compiled for its assembly: loads to LDS that are written as instructions between the compiler's own ones.  Each has a place of its own. */
#include "expert_tiles.hpp"

extern "C" __global__ void two_places(const uint8_t *p, uint32_t bytes, uint32_t *out)
{
	using namespace ofi_amd;
	__shared__ __attribute__((aligned(1024))) uint8_t own[1024], other[1024];
	auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p), 0, (int)bytes, 0x00020000);
	__builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (lds_void_t *)own, 4, threadIdx.x * 4, 0, 0, 0);
	to_lds(p, (int)bytes, threadIdx.x * 16, other);
	__builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (lds_void_t *)own, 4, threadIdx.x * 4, 0, 256, 0);
	words_to_lds(p, (int)bytes, threadIdx.x * 4, other);
	__builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (lds_void_t *)own, 4, threadIdx.x * 4, 0, 512, 0);
	landed<0>();
	__syncthreads();
	out[threadIdx.x] = own[threadIdx.x] + other[threadIdx.x];
}
