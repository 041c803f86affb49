// Attention of groups with shared prefixes (hyq_paged_shared.cu; small calls,
// hyq_paged_line.cu).
#pragma once

#include "hyq_paged.cuh"

namespace hyq {
namespace paged {

size_t shared_workspace_bytes(int heads, int dim, int64_t tokens);
// a.groups: start, shared and n; the rest is set here.
bool shared_supported(const AttendArgs& a, Kv kv);
cudaError_t launch_shared(const AttendArgs& a, Kv kv, int64_t max_shared, cudaStream_t st);

size_t line_workspace_bytes(int heads, int dim, int64_t tokens);
bool line_supported(const AttendArgs& a, Kv kv);
cudaError_t launch_line(const AttendArgs& a, Kv kv, void* workspace, cudaStream_t st);

}  // namespace paged
}  // namespace hyq
