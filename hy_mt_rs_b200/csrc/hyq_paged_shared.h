// Attention of groups with shared prefixes (hyq_paged_shared.cu).
#pragma once

#include "hyq_paged.cuh"

namespace hyq {
namespace paged {

size_t shared_workspace_bytes(int heads, int dim, int64_t tokens);
// a.groups: start, shared, n and max_new; the rest is set here.
bool worth_sharing(const AttendArgs& a, Kv kv, int64_t groups, int64_t max_shared);
bool shared_supported(const AttendArgs& a, Kv kv);
cudaError_t launch_shared(const AttendArgs& a, Kv kv, cudaStream_t st);

}  // namespace paged
}  // namespace hyq
