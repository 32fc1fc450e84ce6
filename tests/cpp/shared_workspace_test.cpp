// What the C++ mirror does with the workspace of shared-prefix attention when it is reserved again, on the CPU: the CUDA calls
// and the library are stand-ins that record. A captured graph keeps the address that it was captured with, so no
// workspace that was handed to a launch may be freed while the object lives. Exit code 0 = pass.
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>

#include "talker_attention_b200.hpp"

static std::set<void*> alive;
static std::vector<void*> launched;            // workspaces that launches were given
static std::vector<int64_t> launched_bytes;
static int prepared = 0, prepare_answer = QM_OK;

extern "C" {
cudaError_t cudaMalloc(void** p, size_t n) { alive.insert(*p = std::malloc(n)); return cudaSuccess; }
cudaError_t cudaFree(void* p) { if (p) { alive.erase(p); std::free(p); } return cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
const char* qm_last_error_string() { return "stand-in"; }
int32_t qm_validate_b200_device(int32_t, int32_t*) { return QM_OK; }
int32_t qm_kv_pool_create(int32_t, int32_t, int32_t, qm_kv_pool**) { return QM_OK; }
int32_t qm_kv_pool_destroy(qm_kv_pool*) { return QM_OK; }
int32_t qm_rope_table_fill(uint16_t*, uint16_t*, int32_t, int32_t, double, void*) { return QM_OK; }
int64_t qm_decode_workspace_bytes(int32_t, int32_t) { return 16; }
int32_t qm_decode_workspace_init(void*, int64_t, void*) { ++prepared; return prepare_answer; }
int64_t qm_decode_shared_workspace_bytes(const qm_kv_pool*, int32_t batch) { return 100 * (int64_t)batch; }
int32_t qm_decode_attention_shared(qm_kv_pool*, int32_t, const uint16_t*, const int32_t*, const int32_t*, int32_t, int32_t batch, int32_t,
                                   const int32_t*, const int32_t*, int32_t, int32_t, uint16_t*, void* workspace, int64_t bytes, void*) {
    if (!workspace || bytes < 100 * (int64_t)batch) return QM_EINVAL;
    launched.push_back(workspace);
    launched_bytes.push_back(bytes);
    return QM_OK;
}
}

#define NEED(x) do { if (!(x)) { std::fprintf(stderr, "line %d: %s\n", __LINE__, #x); return 1; } } while (0)

int main() {
    {
        qm::TalkerAttentionB200 engine(1, 1, 4, 2, 8, 8, nullptr);
        auto launch = [&](int batch) { engine.launch_attention_shared(0, nullptr, nullptr, nullptr, 1, batch, nullptr, nullptr, 1, 1, nullptr); };
        engine.reserve_shared_prefixes(4);
        launch(4);
        engine.reserve_shared_prefixes(200);       // the launch above may sit in a graph
        launch(200);
        NEED(alive.count(launched[0]) == 1 && alive.count(launched[1]) == 1);
        NEED(launched[0] != launched[1]);
        const int so_far = prepared;
        engine.reserve_shared_prefixes(8);         // covered already
        launch(8);
        NEED(launched[2] == launched[1] && launched_bytes[2] == launched_bytes[1] && prepared == so_far);
        // a workspace that could not be prepared is not used
        prepare_answer = QM_ECUDA;
        bool threw = false;
        try { engine.reserve_shared_prefixes(256); } catch (const std::runtime_error&) { threw = true; }
        NEED(threw);
        launch(200);
        NEED(launched[3] == launched[1]);
        prepare_answer = QM_OK;
        engine.reserve_shared_prefixes(256);
        launch(256);
        NEED(alive.count(launched[0]) == 1 && alive.count(launched[1]) == 1 && alive.count(launched[4]) == 1);
    }
    NEED(alive.empty());
    std::puts("SHARED_WORKSPACE_OK");
    return 0;
}
