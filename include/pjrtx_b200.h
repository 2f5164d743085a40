/* C ABI of the B200 execution backend for PjRTx.
 *
 * This is the boundary a PjRTx runtime binds instead of the Zig `Backend`
 * facade of the Metal backend (src/backend/mlx_metal/backend.zig:91-180) and
 * the private C shim under it (src/backend/mlx_metal/api.h:198-477). Every
 * entry point below names the reference interface it replaces.
 *
 * Conventions (the same as src/backend/mlx_metal/api.cc): functions that return
 * a pointer return NULL on any failure and never throw across the ABI;
 * functions that return int return 1 on success and 0 on failure; after a
 * failure pjrtx_b200_last_error() holds a one-line reason for the calling
 * thread. Arrays returned through `out_outputs` are owned by the caller and
 * released with pjrtx_b200_output_array_destroy (the array) and
 * pjrtx_b200_buffer_destroy (each element). Element-type codes equal the
 * reference's (api.h:107-120); 12..14 are additions.
 */
#ifndef PJRTX_B200_H_
#define PJRTX_B200_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PJRTX_B200_DEVICE_NAME_BYTES 128

enum {
  PJRTX_B200_DTYPE_INVALID = 0,
  PJRTX_B200_DTYPE_U8 = 1,
  PJRTX_B200_DTYPE_F32 = 2,
  PJRTX_B200_DTYPE_PRED = 3,
  PJRTX_B200_DTYPE_S32 = 4,
  PJRTX_B200_DTYPE_U32 = 5,
  PJRTX_B200_DTYPE_S8 = 6,
  PJRTX_B200_DTYPE_F16 = 7,
  PJRTX_B200_DTYPE_BF16 = 8,
  PJRTX_B200_DTYPE_C64 = 9,
  PJRTX_B200_DTYPE_U16 = 10,
  PJRTX_B200_DTYPE_U64 = 11,
  PJRTX_B200_DTYPE_S64 = 12,
  PJRTX_B200_DTYPE_S16 = 13,
  PJRTX_B200_DTYPE_F64 = 14,
};

/* Value roles (src/compiler/executable_plan.zig:17-22). */
enum {
  PJRTX_B200_ROLE_PARAMETER = 0,
  PJRTX_B200_ROLE_CONSTANT = 1,
  PJRTX_B200_ROLE_INSTRUCTION_RESULT = 2,
  PJRTX_B200_ROLE_OUTPUT = 3,
};

/* Sharding kinds (src/compiler/topology.zig:69-73). */
enum {
  PJRTX_B200_SHARDING_REPLICATED = 0,
  PJRTX_B200_SHARDING_PARTITIONED = 1,
  PJRTX_B200_SHARDING_MANUAL = 2,
};

/* Compare directions (src/compiler/operation.zig:46-53, api.h:181-188). */
enum {
  PJRTX_B200_COMPARE_EQ = 0,
  PJRTX_B200_COMPARE_NE = 1,
  PJRTX_B200_COMPARE_GE = 2,
  PJRTX_B200_COMPARE_GT = 3,
  PJRTX_B200_COMPARE_LE = 4,
  PJRTX_B200_COMPARE_LT = 5,
};

typedef struct PjrtxB200Buffer PjrtxB200Buffer;
typedef struct PjrtxB200Plan PjrtxB200Plan;
typedef struct PjrtxB200Executable PjrtxB200Executable;
typedef struct PjrtxB200ExecutionEvent PjrtxB200ExecutionEvent;
typedef struct PjrtxB200AsyncHostToDeviceTransfer PjrtxB200AsyncHostToDeviceTransfer;
typedef struct PjrtxB200DeviceEvent PjrtxB200DeviceEvent;

/* Replaces PjrtxMlxMetalDeviceInfo (api.h:12-18). */
typedef struct PjrtxB200DeviceInfo {
  int32_t ordinal;
  uint64_t registry_id;
  uint64_t memory_bytes;
  uint8_t has_unified_memory;
  char name[PJRTX_B200_DEVICE_NAME_BYTES];
} PjrtxB200DeviceInfo;

/* Replaces device.Capabilities (src/backend/mlx_metal/device.zig:7-25). */
typedef struct PjrtxB200Capabilities {
  const char *name; /* "b200_cuda" */
  uint8_t supports_device_buffers;
  uint8_t supports_unified_memory;
  uint8_t supports_async_execution;
} PjrtxB200Capabilities;

/* One integer-list attribute of an instruction, named as the field of
 * ir.PlanInstruction it stands for (src/compiler/executable_plan.zig:56-128):
 * "dims", "permutation", "broadcast_dimensions", "start_indices",
 * "limit_indices", "strides", "slice_sizes", "dimension", "dimensions",
 * "iota_dimension", "reduce_dimensions", "lhs_batch_dimensions",
 * "rhs_batch_dimensions", "lhs_contracting_dimensions",
 * "rhs_contracting_dimensions", "compare_direction", "index_vector_dim",
 * "offset_dims", "collapsed_slice_dims", "start_index_map",
 * "operand_batching_dims", "start_indices_batching_dims". */
typedef struct PjrtxB200Attribute {
  const char *name;
  const int64_t *values;
  uint64_t count;
} PjrtxB200Attribute;

/* Replaces executable_mod.Stats (src/backend/mlx_metal/executable_stats.zig:6-56);
 * fields that only describe MLX/Metal strategies are dropped, kernel-plan
 * counters are added at the end. */
typedef struct PjrtxB200ExecutableStats {
  uint64_t struct_size;
  uint64_t resident_constant_count;
  uint64_t resident_constant_bytes;
  uint64_t program_value_count;
  uint64_t program_node_count;
  uint64_t program_edge_count;
  uint64_t program_schedule_item_count;
  uint64_t program_subprogram_count;
  uint64_t program_control_flow_count;
  uint64_t program_fusion_group_count;
  uint64_t program_materialization_boundary_count;
  uint64_t program_planned_release_count;
  uint64_t program_planned_release_bytes;
  uint64_t program_peak_live_value_count;
  uint64_t program_peak_live_bytes;
  uint64_t program_device_count;
  uint64_t last_execute_device_index; /* UINT64_MAX before the first execute */
  int32_t last_execute_local_hardware_id; /* -1 before the first execute */
  uint64_t execute_count;
  uint64_t compiled_program_execute_count;
  uint64_t compiled_program_output_count;
  uint64_t captured_program_execute_count;
  uint64_t captured_program_dynamic_input_count;
  uint64_t captured_program_captured_input_count;
  uint64_t donation_alias_output_count;
  uint64_t donation_alias_output_bytes;
  uint64_t fusion_group_execute_count;
  uint64_t execute_wall_us_total;
  uint64_t execute_wall_us_peak;
  uint64_t kernel_step_count;
  uint64_t generated_kernel_count;
  uint64_t arena_bytes;
  uint64_t scratch_bytes;
  uint64_t graph_capture_count;
  uint64_t graph_launch_count;
  uint64_t kernel_launch_total;
  uint64_t profile_event_gap_ns; /* profiled executions: what two event records with nothing between them read */
} PjrtxB200ExecutableStats;

/* Replaces MemoryStats (src/runtime/device_memory.zig:258-304). */
typedef struct PjrtxB200MemoryStats {
  uint64_t bytes_in_use;
  uint64_t peak_bytes_in_use;
  uint64_t host_to_device_bytes;
  uint64_t device_to_host_bytes;
} PjrtxB200MemoryStats;

/* ---- library ----------------------------------------------------------- */
/* api.h:198-201 pjrtx_mlx_metal_version_{major,minor,patch}. */
int pjrtx_b200_version_major(void);
int pjrtx_b200_version_minor(void);
int pjrtx_b200_version_patch(void);
/* pjrtx_metalcpp_last_error (api.h:283). */
const char *pjrtx_b200_last_error(void);
/* Backend.capabilities (backend.zig:92). */
int pjrtx_b200_capabilities(PjrtxB200Capabilities *out);

/* ---- devices ----------------------------------------------------------- */
/* pjrtx_mlx_metal_device_count / copy_devices (api.h:202-204); Backend.enumerateDevices (backend.zig:94-98). */
int pjrtx_b200_device_count(void);
int pjrtx_b200_copy_devices(PjrtxB200DeviceInfo *out_devices, int max_devices);
/* PJRT_Device_MemoryStats source (src/plugin/device_memory.zig:273-309). */
int pjrtx_b200_device_memory_stats(int device_ordinal, PjrtxB200MemoryStats *out);
/* Blocks until everything queued on the device's stream is done (mlx synchronize, api.cc:1512-1520). */
int pjrtx_b200_device_synchronize(int device_ordinal);
/* No counterpart in the reference (its failure tests overwrite buffer readiness on the host,
 * src/runtime/execution_call.zig:355-360). Exercises the path by which a device-side wait that cannot complete is
 * reported: enqueues one CTA that waits, with the bounded wait of the streaming kernels, for a barrier nothing ever
 * completes; after `timeout_ms` (1..1000) it gives up, raises the device's error word (code 31) and returns. The next
 * pjrtx_b200_device_synchronize then returns 0 with "gave up a bounded wait (code 31)" and clears the word; the
 * context stays usable. 1 when enqueued. */
int pjrtx_b200_device_bounded_wait_probe(int device_ordinal, uint32_t timeout_ms);

/* Device-side timing on the stream every buffer and executable of the device uses. The reference measures the same
 * interval on the host around a forced device sync (PJRTX_PROFILE_DEVICE_SYNC, src/backend/mlx_metal/api.cc:65-75,
 * PjrtxMlxMetalProgramExecuteProfile.device_sync_wait_us, api.h:25-32). `record` enqueues an event; `elapsed_ms`
 * waits for `stop` and returns the device time between the two. */
PjrtxB200DeviceEvent *pjrtx_b200_device_event_record(int device_ordinal);
int pjrtx_b200_device_event_elapsed_ms(PjrtxB200DeviceEvent *start, PjrtxB200DeviceEvent *stop, double *out_ms);
void pjrtx_b200_device_event_destroy(PjrtxB200DeviceEvent *event);

/* ---- buffers ----------------------------------------------------------- */
/* pjrtx_mlx_metal_buffer_from_host_typed (api.h:208-211); Backend.bufferFromHost (backend.zig:104-106).
 * The host memory may be reused as soon as the call returns. */
PjrtxB200Buffer *pjrtx_b200_buffer_from_host_typed(int device_ordinal, const void *data, uint64_t byte_size, int dtype,
                                                   const int64_t *dims, uint64_t rank);
/* pjrtx_mlx_metal_buffer_zeros (api.h:223-225); Backend.allocateBuffer (backend.zig:124-126). */
PjrtxB200Buffer *pjrtx_b200_buffer_zeros(int device_ordinal, int dtype, const int64_t *dims, uint64_t rank);
/* pjrtx_mlx_metal_buffer_clone (api.h:233); Backend.cloneBuffer (backend.zig:128). */
PjrtxB200Buffer *pjrtx_b200_buffer_clone(PjrtxB200Buffer *src);
/* pjrtx_mlx_metal_buffer_size (api.h:447). */
uint64_t pjrtx_b200_buffer_size(PjrtxB200Buffer *buffer);
int pjrtx_b200_buffer_dtype(PjrtxB200Buffer *buffer);
uint64_t pjrtx_b200_buffer_rank(PjrtxB200Buffer *buffer);
int pjrtx_b200_buffer_dims(PjrtxB200Buffer *buffer, int64_t *out_dims, uint64_t max_rank);
int pjrtx_b200_buffer_device(PjrtxB200Buffer *buffer);
/* 1 when the buffer's storage was moved into an execution output (donation). */
int pjrtx_b200_buffer_is_donated(PjrtxB200Buffer *buffer);
/* pjrtx_mlx_metal_buffer_copy_to_host (api.h:452-453); Backend.copyToHost (backend.zig:177). Synchronous. */
int pjrtx_b200_buffer_copy_to_host(PjrtxB200Buffer *buffer, void *dst, uint64_t dst_size);
/* pjrtx_mlx_metal_buffer_destroy (api.h:454); Backend.destroyBuffer (backend.zig:179). */
void pjrtx_b200_buffer_destroy(PjrtxB200Buffer *buffer);

/* pjrtx_mlx_metal_async_h2d_{create,write,finish,destroy} (api.h:212-222);
 * Backend.{begin,write,finish,destroy}AsyncHostToDeviceTransfer (backend.zig:108-122). */
PjrtxB200AsyncHostToDeviceTransfer *pjrtx_b200_async_h2d_create(int device_ordinal, int dtype, const int64_t *dims,
                                                                uint64_t rank, uint64_t byte_size);
int pjrtx_b200_async_h2d_write(PjrtxB200AsyncHostToDeviceTransfer *transfer, uint64_t offset, const void *data,
                               uint64_t byte_size);
PjrtxB200Buffer *pjrtx_b200_async_h2d_finish(PjrtxB200AsyncHostToDeviceTransfer *transfer);
void pjrtx_b200_async_h2d_destroy(PjrtxB200AsyncHostToDeviceTransfer *transfer);

/* ---- executable plan ---------------------------------------------------- */
/* The plan is the reference's ir.ExecutablePlan (src/compiler/executable_plan.zig:131-147)
 * built field by field, the way the reference's own backend tests build one
 * (src/backend/mlx_metal/execution_call.zig:147-211). */
PjrtxB200Plan *pjrtx_b200_plan_create(int32_t num_replicas, int32_t num_partitions, const int32_t *device_assignment,
                                      uint64_t device_assignment_count);
void pjrtx_b200_plan_destroy(PjrtxB200Plan *plan);
/* Appends a value; returns its id (== table index) or UINT32_MAX. */
uint32_t pjrtx_b200_plan_add_value(PjrtxB200Plan *plan, int role, int dtype, const int64_t *dims, uint64_t rank);
/* Appends an instruction. `kind` is the reference's PlanInstructionKind tag name
 * (src/compiler/operation.zig:84-168), e.g. "add", "dot_general", "reduce_sum";
 * "all_reduce" / "all_gather" are the collective kinds the tensor-parallel planner adds. */
int pjrtx_b200_plan_add_instruction(PjrtxB200Plan *plan, const char *kind, const uint32_t *inputs, uint64_t input_count,
                                    const uint32_t *outputs, uint64_t output_count, const PjrtxB200Attribute *attributes,
                                    uint64_t attribute_count, const void *literal, uint64_t literal_size,
                                    const char *custom_call_target);
int pjrtx_b200_plan_set_outputs(PjrtxB200Plan *plan, const uint32_t *value_ids, uint64_t count);
/* Sharding of parameter `index` (in parameter order) / output `index`; split_dim = -1 when replicated. */
int pjrtx_b200_plan_set_parameter_sharding(PjrtxB200Plan *plan, uint64_t index, int kind, const char *mesh_name,
                                           int64_t split_dim);
int pjrtx_b200_plan_set_output_sharding(PjrtxB200Plan *plan, uint64_t index, int kind, const char *mesh_name,
                                        int64_t split_dim);
/* donated_parameter_indices and output_aliases (executable_plan.zig:143-144). */
int pjrtx_b200_plan_set_donation(PjrtxB200Plan *plan, const uint32_t *donated_parameter_indices, uint64_t donated_count,
                                 const uint32_t *alias_output_indices, const uint32_t *alias_parameter_indices,
                                 uint64_t alias_count);
/* verifyExecutablePlan (src/compiler/executable_plan_verify.zig:328-449): 1 when valid; otherwise writes the
 * diagnostic line into `out` (truncated to capacity, always NUL terminated) and returns 0. */
int pjrtx_b200_plan_verify(PjrtxB200Plan *plan, char *out, uint64_t capacity);
/* The plan itself as JSON (values, instructions, attributes, constant payloads in hex, shardings, outputs): the
 * inverse of the builder calls above, used to inspect what pjrtx_b200_plan_partition produced. Returns the full length. */
uint64_t pjrtx_b200_plan_describe(PjrtxB200Plan *plan, char *out, uint64_t capacity);
/* Stable cache key of the plan under the current backend state ("pjrtx-<16 hex digits>"): the fields the reference's
 * executable cache hashes (src/runtime/executable_fingerprint.zig:9-140: capabilities name, custom-call registry
 * version, compile options, shardings, donation, values, instructions with attributes, constants, call targets). A host
 * keeps compiled executables under this key. Same text-out convention as plan_describe. */
uint64_t pjrtx_b200_plan_fingerprint(PjrtxB200Plan *plan, char *out, uint64_t capacity);
/* The same key with the target devices mixed in, as the reference hashes the resolved device ids and local hardware ids
 * of the executable's devices (src/runtime/executable_fingerprint.zig:38-56): the key to use with the executable cache,
 * whose acquire refuses a resident executable that was compiled for other devices. */
uint64_t pjrtx_b200_plan_fingerprint_for_devices(PjrtxB200Plan *plan, const int32_t *device_ordinals, uint64_t device_count,
                                                 char *out, uint64_t capacity);
/* Backend program graph (nodes, edges, fusion groups, schedule, liveness) as JSON; needs no device.
 * Returns the full length; writes at most capacity-1 bytes. program_build.build (program_build.zig:10-207). */
uint64_t pjrtx_b200_plan_describe_program(PjrtxB200Plan *plan, char *out, uint64_t capacity);
/* Kernel plan (steps, generated sources, arena size) as JSON; needs no device. 0 on failure. */
uint64_t pjrtx_b200_plan_describe_kernels(PjrtxB200Plan *plan, char *out, uint64_t capacity);
/* Tensor-parallel planner: rewrites a full-size plan whose parameter shardings carry split dimensions into the
 * per-partition plan of `partition` (column/row-parallel contractions, all_reduce after row-parallel ones).
 * New capability on top of the reference's sharding metadata (src/compiler/stablehlo_sharding.zig:40-93). */
PjrtxB200Plan *pjrtx_b200_plan_partition(PjrtxB200Plan *plan, int32_t partition, int32_t num_partitions);

/* ---- compile / execute --------------------------------------------------- */
/* Backend.compileExecutable (backend.zig:130-132). */
PjrtxB200Executable *pjrtx_b200_compile_executable(PjrtxB200Plan *plan, const int32_t *device_ordinals,
                                                   uint64_t device_count);
/* Backend.writeExecutableLoweringDiagnostic (backend.zig:134-136). Returns the full length (0 = no issue). */
uint64_t pjrtx_b200_write_executable_lowering_diagnostic(PjrtxB200Plan *plan, uint64_t device_count, char *out,
                                                         uint64_t capacity);
/* Backend.executeExecutable (backend.zig:138-140); output ownership as pjrtx_mlx_metal_program_execute (api.h:464-476).
 * `out_event` may be NULL. */
int pjrtx_b200_execute_executable(PjrtxB200Executable *executable, uint64_t device_index, PjrtxB200Buffer *const *arguments,
                                  uint64_t argument_count, PjrtxB200Buffer ***out_outputs, uint64_t *out_output_count,
                                  PjrtxB200ExecutionEvent **out_event);
/* pjrtx_mlx_metal_program_output_array_destroy (api.h:477). Frees the array, not the buffers. */
void pjrtx_b200_output_array_destroy(PjrtxB200Buffer **outputs);
/* Backend.executionEventStatus / destroyExecutionEvent (backend.zig:142-144): 0 pending, 1 complete, -1 failed. */
int pjrtx_b200_execution_event_status(PjrtxB200ExecutionEvent *event);
int pjrtx_b200_execution_event_await(PjrtxB200ExecutionEvent *event);
void pjrtx_b200_execution_event_destroy(PjrtxB200ExecutionEvent *event);
/* Backend.executableStats (backend.zig:146). Set out->struct_size before the call. */
int pjrtx_b200_executable_stats(PjrtxB200Executable *executable, PjrtxB200ExecutableStats *out);
uint64_t pjrtx_b200_executable_describe(PjrtxB200Executable *executable, char *out, uint64_t capacity);
/* Per-step device times (the reference's `backend_schedule_item` profile events, src/backend/mlx_metal/
 * profiling_writer.zig:160). While enabled, executions run the step list without graph replay and time every step
 * with a CUDA event pair; step_times copies the latest execution's durations (ms, step order) and returns the
 * step count. */
int pjrtx_b200_executable_set_profiling(PjrtxB200Executable *executable, int enabled);
uint64_t pjrtx_b200_executable_step_times(PjrtxB200Executable *executable, float *out_ms, uint64_t capacity);
/* Backend.destroyExecutable (backend.zig:148). */
void pjrtx_b200_executable_destroy(PjrtxB200Executable *executable);

/* ---- resident-executable cache ----------------------------------------------- */
/* Replaces the runtime's executable residency (src/runtime/executable_cache.zig): compile requests are keyed by
 * fingerprint (pjrtx_b200_plan_fingerprint), a compiled executable stays resident while leased and afterwards until
 * the byte budget or a memory-pressure trim needs its device memory. Victim order among idle entries: most resident
 * bytes, then cheapest to compile, then least recently used, then smaller fingerprint (:284-313). An executable's
 * resident bytes are the device memory it owns (resident constants + arena + contraction scratch). */
typedef struct PjrtxB200ExecutableCache PjrtxB200ExecutableCache;

/* executable_cache.Stats (src/runtime/executable_cache.zig:10-25). */
typedef struct PjrtxB200ExecutableCacheStats {
  uint64_t hits;
  uint64_t misses;
  uint64_t evictions;
  uint64_t evicted_resident_bytes;
  uint64_t resident_entries;
  uint64_t resident_bytes;
  uint64_t peak_resident_bytes;
  uint64_t largest_resident_bytes;
  uint64_t compile_latency_samples;
  uint64_t compile_latency_us_total;
  uint64_t compile_latency_us_peak;
  uint64_t pressure_trim_requests;
  uint64_t pressure_trimmed_bytes;
  uint64_t pressure_trim_failures;
} PjrtxB200ExecutableCacheStats;

/* executable_cache.Trim (:66-73). */
typedef struct PjrtxB200ExecutableCacheTrim {
  uint64_t requested_bytes;
  uint64_t target_resident_bytes;
  uint64_t freed_bytes;
  uint64_t evicted_entries;
  uint64_t remaining_resident_bytes;
  int32_t still_over_capacity;
} PjrtxB200ExecutableCacheTrim;

/* executable_cache.EntrySnapshot (:58-63). */
typedef struct PjrtxB200ExecutableCacheEntry {
  int32_t resident;
  uint64_t resident_bytes;
  uint64_t reference_count;
  uint64_t compile_latency_us;
} PjrtxB200ExecutableCacheEntry;

/* Residency.init / deinit (:333-343). `capacity_bytes` is the device memory that buffers and resident executables
 * share (0 = untracked: no pressure trims). Destroying the cache destroys every resident executable. */
PjrtxB200ExecutableCache *pjrtx_b200_executable_cache_create(uint64_t capacity_bytes);
void pjrtx_b200_executable_cache_destroy(PjrtxB200ExecutableCache *cache);
/* Residency.recordCompile (:346-352): 1 = seen before (hit), 0 = new (miss), -1 = error. */
int pjrtx_b200_executable_cache_record_compile(PjrtxB200ExecutableCache *cache, const char *fingerprint);
/* Residency.acquireBackendExecutable (:379-391, 429-470): leases the resident executable of a recorded fingerprint, or
 * compiles `plan` for the devices, trims idle entries to make room for its device bytes (`out_compile_trim`), and makes
 * it resident with one lease. `*out_reused` = 1 when no compile ran. The executable belongs to the cache: give the lease
 * back with pjrtx_b200_executable_cache_release, never pjrtx_b200_executable_destroy. NULL on failure or for a
 * fingerprint that was never recorded. */
PjrtxB200Executable *pjrtx_b200_executable_cache_acquire(PjrtxB200ExecutableCache *cache, const char *fingerprint,
                                                         PjrtxB200Plan *plan, const int32_t *device_ordinals,
                                                         uint64_t device_count, int *out_reused,
                                                         PjrtxB200ExecutableCacheTrim *out_compile_trim);
/* Residency.release (:394-399): returns one lease; idle entries beyond the byte budget are evicted. */
void pjrtx_b200_executable_cache_release(PjrtxB200ExecutableCache *cache, const char *fingerprint);
/* Residency.setMaxResidentBytes (:366-371). */
void pjrtx_b200_executable_cache_set_max_resident_bytes(PjrtxB200ExecutableCache *cache, uint64_t max_resident_bytes);
/* Residency.trimForAllocation (:374-376, 404-426): `bytes_in_use` = buffer bytes outside the cache. */
int pjrtx_b200_executable_cache_trim_for_allocation(PjrtxB200ExecutableCache *cache, uint64_t bytes_in_use,
                                                    uint64_t allocation_bytes, PjrtxB200ExecutableCacheTrim *out);
/* The capacity that pressure trims work against (the reference's tests set memory.stats.capacity_bytes directly). */
void pjrtx_b200_executable_cache_set_capacity(PjrtxB200ExecutableCache *cache, uint64_t capacity_bytes);
/* Residency.statsSnapshot / entrySnapshot (:355-362). entry returns 0 for an unknown fingerprint. */
int pjrtx_b200_executable_cache_stats(PjrtxB200ExecutableCache *cache, PjrtxB200ExecutableCacheStats *out);
int pjrtx_b200_executable_cache_entry(PjrtxB200ExecutableCache *cache, const char *fingerprint,
                                      PjrtxB200ExecutableCacheEntry *out);
/* Policy-test hooks (the reference's Testing namespaces: setCompileLatencyForTest :167-170, initBorrowedResident):
 * install_placeholder makes a recorded fingerprint resident with one lease and `resident_bytes` of accounted memory
 * but no executable behind it, so the eviction policy runs without a device; it returns 1 when the placeholder became
 * resident, 2 when the fingerprint was resident already (the lease is taken on that entry), 0 on error. */
int pjrtx_b200_executable_cache_install_placeholder(PjrtxB200ExecutableCache *cache, const char *fingerprint,
                                                    uint64_t resident_bytes, uint64_t bytes_in_use,
                                                    PjrtxB200ExecutableCacheTrim *out_compile_trim);
void pjrtx_b200_executable_cache_set_compile_latency(PjrtxB200ExecutableCache *cache, const char *fingerprint,
                                                     uint64_t latency_us);

/* ---- StableHLO text ------------------------------------------------------- */
/* Reads `func.func @main` of a textual StableHLO module into a plan (the subset of operations the backend executes;
 * static shapes; pretty or generic operation syntax). Replaces, for text, the MLIR-based importer
 * (src/compiler/stablehlo_module_import.zig:241-264, stablehlo_operation_import.zig:22-456). NULL on failure with
 * last_error holding one line in the reference's format (src/compiler/stablehlo_decode.zig:117-140):
 *   unsupported op: op=<name> loc=L:C dtype=<t> rank=<r|unknown> sharding=<...> feature=stablehlo-op
 * or, for malformed text, `invalid module: loc=L:C detail="..." feature=stablehlo-text`. */
PjrtxB200Plan *pjrtx_b200_plan_from_stablehlo_text(const char *text, uint64_t length);

/* ---- custom calls -------------------------------------------------------- */
/* Backend.register{Identity,Unary,Binary}CustomCall / unregisterCustomCall / customCallRegistryVersion
 * (backend.zig:150-175). `op_name` is "identity" or an elementwise kind name; arity 1 or 2. */
int pjrtx_b200_register_custom_call(const char *target, const char *op_name, int arity);
void pjrtx_b200_unregister_custom_call(const char *target);
uint64_t pjrtx_b200_custom_call_registry_version(void);

/* ---- tensor-parallel communicator (no counterpart: the reference has no collectives) ---- */
int pjrtx_b200_comm_unique_id(uint8_t out_id[128]);
int pjrtx_b200_comm_init(int device_ordinal, const uint8_t id[128], int rank, int world_size);
void pjrtx_b200_comm_destroy(int device_ordinal);
/* Peer-memory all-reduce (no counterpart in the reference). Optional, after comm_init: every rank calls
 * comm_peer_export (allocates this rank's region and returns its 64-byte CUDA IPC handle), the host ships all handles
 * to all ranks in rank order, every rank calls comm_peer_import with the world_size x 64 bytes; from then on sums of up
 * to world_size x 512 KiB inside executables run as one kernel per rank (reduce-scatter and all-gather through the
 * peers' regions over NVLink) instead of a library collective. All ranks must have exported before any of them executes (the exchange of the handles is that
 * barrier). Ranks are processes on one node, one GPU each, 2..8 of them. 1 on success, 0 with last_error set. */
int pjrtx_b200_comm_peer_export(int device_ordinal, uint8_t out_handle[64]);
int pjrtx_b200_comm_peer_import(int device_ordinal, const uint8_t *handles, int rank, int world_size);

/* ---- contraction without allocation ---------------------------------------- */
/* No counterpart in the reference. out[m, n] = lhs[m, k] . rhs[k, n] for dense row-major device pointers, 1 <= m <= 8,
 * element type f32 / f16 / bf16, n a multiple of 16 bytes' worth of elements, rhs and out 16-byte aligned.
 *
 * For callers that cannot allocate device memory where they need the product: a runtime whose arena already owns all
 * of HBM, code running under another allocator's lock, a serving loop that forbids allocator calls after start-up.
 * The split-K scratch of the streaming kernel (f32 partial sums, per-tile counters) comes from a fixed 8 MiB + 64 KiB
 * array inside the library image, so the call makes no cudaMalloc / cudaFree / pool call. Consequences:
 *  - problems whose scratch does not fit are refused with a message that names the sizes (m <= 8 against rhs up to
 *    4096 x 128256 fits);
 *  - every GPU that loads the library holds the array until the process exits;
 *  - all calls share the array, and it keeps the previous call's contents (the counters and the error word are
 *    cleared on the stream before each launch): two calls that overlap on the GPU race, so keep them on one stream
 *    or order them with events;
 *  - the first call on a device resolves the array's address and raises the kernel's shared-memory limit; make that
 *    first call before any stream capture begins.
 * The caller's current CUDA device is left as it was. `stream` is a cudaStream_t (NULL = the default stream).
 * Returns 1 when the work was enqueued, 0 with pjrtx_b200_last_error() set. */
int pjrtx_b200_dot_static_scratch(int device_ordinal, int dtype, const void *lhs, const void *rhs, void *out, int64_t m,
                                  int64_t k, int64_t n, void *stream);
/* No counterpart in the reference. Completion status of the most recent pjrtx_b200_dot_static_scratch call on the
 * device: waits for `stream`, reads the kernel's error word out of the static array (a 4-byte copy into a stack
 * variable; nothing is allocated) and returns 1 when the kernel ran to completion, 0 with last_error set when one of
 * its bounded device-side waits gave up (the output of that call is then not valid). Ask before the next call on the
 * device: every call clears the word. */
int pjrtx_b200_dot_static_scratch_status(int device_ordinal, void *stream);

/* ---- operators on device memory ---------------------------------------------- */
/* No counterparts in the reference. Operators that a host calls directly, with device pointers and a stream of its own:
 * a paged key-value cache (append, attend, evict) and the scoring of a decoder's logits (log probabilities, entropy,
 * likeliest tokens, and the gradient). They read and write the caller's memory, allocate nothing per call, and enqueue on
 * `stream` (a cudaStream_t; NULL = the default stream); pjrtx_b200_device_stream gives the stream that buffers and
 * executables of a device use, pjrtx_b200_buffer_device_pointer a buffer's memory. That stream is ordered with no other, the
 * default stream included. Buffers are filled and freed on it: a call on another stream that is given a buffer's memory has to
 * be ordered behind the upload, and the buffer's destruction behind the call. The caller's current device is left as it was.
 * Set struct_size of every argument struct to its sizeof. Element types are f32, f16 and bf16; statistics and
 * weights are f32, ids and lengths s32. Strides count elements; the innermost axis is dense.
 * 1 when enqueued, 0 with last_error set. What only the device sees (a page id outside the pool, a length outside the page
 * table, a token id outside the vocabulary) is never followed out of bounds: the kernel skips it and sets a word of its code
 * (40, 41, 42). pjrtx_b200_operators_status waits for the stream of a call and tells. The words are the device's, not the
 * call's: pjrtx_b200_device_synchronize and copies to the host, which wait for the stream of pjrtx_b200_device_stream alone,
 * return 0 for what is set by then, whichever stream it came from, and what has been named once is not named again. */
void *pjrtx_b200_device_stream(int device_ordinal);
/* NULL for a deleted or donated buffer, and for one without elements. */
void *pjrtx_b200_buffer_device_pointer(PjrtxB200Buffer *buffer);

/* A paged cache: keys and values of all sequences in two pools of `num_pages` pages of `page_size` rows. Row t of sequence b
 * is row t % page_size of page page_table[b * table_stride + t / page_size]; entries beyond a sequence's rows are not read.
 * The handle holds geometry and workspaces, not the pools, so one serves all layers of a shape. Calls on one handle share
 * its workspaces: keep them on one stream or order them with events. */
typedef struct PjrtxB200PagedCache PjrtxB200PagedCache;

typedef struct PjrtxB200PagedCacheConfig {
  uint64_t struct_size;
  int32_t dtype;     /* of queries, keys, values and results */
  int32_t track;     /* 1: attend can add up attention weights, evict can go by them (workspace for the scores) */
  int64_t batch;     /* sequences of a call, at most */
  int64_t heads;     /* query heads, a multiple of kv_heads: head h reads KV head h / (heads / kv_heads) */
  int64_t kv_heads;
  int64_t head_dim;  /* up to 256, a multiple of 16 bytes */
  int64_t page_size; /* rows of a page, any number */
  int64_t max_pages; /* pages of a sequence, at most; capacity = page_size * max_pages rows */
} PjrtxB200PagedCacheConfig;

/* What every call is told of the pools and of the batch. Pointers to pages and their strides keep 16-byte alignment. */
typedef struct PjrtxB200PagedView {
  uint64_t struct_size;
  void *k_pages;             /* [num_pages, page_size, kv_heads, head_dim] through the strides, the same for both pools */
  void *v_pages;
  int64_t num_pages;
  int64_t page_stride;
  int64_t row_stride;
  int64_t head_stride;
  const int32_t *page_table; /* [batch, max_pages] */
  int64_t table_stride;
  const int32_t *lengths;    /* [batch]: rows of each sequence, those that the call appends among them; 0 = idle */
  int64_t batch;             /* 0: the call does nothing, and arrays along the batch may be NULL */
  const int32_t *tokens;     /* [batch]: tokens each sequence has seen, the new ones among them; NULL without tracking */
  float *weights;            /* [batch, kv_heads, capacity]: attention weight each row has had; NULL without tracking */
  int32_t *positions;        /* [batch, kv_heads, capacity]: token of each row; NULL without tracking */
} PjrtxB200PagedView;

PjrtxB200PagedCache *pjrtx_b200_paged_cache_create(int device_ordinal, const PjrtxB200PagedCacheConfig *config);
/* Waits for the device, then frees the workspaces. Not while a stream of the process is captured: the wait ends the capture. */
void pjrtx_b200_paged_cache_destroy(PjrtxB200PagedCache *cache);

/* Row lengths[b] - counts[b] + t of sequence b becomes new row t, t < counts[b]. Tracking: weight 0, position
 * tokens[b] - counts[b] + t. */
typedef struct PjrtxB200PagedAppendArgs {
  uint64_t struct_size;
  const void *k_new; /* [batch, rows, kv_heads, head_dim] through the strides */
  const void *v_new;
  int64_t rows;
  int64_t batch_stride;
  int64_t row_stride;
  int64_t head_stride;
  const int32_t *counts; /* [batch], NULL: `rows` for every sequence */
} PjrtxB200PagedAppendArgs;
int pjrtx_b200_paged_cache_append(PjrtxB200PagedCache *cache, const PjrtxB200PagedView *view,
                                  const PjrtxB200PagedAppendArgs *args, void *stream);

/* Attention of one query position per sequence over its rows: out = softmax(scale * q . k) v, lse = ln sum e^(scale * q . k).
 * A sequence without rows gives zeros and -inf, and so do scores that are all -inf. Infinities and NaN in rows that count go on
 * as in the formula, with probabilities below 2^-126 of the largest (f16: 2^-141) as zero; what lies beyond the length enters
 * nothing. With k_new / v_new, row lengths[b] - 1 is taken from there and stored.
 * Tracking: weights[b, g, t] grows by the weights that the query heads of KV head g give row t (a new row's starts with
 * them, its position is tokens[b] - 1). */
typedef struct PjrtxB200PagedAttendArgs {
  uint64_t struct_size;
  const void *q; /* [batch, heads, head_dim] through the strides */
  int64_t q_batch_stride;
  int64_t q_head_stride;
  void *out;     /* the same axes */
  int64_t out_batch_stride;
  int64_t out_head_stride;
  float *lse;    /* [batch, heads], may be NULL */
  const void *k_new; /* [batch, kv_heads, head_dim] through the strides, NULL: the row is in the pool already */
  const void *v_new;
  int64_t new_batch_stride;
  int64_t new_head_stride;
  float scale;
} PjrtxB200PagedAttendArgs;
int pjrtx_b200_paged_cache_attend(PjrtxB200PagedCache *cache, const PjrtxB200PagedView *view,
                                  const PjrtxB200PagedAttendArgs *args, void *stream);

/* Cuts every sequence of more than `keep` rows to `keep`, each KV head by itself: rows of the first `sinks` and the last
 * `recent` tokens stay, then those with the most weight, of equal ones the lower row. The i-th kept row at or beyond `keep`
 * moves into the place of the i-th dropped row before it; the others stay where they are. Rows without a token get weight
 * 0 and position -1. The results may be the view's own arrays, but layers that share an array of lengths need another one for
 * the new lengths, or the first would cut it for all. Pages must not be shared between sequences. */
typedef struct PjrtxB200PagedEvictArgs {
  uint64_t struct_size;
  int64_t keep;   /* at least sinks + recent, and 1 */
  int64_t recent;
  int64_t sinks;
  int32_t *lengths_out;
  float *weights_out;
  int32_t *positions_out;
} PjrtxB200PagedEvictArgs;
int pjrtx_b200_paged_cache_evict(PjrtxB200PagedCache *cache, const PjrtxB200PagedView *view,
                                 const PjrtxB200PagedEvictArgs *args, void *stream);

/* Scores rows of logits. With p = softmax(scale * logits) of a row: log_probs = ln p[token], entropy = -sum p ln p,
 * lse = ln sum e^(scale * logits), and the `top` likeliest ids with their log probabilities, likeliest first, of equal
 * logits the lower id. Logits of -inf rule tokens out; a row of nothing else gives log probabilities and lse of -inf and
 * entropy 0. NaN and +inf make a row's statistics NaN (NaN counts as likeliest). A negative token id: no token, log probability 0. */
typedef struct PjrtxB200TokenLogProbsArgs {
  uint64_t struct_size;
  int32_t dtype;
  int32_t top;           /* 0..64, at most vocab */
  const void *logits;    /* [rows, vocab], rows row_stride elements apart, aligned to the element type */
  int64_t rows;
  int64_t vocab;         /* up to 2^22 */
  int64_t row_stride;
  const int32_t *tokens; /* [rows] */
  float scale;           /* positive: 1 / temperature */
  float *log_probs;      /* [rows] */
  float *entropy;        /* [rows], may be NULL, as may the next three (one of the last two where top > 0) */
  float *lse;            /* [rows] */
  int32_t *top_ids;      /* [rows, top] */
  float *top_log_probs;  /* [rows, top] */
} PjrtxB200TokenLogProbsArgs;
int pjrtx_b200_token_log_probs(int device_ordinal, const PjrtxB200TokenLogProbsArgs *args, void *stream);

/* Gradient of sum_r (grad_log_probs[r] * log_probs[r] + grad_entropy[r] * entropy[r]) by the logits, in their element type.
 * lse and entropy are the forward call's. A ruled-out logit has gradient 0 unless it is the token. */
typedef struct PjrtxB200TokenLogProbsBackwardArgs {
  uint64_t struct_size;
  int32_t dtype;
  float scale;
  const void *logits;
  void *grad_logits;     /* [rows, vocab]; may be the logits, with the same row stride */
  int64_t rows;
  int64_t vocab;
  int64_t row_stride;
  int64_t grad_row_stride;
  const int32_t *tokens;
  const float *lse;
  const float *entropy;        /* with grad_entropy */
  const float *grad_log_probs; /* [rows]; one of the two may be NULL */
  const float *grad_entropy;   /* [rows] */
} PjrtxB200TokenLogProbsBackwardArgs;
int pjrtx_b200_token_log_probs_backward(int device_ordinal, const PjrtxB200TokenLogProbsBackwardArgs *args, void *stream);

/* Waits for `stream`; 1, or 0 with last_error naming what the operators' kernels on the device met since it was last asked
 * (all of codes 40, 41 and 42 that are set). A bounded wait of an executable's kernel that gave up is not among it and stays
 * for pjrtx_b200_device_synchronize. Not during a stream capture. */
int pjrtx_b200_operators_status(int device_ordinal, void *stream);

/* ---- generated-kernel check (no device needed) ---------------------------- */
/* Compiles CUDA source for sm_100a with the run-time compiler; 1 when it compiles. The log goes to `out`. */
int pjrtx_b200_compile_check(const char *source, char *out, uint64_t capacity);

#ifdef __cplusplus
}
#endif

#endif /* PJRTX_B200_H_ */
