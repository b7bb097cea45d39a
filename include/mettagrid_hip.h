/* mettagrid_hip.h -- C-ABI of the MI355X-native batched MettaGrid step path (libmettagrid_hip.so).
 *
 * Drop-in boundary for the reference's native environment core: the pybind11 class `MettaGrid`
 * (packages/mettagrid/cpp/bindings/mettagrid_c.cpp:998-1093).  One handle owns E independent environments of one
 * game configuration, resident in HBM; `mg_step` advances all of them by one tick.  Plain pointers and sizes only:
 * any host language binds it with its FFI (ctypes stub: metta_amd/native.py; others: INTEGRATION.md).
 *
 * Conventions: every call returns 0 on success, non-zero on error; `mg_last_error()` then describes it
 * (the reference throws std::runtime_error -> Python RuntimeError).  Device pointers returned by `mg_get_buffers`
 * stay valid until `mg_destroy`.  `stream` is a hipStream_t passed as void* (NULL = the default stream); the
 * step/reset calls are asynchronous on it.  A handle is thread-compatible (one caller at a time), no globals.
 */
#ifndef METTAGRID_HIP_H_
#define METTAGRID_HIP_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct mg_handle mg_handle;

/* Device buffers of a handle (reference: the numpy buffers adopted by `MettaGrid::set_buffers`,
 * mettagrid_c.cpp:721-738, and the pufferlib buffer set, pufferlib.py:18-45).  N = num_envs * num_agents. */
typedef struct mg_buffers {
  uint8_t* observations;   /* u8  [N][num_tokens][3]  (location, feature_id, value); 0xFF = empty      */
  float* rewards;          /* f32 [N]                                                                  */
  uint8_t* terminals;      /* u8  [N]  0/1  (numpy bool layout)                                        */
  uint8_t* truncations;    /* u8  [N]  0/1                                                             */
  int32_t* actions;        /* i32 [N]  INPUT: written by the caller before mg_step                     */
  uint8_t* masks;          /* u8  [N]  all ones (reference: `MettaGrid::masks`, mettagrid_c.cpp:983-995) */
  float* episode_rewards;  /* f32 [N]  (reference: `get_episode_rewards`, mettagrid_c.cpp:928-930)      */
  uint8_t* action_success; /* u8  [N]  (reference: `action_success`, mettagrid_c.cpp:955-957)           */
  int32_t num_envs, num_agents, num_tokens, num_actions;
} mg_buffers;

/* Last error message of the calling thread (never NULL). */
const char* mg_last_error(void);

/* Library version / build info string. */
const char* mg_version(void);

/* Resources an inventory of this build can hold: 16 for libmettagrid_hip.so, 32 for libmettagrid_hip_r32.so (the
 * same sources with wider agent records).  The reference takes any `resource_names`
 * (config/mettagrid_config.py:522-535); observation feature ids (uint8) bound it near 60 in practice. */
int mg_max_resources(void);

/* Create E environments from a packed game configuration (the int32 stream of csrc/mg_blob.h, written by
 * metta_amd/compile.py).  Replaces `MettaGrid::MettaGrid(GameConfig, map, seed)` (mettagrid_c.cpp:46-155) for the
 * config part; maps and seeds arrive through mg_set_maps / mg_reset.  `device_id` < 0 = current device. */
int mg_create(const int32_t* cfg_blob, size_t cfg_words, int num_envs, int device_id, mg_handle** out);

/* Upload a pool of P maps, each `height x width` uint8 cell codes (0 = empty; code -> object via the config's cell
 * table), replacing the `list[list[str]]` map argument of the constructor (mettagrid_c.cpp:159-245).  Every map
 * must hold exactly num_agents agent cells.  Object ids / agent ids follow row-major creation order. */
int mg_set_maps(mg_handle* h, const uint8_t* maps, int num_maps, int height, int width);

/* As mg_set_maps for a pool whose maps differ in size (the navigation suite, SURVEY.md §8d config 3: the reference
 * builds one `MettaGrid` per map, each with its own `map_height/map_width`): `maps` holds the P maps back to back,
 * map m being heights[m] x widths[m] row-major.  Everything that depends on the map size (bounds, the compass
 * token's map centre, mettagrid_c.cpp:483-517) uses the size of the map an environment currently plays. */
int mg_set_maps_ragged(mg_handle* h, const uint8_t* maps, int num_maps, const int32_t* heights, const int32_t* widths);

/* Per-map episode length: max_steps[P] (0 = the configuration's `max_steps`), host array; NULL restores the
 * configuration's value for every map.  The reference gives every map of an evaluation suite its own environment
 * config whose only difference is `game.max_steps` (recipes/experiment/navigation.py:32-59, cfg.py NAVIGATION_EVALS);
 * the termination test and the episode-completion token (mettagrid_c.cpp:433-447,667-677) then use the value of the map
 * an environment plays.  Call after mg_set_maps (a new pool clears it). */
int mg_set_map_max_steps(mg_handle* h, const int32_t* max_steps);

/* Per-slot configurations: the device side of `CurriculumEnv` (metta/cogworks/curriculum/curriculum_env.py:96-142), which
 * gives an environment a new `MettaGridConfig` (`set_mg_config`, mettagrid_puffer_env.py) at every episode end.  Here a
 * task is a (configuration, map) pair living in the pool: the handle keeps `num_slots` configuration streams, map slot m
 * plays stream map_cfg[m] (0 at first), and an environment takes up the configuration of the map slot it restarts on.
 * Call before mg_set_maps.  `headroom_words`: extra int32 words per slot for tasks whose stream is longer than the
 * handle's own configuration (< 0: a quarter of it + 64). */
int mg_set_config_slots(mg_handle* h, int num_slots, int headroom_words);

/* Compile a task's configuration (same blob format as mg_create) into slot `slot` and rebuild the episode-start
 * templates of the map slots that play it, stream-ordered after the steps already queued.  The task must agree with
 * the handle's configuration in everything that sizes buffers and observations (agents, resources, actions, object
 * types, feature ids, statistics layout): rewards, limits, initial inventories, protocols, attack costs, max_steps ...
 * may differ, which is what the reference's curricula vary (recipes/prod/arena_basic_easy_shaped.py:60-80).  A task
 * outside the fast kernels' class (attack handlers on the move path, regeneration, ...) moves the handle to the general
 * kernels.  The caller makes sure no environment is on a map slot that plays `slot` (as for mg_refresh_maps: write
 * the idle twin). */
int mg_write_config_slot(mg_handle* h, int slot, const int32_t* cfg_blob, size_t cfg_words, void* stream);

/* The same in two halves, for curricula that hand out a few distinct tasks thousands of times
 * (`CurriculumEnv` draws a task per episode, curriculum_env.py:111-126; with thousands of environments ten episodes end
 * per step): mg_register_config compiles a task ONCE into a device-side registry and returns its id (host-synchronous,
 * the checks and kernel-choice effects of mg_write_config_slot happen here); mg_write_config_slots then copies
 * registered streams into `n` slots with one kernel and rebuilds the templates of the map slots that play them with one
 * more, stream-ordered, no host synchronisation.  Same rule as above: only slots no environment is on. */
int mg_register_config(mg_handle* h, const int32_t* cfg_blob, size_t cfg_words, int32_t* config_id);
int mg_write_config_slots(mg_handle* h, int n, const int32_t* slots, const int32_t* config_ids, void* stream);

/* map_cfg[map_ids[i]] = cfg_slots[i] for i < n, and rebuild those map slots' episode-start templates (host arrays;
 * stream-ordered).  Same rule: only map slots no environment is on. */
int mg_assign_map_configs(mg_handle* h, int n, const int32_t* map_ids, const int32_t* cfg_slots, void* stream);

/* A pool of `num_maps` slots drawn ON THE DEVICE instead of uploaded: replaces the per-episode
 * `map_builder.build()` of the reference's simulator (python/src/mettagrid/simulator/simulator.py:264-267) for its two
 * random builders, which are a border plus one uniform shuffle -- `RandomMapBuilder.build`
 * (map_builder/random_map.py:29-96: one room inside the border) and MapGen's `Random` scene
 * (mapgen/scenes/random.py:19-69: one room per instance).  The map is `height x width`, `fill_code` (0 or a wall
 * type's cell code) everywhere outside the rooms; rooms[n_rooms][4] = (r0, c0, h, w), disjoint; room r receives
 * sym_count[j] cells of code sym_code[j] for j in [room_sym_begin[r], room_sym_begin[r+1]), placed uniformly at random
 * over the room's cells (every arrangement equally likely; numpy's bit stream is not reproduced -- maps are inputs).
 * All rooms together must hold exactly num_agents agent cells.  Slot m of generation g is a function of
 * (seed, g, m) only.  Host arrays; the handle then needs mg_reset like after mg_set_maps. */
int mg_set_generated_maps(mg_handle* h, int height, int width, int fill_code, int n_rooms, const int32_t* rooms,
                          const int32_t* room_sym_begin, const int32_t* sym_code, const int32_t* sym_count, int num_maps,
                          uint64_t seed);

/* Redraw slots of a generated pool, asynchronously on `stream`, without host involvement or allocation: every slot
 * that an episode has used since it was last drawn and that no environment is on now (so a map never changes under
 * an episode), or with `force` != 0 every slot (mg_reset must follow).  The episode-start templates of the redrawn
 * slots are rebuilt in the same stream.  With 2E slots and map_stride E (mg_set_auto_reset) an environment alternates
 * between two slots, and one call per episode length gives every episode a fresh map. */
int mg_refresh_maps(mg_handle* h, int force, void* stream);

/* Replace ONE slot of the pool by a map built on the host (height x width cell codes, as for mg_set_maps): the
 * per-episode `map_builder.build()` of the reference's simulator (python/src/mettagrid/simulator/simulator.py:264-267)
 * for builders that have no device generator (ASCII maps, MapGen scene trees, a curriculum task's own map).  The pool
 * entries of the slot (object cells, spawn / assembler / chest lists, object counts) and its episode-start template are
 * rebuilt on `stream`; nothing else is touched and no environment is reset.  Every map of the pool must have the same
 * size; the map must hold num_agents agents and no more assemblers / chests than the largest map given to
 * mg_set_maps / drawn by mg_set_generated_maps (the pool is sized at that call).  The caller keeps episodes off the
 * slot while writing, as for mg_assign_map_configs: write the slot an environment will enter NEXT.  `cells` is a
 * host array and may be reused on return. */
int mg_write_map_slot(mg_handle* h, int slot, const uint8_t* cells, void* stream);

/* Copy slot `map_id` of a generated pool to the host as height x width cell codes (inspection / parity tests). */
int mg_get_map(mg_handle* h, int map_id, uint8_t* out, void* stream);

/* `MettaGrid.map_height / map_width` (mettagrid_c.cpp:1040-1041) of map `map_id` of the pool. */
int mg_map_dims(mg_handle* h, int map_id, int32_t* height, int32_t* width);

/* (Re)start environments: env_ids[n] (NULL = all E, then n is ignored), each with seeds[i] (std::mt19937 seed of
 * the env, mettagrid_c.cpp:56-57) and map_ids[i] (index into the pool).  Computes the step-0 observations exactly
 * like `_init_buffers` (mettagrid_c.cpp:264-289).  Host arrays. */
int mg_reset(mg_handle* h, const int32_t* env_ids, int n, const uint32_t* seeds, const int32_t* map_ids, void* stream);

/* Advance every environment one tick: `MettaGrid::step` (mettagrid_c.cpp:740-752, 572-678).  Reads the actions
 * buffer in place; invalid action ids are not errors (stat + failed action, :605-608).  With auto-reset enabled an
 * environment whose episode ended on the previous tick is first restarted (same seed, next map of the pool), which
 * is `MettaGridPufferEnv.step` (python/src/mettagrid/envs/mettagrid_puffer_env.py:158-171). */
int mg_step(mg_handle* h, void* stream);

/* As mg_step, but reads the i32[N] actions from `device_actions` (e.g. a policy's output tensor in HBM) instead
 * of the handle's own action buffer -- the device-resident form of `np.copyto(buffers.actions, actions)` in
 * `MettaGridPufferEnv.step` (mettagrid_puffer_env.py:166-169). */
int mg_step_actions(mg_handle* h, const int32_t* device_actions, void* stream);

/* mg_step_actions for n handles in one call: hs[i] steps with device_actions[i] on streams[i].  The handles are the
 * independent environment groups of an asynchronous vecenv (the reference's `async_factor` groups,
 * metta/rl/training/training_environment.py:45-46,151-170; pufferlib vector.py:415-503: each group's step is ordered
 * on its own stream only); one call instead of n keeps the host cost of a step below the kernels' duration when the
 * groups are many and small.  Stops at the first failing handle. */
int mg_step_groups(int n, mg_handle* const* hs, const int32_t* const* device_actions, void* const* streams);

/* Allocation-free step.  No counterpart in the reference: it is for callers that cannot allocate -- code under HIP
 * graph capture, tight serving loops, harnesses that forbid hipMalloc.  Same kernels and results as mg_step /
 * mg_step_actions (`device_actions` NULL = the handle's own action buffer), but the per-step hand-over buffers
 * between the action and the observation kernels (executed action per agent, per-env mode word, pending assembler
 * uses) live in a file-scope device array of the library instead of the handle's own buffers; the call itself
 * performs no hipMalloc / hipFree / allocating library routine.  Limits: num_envs * num_agents <= 131072 and
 * num_envs <= 16384, else an error.  All handles on one GPU share that GPU's array: calls that overlap in time on
 * one GPU (different streams / threads) race; calls on one stream, or serialised by the caller, do not. */
int mg_step_noalloc(mg_handle* h, const int32_t* device_actions, void* stream);

/* Which kernels one mg_step launches for this handle's configuration and map pool (after mg_set_maps): the fused
 * one-launch step for attack-free configurations with at most 64 agents, else the action + observation kernels.
 * No reference counterpart (diagnostic; bench.py names the measured kernel with it). */
const char* mg_step_path(mg_handle* h);

/* Auto-reset policy used by mg_step: enabled (0/1) and how the next map is chosen: map_id += map_stride (mod P). */
int mg_set_auto_reset(mg_handle* h, int enabled, int map_stride);

/* Per-env step at which the FIRST episode is cut by setting all truncations (0 = never): the reference's
 * EarlyResetHandler (python/src/mettagrid/envs/early_reset_handler.py:6-20).  Host array u32[E] or NULL to clear. */
int mg_set_early_reset(mg_handle* h, const uint32_t* steps);

/* Device pointers and shapes. */
int mg_get_buffers(mg_handle* h, mg_buffers* out);

/* `Simulation.end_episode` (simulator.py:134-136): set all truncations of one env (env < 0: all). */
int mg_end_episode(mg_handle* h, int env, void* stream);

/* Episode statistics of one env (reference: `get_episode_stats`, mettagrid_c.cpp:936-953), as raw slots:
 * agent_values f32[A][n_agent_slots], agent_touched u8[A][n_agent_slots], game_values f32[n_game_slots],
 * game_touched u8[n_game_slots]; slot -> key string tables live with the host language (metta_amd/stats.py).
 * Synchronises the stream.  With `last_finished` != 0 returns the stats captured when the env's most recent
 * episode ended (kept across the auto-reset), else the running episode's. */
int mg_episode_stats(mg_handle* h, int env, int last_finished, float* agent_values, uint8_t* agent_touched,
                     float* game_values, uint8_t* game_touched, void* stream);
int mg_stat_slots(mg_handle* h, int* n_agent_slots, int* n_game_slots);

/* `current_stat_reward` of every agent of `env` (Agent::current_stat_reward, agent.hpp:36; exposed by
 * `grid_objects`, mettagrid_c.cpp:831): out f32[A]. */
int mg_agent_stat_reward(mg_handle* h, int env, float* out, void* stream);

/* Chests of `env` (the Chest entries of `MettaGrid::grid_objects`, mettagrid_c.cpp:754-918; chest.hpp:20-147), in
 * row-major map order: out i32[n][5 + 2R] = {r, c, chest config index, object id, n_items, (item, amount) pairs in the
 * inventory's iteration order, -1 padded}.  `*n_chests` receives the count; `out` may be NULL to query it. */
int mg_chest_state(mg_handle* h, int env, int32_t* out, int max_chests, int32_t* n_chests, void* stream);

/* Inspection (reference: `grid_objects`, mettagrid_c.cpp:754-918; `current_step`).  Host outputs; synchronises.
 * agent_state: i32 [A][9 + 2R]: r, c, prev_r, prev_c, frozen, vibe, steps_without_motion, object id, n_items,
 * then (item, amount) pairs in inventory iteration order (unused = -1).
 * assembler_state: i32 [n][8]: r, c, cfg, object id, is_clipped, cooldown_end, cooldown_duration, uses_count. */
int mg_agent_state(mg_handle* h, int env, int32_t* out, void* stream);
int mg_num_assemblers(mg_handle* h, int env);
int mg_assembler_state(mg_handle* h, int env, int32_t* out, void* stream);

/* The Clipper's view of environment `env` (packages/mettagrid/cpp/include/mettagrid/systems/clipper.hpp:19-30:
 * `assembler_infection_weight`, `length_scale`): weights[mg_num_assemblers(h, env)] = infection weight of every assembler
 * in map (row-major) order, 0 for clip-immune ones; *length_scale = the scale in use (the configured one, or the one
 * derived from the map's sparsity, clipper.hpp:65-98).  Inspection / parity tests; synchronises `stream`.  An
 * assembler's clipped state is column 4 of mg_assembler_state: 0 = no, 1 = clipped without an unclipping protocol
 * (it started clipped and no clipper exists), 2 + k = clipped by the clipper with its k-th unclipping protocol. */
int mg_clipper_state(mg_handle* h, int env, uint32_t* weights, int32_t* length_scale, void* stream);
int mg_env_info(mg_handle* h, int env, uint32_t* current_step, int32_t* map_id, uint32_t* seed, uint32_t* episodes,
                void* stream);

/* Error surfacing.  An environment that leaves reference parity (RNG window overflow, a frozen agent on the
 * attack-free fast path, a chest work list overflow) sets bits in its `error` word (mg_env_table column 7); the step
 * kernels OR them into one sticky device word that a caller can read without touching every environment:
 * mg_status_buffer returns u32[4] in HBM = {OR of error bits, finished episodes (count), 0, 0};
 * mg_check_errors synchronises, and fails with a decoded message naming the first offending environment.
 * (Reference: the C++ core throws std::runtime_error out of step(); there is no silent corruption mode.) */
int mg_status_buffer(mg_handle* h, uint32_t** device_ptr, int32_t* n);
int mg_check_errors(mg_handle* h, void* stream);
/* Diagnostic (tests): set the error word of one environment; the next step publishes it like a real fault. */
int mg_debug_inject_error(mg_handle* h, int env, uint32_t bits);

/* All environments' bookkeeping words in one copy: u32 out[E][8] = {current_step, rng index, seed, map_id,
 * episodes finished, pending early-reset step, done flag, error flag}.  (Reference: `current_step`, `_seed`; the
 * episode counter lets a host poll for finished episodes every k steps instead of every step.) */
int mg_env_table(mg_handle* h, uint32_t* out, void* stream);

/* Per-agent episode rewards f32[A] and length of the most recently FINISHED episode of `env`
 * (reference: `get_episode_rewards`, mettagrid_c.cpp:928-930, read by StatsTracker.on_episode_end). */
int mg_finished_rewards(mg_handle* h, int env, float* rewards, uint32_t* steps, void* stream);

/* The episodes that finished between two readings of the finished-episode counter (status word 1, mg_status_buffer),
 * in the order they ended: env_ids[i], map_ids[i] = the environment and the map slot it played, for
 * i < to_count - from_count.  The device keeps the last mg_finished_ring_capacity() entries (>= 16 x num_envs, >= 1024;
 * a larger span is an error: read the newest `capacity` entries and count the rest as lost).  Steps still queued while the
 * copy runs append behind `to_count`; they reach the entries being read only after capacity - (to_count - from_count)
 * more episodes -- and then the call fails instead of returning them: every entry carries its position in the sequence
 * (12 bits), checked against the range asked for.  This replaces a scan over every
 * environment's episode counter (the reference learns of an episode's end from the step call that ends it,
 * mettagrid_puffer_env.py:158-183; here the host polls).  Entries below a counter value the host has read are complete,
 * so the copy runs on `stream` and waits for nothing else: give it a stream of its own, beside the one the steps are
 * queued on (the legacy default stream would make it wait for all of them). */
int mg_finished_ring_capacity(mg_handle* h);
int mg_finished_ring(mg_handle* h, uint32_t from_count, uint32_t to_count, int32_t* env_ids, int32_t* map_ids, void* stream);

/* The same for n environments at once (what `StatsTracker.on_episode_end`, envs/stats_tracker.py:26-107, reads per episode:
 * `get_episode_stats()` + `get_episode_rewards()` of the episode that has just ended): agent_values / agent_touched
 * [n][A][SA], game_values / game_touched [n][SG], rewards [n][A], steps [n], host arrays.  One gather launch and one
 * device -> host copy per 256 environments, so a vecenv that reports several finished episodes per step stays off the
 * critical path. */
int mg_finished_batch(mg_handle* h, int n, const int32_t* env_ids, float* agent_values, uint8_t* agent_touched,
                      float* game_values, uint8_t* game_touched, float* rewards, uint32_t* steps, void* stream);

/* `MettaGrid::set_inventory` (mettagrid_c.cpp:959-965; Agent::set_inventory, agent.cpp:54-72): items/amounts in
 * the iteration order of the converted map (the host language orders them, metta_amd/umap.py). */
int mg_set_inventory(mg_handle* h, int env, int agent, int n, const int32_t* items, const int32_t* amounts, void* stream);

/* Sum over all environments of the finished-episode accumulators since the last call with `clear` != 0:
 * out f64[3 + n_game_slots] = {episodes, sum of episode lengths, sum of per-agent episode reward,
 * sum of game stat slots...}.  This is the vector the multi-GPU path all-reduces. */
int mg_finished_summary(mg_handle* h, double* out, int clear, void* stream);

/* The same accumulator vector in place: f64[*n] in HBM, added to by the step kernels when an episode ends.  A
 * multi-GPU caller all-reduces (a copy of) it on its own stream and zeroes it, without a host round trip. */
int mg_summary_buffer(mg_handle* h, double** device_ptr, int32_t* n);

/* Per-step kernel timing with HIP events recorded on the stream each step kernel is launched on (no host sync in
 * the step call).  mg_set_profiling(h, 1) starts recording (up to 4096 steps); mg_profile_read waits for the
 * recorded steps, writes their durations in milliseconds and restarts recording.  bench.py's roofline line.
 * mg_set_profiling(h, 2) brackets the observation kernel only (SURVEY.md §8d metric 2: obs-encode GB/s). */
int mg_set_profiling(mg_handle* h, int enabled);
/* Record only every `stride`-th step (default 1).  The event pair is not free: on a 90 us step it costs about 7 % of
 * the wall clock, so a benchmark that times itself samples (bench.py: every 8th step of the timed region). */
int mg_set_profiling_stride(mg_handle* h, int stride);
int mg_profile_read(mg_handle* h, float* ms, int max_steps, int* n_steps);

/* Diagnostic (no reference counterpart): enable / read per-environment cycle stamps u64[E][16] of the observation
 * kernel's phases. */
int mg_debug_stamps(mg_handle* h, unsigned long long* out, int enable);

int mg_destroy(mg_handle* h);

/* ---- rollout post-processing ------------------------------------------------------------------
 * V-trace / GAE advantages over [num_rows][horizon] f32 device arrays (row-major, contiguous), on `stream`:
 *   for t = horizon-2 .. 0:  nn = 1 - dones[t+1];  rho = min(importance[t], rho_clip);  c = min(importance[t], c_clip)
 *                            delta = rho * (rewards[t+1] + gamma * values[t+1] * nn - values[t])
 *                            advantages[t] = last = delta + gamma * lambda * c * last * nn
 * advantages[horizon-1] is left as the caller set it.  Replaces `torch.ops.pufferlib.compute_puff_advantage`
 * (packages/pufferlib-core/src/pufferlib/extensions/cuda/pufferlib.cu:7-86; CPU twin extensions/pufferlib.cpp:28-85),
 * whose call site metta/rl/advantage.py:94-97 falls back to a Python loop on ROCm (metta/rl/mps.py:5-41).
 * Bit-identical to the reference's CPU function (sequential per row, no fused multiply-add).  Needs no handle. */
int mg_compute_advantage(const float* values, const float* rewards, const float* dones, const float* importance,
                         float* advantages, float gamma, float lambda, float rho_clip, float c_clip, int num_rows,
                         int horizon, void* stream);

/* ---- recurrent core and action head of a policy ------------------------------------------------------------------
 * Element types of the tensors below (all device memory, columns adjacent, strides in elements). */
#define MG_F32 0
#define MG_BF16 1
#define MG_F16 2

/* Gated linear recurrence over [rows][steps][width], per row and column, with a = sigmoid(gate):
 *   h[t] = a[t] * (resets[t] ? 0 : h[t-1]) + (1 - a[t]) * x[t],  h[-1] = state
 * x and gate are of `type` and may be strided (halves of one projection, time-major views); state f32 [rows][width] and
 * resets u8 [rows][steps] are contiguous and may be NULL (zeros / none). */
typedef struct mg_recurrence {
  const void* x;
  const void* gate;
  const float* state;
  const uint8_t* resets;
  int64_t rows, steps, width;      /* rows * width up to 2^31 */
  int64_t x_row, x_step, gate_row, gate_step;
  void* workspace;                 /* mg_gated_recurrence_workspace bytes of device memory, for this call alone */
  int64_t workspace_bytes;
  int32_t type;
} mg_recurrence;

/* Bytes of workspace that a call with this shape needs, forward or backward (0: none; few columns and many steps). */
int64_t mg_gated_recurrence_workspace(const mg_recurrence* r);

/* The states kept for the backward pass: the one entering every 16th step after step 0. */
#define MG_RECURRENCE_MARK_STEPS 16

/* h [rows][steps][width] of `type` (NULL: only the last state is wanted), last f32 [rows][width], marks f32
 * [rows][(steps - 1) / 16][width] or NULL (no backward pass will follow, or h is f32 and serves as marks).  `last` may
 * be `state` itself where steps is 1.  Nothing is written where rows, steps or width is 0. */
int mg_gated_recurrence(const mg_recurrence* r, void* h, float* last, float* marks, void* stream);

/* Gradients of the above: dh (of `type`, strided) and dlast (f32 [rows][width]) in, each may be NULL (zeros); dx and
 * dgate (of `type`, strided), dstate (f32 [rows][width], may be NULL) out. */
typedef struct mg_recurrence_gradients {
  const void* dh;
  const float* dlast;
  void* dx;
  void* dgate;
  float* dstate;
  int64_t dh_row, dh_step, dx_row, dx_step, dgate_row, dgate_step;
} mg_recurrence_gradients;

/* The state entering step 16 k (k >= 1) of a row is read at marks[row * marks_row + (k - 1) * marks_stride + column]:
 * the marks of the forward pass, or an f32 h at 15 * width. */
int mg_gated_recurrence_backward(const mg_recurrence* r, const float* marks, int64_t marks_row, int64_t marks_stride,
                                 const mg_recurrence_gradients* d, void* stream);

/* Logits [rows][width] of `type` and their controls.  Per row, with c = occurrences of v in its history:
 *   l1 = c > 0 ? (l > 0 ? l / repetition : l * repetition) : l;   l2 = l1 - frequency * c - presence * (c > 0)
 *   adjusted = allowed ? (l2 + bias) / temperature : -infinity
 * allowed: one byte per token (MG_ALLOWED_BOOL) or bit v % 32 of i32 word v / 32 (MG_ALLOWED_BITS); bias f32; history
 * i32, entries outside [0, width) count for nothing.  temperature and repetition: 1e-30 to 1e30.  A row stride of 0
 * shares a control among all rows; NULL: none. */
#define MG_ALLOWED_BOOL 1
#define MG_ALLOWED_BITS 2
/* Rows up to this many tokens are held in registers: their backward pass wants neither stats nor entropy back. */
#define MG_EVALUATE_STATS_WIDTH 1024
typedef struct mg_logits {
  const void* logits;
  const float* bias;
  const void* allowed;
  const int32_t* history;
  int64_t rows;
  int64_t logits_row, bias_row, allowed_row, history_row;
  double temperature, repetition, presence, frequency;
  void* workspace;                 /* mg_logits_workspace bytes of device memory, for this call alone */
  int64_t workspace_bytes;
  int32_t width, history_len, allowed_kind, type;
} mg_logits;

/* Bytes of workspace that mg_sample_actions and mg_evaluate_actions need (0 up to 8192 tokens). */
int64_t mg_logits_workspace(const mg_logits* a);

/* Adjusted logits, contiguous and of `type`; backward: dlogits = dout * d adjusted / d logits (0 where masked). */
int mg_adjust_logits(const mg_logits* a, void* out, void* stream);
int mg_adjust_logits_backward(const mg_logits* a, const void* dout, void* dlogits, void* stream);

/* One action per row from the adjusted logits: the first v whose running sum of exp exceeds u * (the whole sum), as
 * 64-bit arithmetic finds it; without uniforms (NULL) the first of the largest.  log_prob and entropy f32 [rows].
 * A row without an allowed token: -1, 0, 0; with NaN or +infinity at an allowed token, or a uniform of NaN: -1, NaN,
 * NaN.  Uniforms below 0 are taken as 0; from 1 on they pick the last token with any weight. */
int mg_sample_actions(const mg_logits* a, const float* uniforms, int32_t* actions, float* log_prob, float* entropy,
                      void* stream);

/* log_prob and entropy of given actions; an action that is masked or outside [0, width) has -infinity and passes no
 * gradient.  stats f64 [rows][2] (may be NULL) is what the backward pass wants back. */
int mg_evaluate_actions(const mg_logits* a, const int32_t* actions, float* log_prob, float* entropy, double* stats,
                        void* stream);
int mg_evaluate_actions_backward(const mg_logits* a, const int32_t* actions, const float* entropy, const double* stats,
                                 const float* dlog_prob, const float* dentropy, void* dlogits, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* METTAGRID_HIP_H_ */
