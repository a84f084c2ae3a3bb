"""GraphCacheServer — MI355X-native counterpart of PaGraph/storage/storage.py:18-227.

Same constructor, attributes and methods as the reference class so that
examples/profile/pa_gcn.py drops in; underneath, the per-layer torch index ops
and boolean-mask compactions are one HIP gather launch (pagraph_amd/csrc/
pg_gather.hip) and the miss path is a pinned-host staging buffer + async H2D +
row-scatter kernel (or a zero-copy device read of the pinned host table).

HBM layout
  nid_map      int64 [V_sub]   local -> full id                  (storage.py:34)
  slot_map     int32 [V_sub]   cache slot or -1; fuses gpu_flag (storage.py:38)
                               and localid2cacheid (storage.py:50)
  gpu_fix_cache[name] fp32 [cached_num, dim] row-major, row = slot (storage.py:151)
"""
import ctypes
import os

import torch

from .. import _lib as L


class _Col:
    def __init__(self, data):
        self.data = data


class _NodeFrame:
    def __init__(self, cols):
        self._frame = cols


_THP_MIN_BYTES = 64 << 20


def huge_page_tensor(shape, dtype=torch.float32, register=True):
    """A host tensor in an anonymous mapping backed by transparent huge pages (`madvise(MADV_HUGEPAGE)`), page-locked with
    hipHostRegister so that copy engines and zero-copy kernels may read it: (tensor, device_addressable).
    Why (round 5, profiles/r05/host_gather_sweep.txt): the miss path's CPU row gather reads ~3 300 random 2.4 KB rows per step out
    of a 24 GB table (storage.py:128 `table[nids]`); in 4 KB pages that is 6 M TLB entries and one page walk per row — the same
    gather takes 248 / 127 / 82 us on 2 / 4 / 8 threads out of huge pages against 309 / 176 / 115 us out of hipHostMalloc'ed
    memory, i.e. FOUR threads hold the step on its PCIe floor (0.1500 ms at 5.9 CPUs) where eight were needed.
    Falls back to what the kernel gives (MADV_HUGEPAGE refused: ordinary pages, still registered)."""
    import mmap
    import weakref
    import numpy as np
    n = 1
    for d in shape:
        n *= int(d)
    itemsize = torch.empty((), dtype=dtype).element_size()
    nbytes = max(n * itemsize, itemsize)
    mm = mmap.mmap(-1, nbytes, flags=mmap.MAP_PRIVATE | mmap.MAP_ANONYMOUS)
    try:
        mm.madvise(mmap.MADV_HUGEPAGE)
    except (AttributeError, OSError, ValueError):
        pass
    arr = np.frombuffer(mm, dtype=np.uint8, count=n * itemsize)
    t = torch.from_numpy(arr).view(dtype).reshape(tuple(int(d) for d in shape))     # storage -> ndarray -> mmap stay alive together
    ok = False
    if register and torch.cuda.is_available() and n:
        try:
            ptr = t.data_ptr()
            ok = L.host_register(ptr, n * itemsize)
            if ok:
                weakref.finalize(arr, _unregister, ptr)          # before the mapping goes
        except Exception:
            ok = False
    return t, ok


def _unregister(ptr):
    try:
        torch.cuda.cudart().cudaHostUnregister(ptr)
    except Exception:
        pass


class HostFeatureStore:
    """In-process stand-in for the DGL shared-memory graph store the reference
    attaches to (server/pa_server.py:33-54, examples/profile/pa_gcn.py:33): a
    name -> host tensor table.  Tables are pinned when possible so the miss path
    can DMA / zero-copy from them.  `_node_frame._frame[name].data` is the
    attribute path the reference reads (storage.py:128).

    Fields that are the SAME tensor (GraphSAGE --preprocess publishes `features` twice, as 'features' and
    'neigh') stay one host allocation. `pinned[name]` says whether the device may address the table
    (page-locked by torch or registered with hipHostRegister); `device_visible` overrides the probe for
    tables the caller registered itself."""

    def __init__(self, fields, pin=True, device_visible=None):
        cols = {}
        self.pinned = {}
        done = {}                          # data_ptr of the caller's tensor -> (prepared tensor, pinned?)
        for name, t in fields.items():
            t = torch.as_tensor(t)
            key = (t.data_ptr(), tuple(t.shape), tuple(t.stride()))
            if key not in done:
                u = t.unsqueeze(1) if t.dim() == 1 else t
                u = u.to(torch.float32).contiguous()
                vis = None
                if (pin and torch.cuda.is_available() and not u.is_pinned() and u.numel() * 4 >= _THP_MIN_BYTES
                        and os.environ.get("PG_HOST_TABLE_THP", "1") != "0"):
                    # a large table moves into huge pages (huge_page_tensor: the CPU row gather's TLB reach), registered
                    try:
                        h, ok = huge_page_tensor(u.shape)
                        if ok:
                            h.copy_(u)
                            u, vis = h, True
                    except (OSError, RuntimeError, ValueError):
                        pass
                if vis is None and pin and torch.cuda.is_available() and not u.is_pinned():
                    try:
                        u = u.pin_memory()
                    except RuntimeError:
                        pass  # too large to pin: the staged / async miss paths still work from pageable memory
                if vis is None:
                    vis = u.is_pinned() if torch.cuda.is_available() else False
                done[key] = (u, vis)
            u, vis = done[key]
            if device_visible is not None and name in device_visible:
                vis = bool(device_visible[name])
            self.pinned[name] = vis
            cols[name] = _Col(u)
        self._node_frame = _NodeFrame(cols)

    @property
    def ndata(self):
        return {k: c.data for k, c in self._node_frame._frame.items()}

    @classmethod
    def shared(cls, build_fields, local_rank, tag="store", register=True):
        """ONE host copy of every table per node, mapped by all of its ranks — what the reference's shared-memory
        graph store is (pa_server.py:33-54: one server process publishes, every trainer attaches). Collective over
        the default process group: local rank 0 calls `build_fields()` -> {name: tensor} and copies each distinct
        tensor into a /dev/shm file; the other ranks never build or load anything, they map the files. The files
        are unlinked as soon as everyone holds a mapping (nothing is left behind if the job dies). Each process
        then page-locks its mapping with hipHostRegister so the copy engines / zero-copy kernels may read it."""
        import torch.distributed as dist
        assert dist.is_available() and dist.is_initialized(), "HostFeatureStore.shared needs an initialised process group"
        port = os.environ.get("MASTER_PORT", "0")
        meta = [None]
        maps = {}
        if local_rank == 0:
            fields = build_fields()
            uniq, metas = {}, []
            for name, t in fields.items():
                t = torch.as_tensor(t)
                u = t.unsqueeze(1) if t.dim() == 1 else t
                key = (t.data_ptr(), tuple(u.shape))
                if key not in uniq:
                    path = f"/dev/shm/pagraph_{tag}_{port}_{len(uniq)}.bin"
                    m = torch.from_file(path, shared=True, size=u.numel(), dtype=torch.float32).view(u.shape)
                    m.copy_(u)                      # converts to fp32 on the way; the source may be a numpy memmap
                    uniq[key] = (path, m)
                path, m = uniq[key]
                maps[name] = m
                metas.append((name, path, tuple(u.shape)))
            del fields
            meta = [metas]
        # node-local broadcast: ranks of other nodes would have their own local rank 0; single-node here
        dist.broadcast_object_list(meta, src=0)
        if local_rank != 0:
            opened = {}
            for name, path, shape in meta[0]:
                if path not in opened:
                    n = 1
                    for d in shape:
                        n *= d
                    opened[path] = torch.from_file(path, shared=True, size=n, dtype=torch.float32).view(shape)
                maps[name] = opened[path]
        dist.barrier()
        if local_rank == 0:
            for path in set(p for _, p, _ in meta[0]):
                try:
                    os.unlink(path)
                except OSError:
                    pass
        vis = {}
        seen = {}
        for name, t in maps.items():
            if t.data_ptr() not in seen:
                ok = False
                if register and torch.cuda.is_available():
                    try:
                        ok = L.host_register(t.data_ptr(), t.numel() * 4)
                    except Exception:
                        ok = False
                seen[t.data_ptr()] = ok
            vis[name] = seen[t.data_ptr()]
        return cls(maps, pin=False, device_visible=vis)


def _table(graph, name):
    return graph._node_frame._frame[name].data


def default_host_threads(world_size=1):
    """threads for the miss path's CPU row gather: the CPUs this process may really use (cgroup quota and
    affinity, not the machine's core count), shared between the ranks of a node, minus room for the launch
    thread, the miss-queue worker and the HIP runtime's own threads. The gather is latency bound (a random
    2.4 KB row per ~0.4 us per thread), so it scales with the thread count until the quota is hit; beyond it
    the step gets slower (measured on a 16-CPU quota: 4 threads 0.31 ms/step, 8 0.25, 12 0.24, 32 0.26-0.30)."""
    import os
    cpus = len(os.sched_getaffinity(0)) if hasattr(os, "sched_getaffinity") else (os.cpu_count() or 8)
    try:
        quota, period = open("/sys/fs/cgroup/cpu.max").read().split()[:2]
        if quota != "max":
            cpus = min(cpus, max(1, int(int(quota) / int(period))))
    except (OSError, ValueError):
        pass
    # Round 4: with six whole rows prefetched per thread (pg_missq.hip) 6 threads keep the step on its PCIe floor (0.1506-0.152
    # ms/step for every prefetch setting tried, 7.8 CPUs busy instead of 13.4 with 12 threads): at most 8.
    return max(2, min(8, (cpus - 4 * max(1, world_size)) // max(1, world_size) if cpus > 8 else cpus // 2))


# How a consumer stream is ordered after the async queue's miss rows. Default: on the DEVICE — an event when the worker has
# already enqueued the slot's copy, else a one-wave kernel sleeping on the flag the copy stream raises; the trainer thread
# never waits. PG_MISSQ_HOST_WAIT=1 (GraphCacheServer.host_wait): the trainer thread waits on the host until the worker
# has enqueued the copy, then the stream waits on its event — no spin kernel is ever parked on the consuming stream.
# Measured over 8 + 8 whole-epoch runs on one box (GCN, 10M/100M): same median step (0.168 vs 0.169 ms), but a stall of the
# launch thread now stalls the step directly: 5 of 8 runs had a 20-step window at 0.4-0.7 ms/step (2 of 8 with the
# device-side wait), and in an earlier batch 2 of 8 runs sat at 0.278 ms/step for the whole epoch (the "just in time"
# cycle round 1 described). The host-side wait cannot dead-lock when the runtime maps the consuming stream and the copy
# stream onto one hardware queue, which is why the copy stream lives in another priority class (pg_missq.hip) and
# why bench.py falls back to it when a device-side wait timed out; it is also what rocprofv3 --pmc needs.
_HOST_WAIT = bool(os.environ.get("PG_MISSQ_HOST_WAIT"))


class _FetchPlan:
    __slots__ = ("names", "row_lo", "rows", "out", "fields", "n_fields", "optrs", "ostr", "cache_epoch",
                 # fused layer-0 path (virtual rows): per-plan slot array, dense sub-range, RowSources by (layer, field)
                 "slots", "dense_lo", "dense_rows", "poslo", "row_sources", "virtual",
                 # miss-list index dedup: layer boundaries inside the launch, what _dedup_for needs, the pg_dedup_t
                 "layer_lo", "first_layer", "num_layers", "same_fields", "dedup")


_DEFERRED_MISSQ = []      # miss queues whose owner was finalised where it could not wait for the device (close())


class GraphCacheServer:
    """Manage graph features: static top-out-degree HBM cache + hit/miss gather."""

    def __init__(self, graph, node_num, nid_map, gpuid, miss_mode="staged", host_threads=None):
        self.lib = L.load()  # fails loudly when the HIP library is missing
        self.graph = graph
        self.gpuid = gpuid
        self.node_num = int(node_num)
        self.device = torch.device("cuda", gpuid)
        self.nid_map = torch.as_tensor(nid_map).clone().detach().to(self.device, torch.int64)
        self.slot_map = torch.empty(self.node_num, dtype=torch.int32, device=self.device)
        with torch.cuda.device(self.device):
            L.check(self.lib.pg_slot_map_reset(L.ptr(self.slot_map), self.node_num, L.stream_ptr()), "pg_slot_map_reset")

        self.cached_num = 0
        self.capability = self.node_num
        self.full_cached = False
        self.dims = {}
        self.total_dim = 0
        self.gpu_fix_cache = dict()

        self.log = False
        self.try_num = 0
        self.miss_num = 0

        # miss path state
        assert miss_mode in ("staged", "zerocopy", "async")
        pinned = getattr(graph, "pinned", None)
        if miss_mode == "zerocopy" and pinned is not None and not all(pinned.values()):
            # a kernel reading pageable host memory faults. The async queue gathers on the CPU and works from
            # pageable tables (and is the faster path anyway): use it, and say so.
            print("GraphCacheServer: host table(s) {} are not page-locked; miss_mode 'zerocopy' -> 'async'".format(
                [n for n, v in pinned.items() if not v]))
            miss_mode = "async"
        self.miss_mode = miss_mode
        self.host_threads = int(host_threads) if host_threads else default_host_threads()
        self._cap = 0
        self._miss_pos = None            # device int32 [cap]
        self._slots = None               # device int32 [cap]: slot of every row of the launch (k_split -> k_gather)
        self._miss_fullid = None         # pinned int64 [cap]
        self._miss_count = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._miss_count_h = torch.zeros(1, dtype=torch.int32).pin_memory()
        self._staging = {}               # name -> pinned fp32 [cap, dim]
        self._staged_dev = {}            # name -> device fp32 [cap, dim]
        self._event = torch.cuda.Event()
        self._stats = torch.zeros(2, dtype=torch.int64, device=self.device)   # [try, miss], accumulated by k_split
        # bench.py: when a list, every gather launch is bracketed by HIP events on its own stream
        # and (timer_handle, rows, misses_or_None) is appended
        self.profile = None
        # miss_mode == "async": libpagraph's worker-thread miss queue (pg_missq_*), one slot per in-flight batch
        self._missq = None
        self._missq_rows = 0
        self._missq_nslots = 0
        self._missq_bufs = {}            # slot -> (miss_pos, miss_fullid, miss_count) pointers
        self._missq_pending = set()      # slots submitted to the queue and not yet waited for by their consumer
        # True: consumers wait for the worker on the HOST and then on an event — never a spin-wait kernel on the consuming
        # stream. Slower pipeline (the launch thread blocks), but it cannot dead-lock when the runtime maps the consuming
        # stream and the copy stream onto one hardware queue; bench.py switches to it when a device-side wait timed out.
        self.host_wait = _HOST_WAIT
        # bench.py: (device int64 [3 * ring], ring) — the fused gather+aggregate kernel stamps its own start / end
        self.rows_prof = None
        self._missq_share = None
        self._missq_tails = False
        self._cache_epoch = 0            # bumped whenever the cache contents / layout change (invalidates fetch plans)
        self.missq_slots = 4
        # miss_mode 'async': the leading share of every miss list goes through the worker thread (CPU gather + copy
        # engine), the rest is read by the device over PCIe on the fetching stream; 1.0 = all through the worker
        self.cpu_share = 1.0
        # index dedup of the miss list (pg_dedup_t): a vertex that misses in several layers of one NodeFlow crosses PCIe
        # once and is copied on the device for the other layers. Async queue only (an attribute: a caller may turn it off).
        self.dedup_misses = True
        self._missq_dup = {}
        # state tensors were filled on the current stream; the fetching stream of a trainer does not synchronise with it
        torch.cuda.current_stream(self.device).synchronize()

    # -- reference-shaped views of the fused slot map --------------------------
    def _export(self):
        flag = torch.empty(self.node_num, dtype=torch.uint8, device=self.device)
        l2c = torch.empty(self.node_num, dtype=torch.int64, device=self.device)
        with torch.cuda.device(self.device):
            L.check(self.lib.pg_slot_map_export(L.ptr(self.slot_map), self.node_num, L.ptr(flag), L.ptr(l2c),
                                                L.stream_ptr()), "pg_slot_map_export")
        return flag.bool(), l2c

    @property
    def gpu_flag(self):
        return self._export()[0]

    @property
    def localid2cacheid(self):
        return self._export()[1]

    # -- storage.py:59-67 -----------------------------------------------------
    def init_field(self, embed_names):
        nid = torch.zeros(1, dtype=torch.int64, device=self.device)
        feats = self.get_feat_from_server(nid, embed_names)
        self.total_dim = 0
        for name in embed_names:
            self.dims[name] = feats[name].size(1)
            self.total_dim += feats[name].size(1)
        if len(self.dims) > L.PG_MAX_FIELDS:
            raise L.PgError(f"at most {L.PG_MAX_FIELDS} feature fields")
        print('total dims: {}'.format(self.total_dim))

    # -- storage.py:70-104 ----------------------------------------------------
    def auto_cache(self, dgl_g, embed_names, cache_ratio=None, policy="degree", freq=None):
        """Reference rule: capability = (total - peak_alloc - peak_reserved - 1 GiB) / (4*total_dim).
        `cache_ratio` (fraction of node_num) overrides it — the reference keeps such overrides
        commented out at storage.py:85-86; on a 288 GB MI355X the rule alone caches everything.
        `policy`: 'degree' (default) = the reference's rule, the `capability` highest out-degree vertices
        (storage.py:97-104). 'presample' (opt-in, beyond the reference): the `capability` vertices a presampled epoch
        looked up most often — `freq` = analysis.access_frequency(...)[0] over the layers the loop fetches, i.e. the
        ORDER examples/opt_cache_hit.py:22-31 evaluates as its upper bound, made the policy; ties (the many vertices
        never seen) fall back to the degree order. On a GPU the sampler does an epoch in tens of milliseconds, which is
        what makes the oracle's order affordable at start-up."""
        if policy not in ("degree", "presample"):
            raise ValueError(f"unknown cache policy {policy!r}")
        if policy == "presample" and freq is None:
            raise ValueError("policy='presample' needs freq (analysis.access_frequency over a presampled epoch)")
        peak_allocated_mem = torch.cuda.max_memory_allocated(device=self.device)
        peak_cached_mem = torch.cuda.max_memory_reserved(device=self.device)
        total_mem = torch.cuda.get_device_properties(self.device).total_memory
        available = total_mem - peak_allocated_mem - peak_cached_mem - 1024 * 1024 * 1024
        self.capability = max(0, int(available / (self.total_dim * 4)))   # the rule goes negative when the peaks
        # (which count freed set-up memory, and count it twice) exceed the device: cache nothing then, do not
        # slice from the end of the degree order
        if cache_ratio is not None:
            self.capability = min(self.capability, int(self.node_num * cache_ratio))
        print('Cache Memory: {:.2f}G. Capability: {}'.format(available / 1024 / 1024 / 1024, self.capability))
        # The rule budgets capability * total_dim * 4 bytes, which is what the reference allocates. This build's
        # rows are padded to whole 128-byte lines (601 -> 608 floats) and the fill stages each chunk on the
        # device, so the same row count needs up to 6 % + one chunk more: never ask for more rows than the
        # memory that is really free right now can hold.
        fit, chunk_rows = self._physical_fit(min(self.capability, self.node_num), embed_names)
        if fit < min(self.capability, self.node_num):
            print('Capability limited by free device memory: {} -> {}'.format(self.capability, fit))
            self.capability = fit
        if self.capability >= self.node_num:
            print('cache the full graph...')
            full_nids = torch.arange(self.node_num, device=self.device)
            self._fill_cache(full_nids, embed_names, is_full=True, chunk_rows=chunk_rows)
        else:
            print('cache the part of graph... caching percentage: {:.4f}'.format(self.capability / self.node_num))
            out_degrees = torch.as_tensor(dgl_g.out_degrees()).to(self.device)
            # descending by out-degree; ties -> lower id first (the reference's torch.argsort is unstable)
            sort_nid = torch.argsort(out_degrees, descending=True, stable=True)
            if policy == "presample":
                f = torch.as_tensor(freq).to(self.device, torch.int64)
                if f.numel() != self.node_num:
                    raise ValueError("freq must have one entry per vertex of the partition")
                # most looked-up first; among equals the degree order (a stable sort of the degree order by frequency)
                sort_nid = sort_nid[torch.argsort(f[sort_nid], descending=True, stable=True)]
                print('cache policy: presampled access frequency ({} of {} vertices seen)'.format(
                    int((f > 0).sum()), self.node_num))
            cache_nid = sort_nid[:self.capability]
            self._fill_cache(cache_nid, embed_names, is_full=False, chunk_rows=chunk_rows)

    def _physical_fit(self, want_rows, embed_names, reserve=1 << 30):
        """(rows, chunk_rows): how many of `want_rows` fused cache rows fit into the device memory that is free now
        (driver-free + what torch's allocator holds unused), next to the fill's per-chunk device staging, keeping
        `reserve` bytes back; the chunk shrinks before the cache does."""
        total_dim = sum(self.dims[n] for n in embed_names)
        row_bytes = self._row_stride(total_dim) * 4
        free, _ = torch.cuda.mem_get_info(self.device)
        free += torch.cuda.memory_reserved(self.device) - torch.cuda.memory_allocated(self.device)
        budget = free - reserve
        for chunk_rows in (1 << 20, 1 << 18, 1 << 16, 1 << 14):
            chunk_rows = max(1, min(chunk_rows, want_rows))
            rows = (budget - chunk_rows * total_dim * 4) // row_bytes
            if rows >= want_rows:
                return want_rows, chunk_rows
        return max(0, int(rows)), chunk_rows

    @staticmethod
    def _row_stride(total_dim):
        """floats per fused cache row: a whole number of 128-byte lines when that wastes < 6 %
        (601 -> 608: every row read touches exactly 19 lines), else a multiple of 16 bytes"""
        s128 = (total_dim * 4 + 127) // 128 * 32
        return s128 if s128 <= total_dim * 1.06 else (total_dim + 3) // 4 * 4

    def _alloc_fused(self, rows, names):
        """All fields of a cached vertex live in ONE HBM row ([features | norm | pad]); the
        per-field `gpu_fix_cache[name]` tensors are column views of it. A narrow field next to
        its wide field shares the DRAM lines the row read fetches anyway — as a separate
        [rows, 1] array every 4-byte lookup cost ~0.5 KB of HBM traffic (PMC, profiles/r01)."""
        total = sum(self.dims[n] for n in names)
        stride = self._row_stride(total)
        fused = torch.empty((rows, stride), dtype=torch.float32, device=self.device)
        views, off = {}, 0
        for n in names:
            views[n] = fused[:, off:off + self.dims[n]]
            off += self.dims[n]
        return fused, views

    def _fill_cache(self, nids, embed_names, is_full, chunk_rows=1 << 20):
        """get_feat_from_server + cache_fix_data (storage.py:94-95,103-104) in bounded chunks."""
        rows = nids.numel()
        fused, views = self._alloc_fused(rows, embed_names)
        for lo in range(0, rows, chunk_rows):
            hi = min(rows, lo + chunk_rows)
            part = self.get_feat_from_server(nids[lo:hi], embed_names, to_gpu=True)
            for name in embed_names:
                views[name][lo:hi] = part[name]
        self._adopt_cache(nids, fused, views, is_full)

    def _adopt_cache(self, nids, fused, views, is_full):
        rows = nids.size(0)
        nids = nids.to(self.device, torch.int64).contiguous()
        with torch.cuda.device(self.device):
            L.check(self.lib.pg_slot_map_assign(L.ptr(self.slot_map), L.ptr(nids), rows, L.stream_ptr()),
                    "pg_slot_map_assign")
        self.cached_num = rows
        self._fused_cache = fused
        self.gpu_fix_cache = dict(views)
        self.full_cached = is_full
        self._cache_epoch += 1

    # -- storage.py:107-132 ---------------------------------------------------
    def get_feat_from_server(self, nids, embed_names, to_gpu=False):
        """rows of `nids` (local ids, on the GPU) from the host store: full = nid_map[nids];
        table[full] gathered by the library's host threads into pinned memory."""
        nids_in_full = self.nid_map[nids].cpu()
        n = nids_in_full.numel()
        frame = {}
        for name in embed_names:
            tab = _table(self.graph, name)
            dim = tab.size(1)
            staged = torch.empty((n, dim), dtype=torch.float32, pin_memory=bool(to_gpu))
            L.check(self.lib.pg_host_gather_rows(L.ptr(tab), tab.stride(0), dim, L.ptr(nids_in_full), n,
                                                 L.ptr(staged), self.host_threads), "pg_host_gather_rows")
            frame[name] = staged.to(self.device, non_blocking=True) if to_gpu else staged
        if to_gpu:
            torch.cuda.current_stream(self.device).synchronize()  # staged buffers die with this scope
        return frame

    # -- storage.py:135-154 ---------------------------------------------------
    def cache_fix_data(self, nids, data, is_full=False):
        rows = nids.size(0)
        for name in data:
            assert (rows == data[name].size(0))
            self.dims[name] = data[name].size(1)
        fused, views = self._alloc_fused(rows, list(data))
        for name in data:
            views[name].copy_(data[name])
        self._adopt_cache(nids, fused, views, is_full)

    # -- buffers for the miss path --------------------------------------------
    def _ensure_capacity(self, n, stream=None):
        """(re)allocate the miss-list scratch for n rows. `stream`: the stream whose kernels FILL these buffers — they are
        allocated from ITS pool (a block of another stream's pool may still be written by that stream's running kernels;
        see GraphedTrainer.prepare)"""
        if n <= self._cap:
            return
        if stream is not None and stream != torch.cuda.current_stream(self.device):
            with torch.cuda.stream(stream):
                return self._ensure_capacity(n)
        cap = max(n, int(self._cap * 1.5), 1024)
        self._miss_pos = torch.empty(cap, dtype=torch.int32, device=self.device)
        self._slots = torch.empty(cap, dtype=torch.int32, device=self.device)
        self._miss_fullid = torch.empty(cap, dtype=torch.int64).pin_memory()
        if self.miss_mode == "staged":
            for name, dim in self.dims.items():
                self._staging[name] = torch.empty((cap, dim), dtype=torch.float32).pin_memory()
                self._staged_dev[name] = torch.empty((cap, dim), dtype=torch.float32, device=self.device)
        self._cap = cap

    # -- storage.py:157-204 ---------------------------------------------------
    def fetch_data(self, nodeflow, out=None, need=None, slot=None, virtual=None):
        """Fill nodeflow._node_frames[i][name] for every layer and field: hits from the HBM
        cache, misses from the host store. One gather launch for all layers; rows of layer i are
        the slice [offsets[i], offsets[i+1]) of one [R, dim] buffer per field.
        `out` (optional): {name: preallocated [>=R, dim] tensor} to gather into — the fixed-shape
        path (hipGraph replay) passes its static frames; padding ids (< 0) leave their rows untouched.
        `need` (optional, SURVEY §8f-2 "fetch only what the model reads"): {layer index: [field names]};
        rows of layers / fields the model never reads are neither gathered nor fetched over PCIe
        (GCN training reads only layer 0's 'features', gcn_nssc.py:64). Default: everything, as the
        reference does.
        `slot` (miss_mode == "async"): index of the in-flight batch; the miss rows land asynchronously,
        call wait_misses(slot) on the consuming stream before reading the frames."""
        if virtual and (self.full_cached or self.miss_mode == "async"):
            # `virtual` (a model's virtual_inputs()): the leading layers' rows are not materialised; their frames
            # hold ops.RowSource objects the aggregation reads in place (see plan_fetch)
            return self._fetch_data_virtual(nodeflow, out, need, slot, virtual)
        if self.full_cached:
            self.fetch_from_cache(nodeflow, out=out)
            return
        with torch.autograd.profiler.record_function('cache-idxload'):
            nf_nids = nodeflow._node_mapping.tousertensor().to(self.device, torch.int64)
            offsets = nodeflow._layer_offsets
        names = list(self.dims)
        row_lo = 0
        if need is not None:
            # the needed layers form a prefix-contiguous row range [lo, hi) of the NodeFlow
            layers = sorted(need)
            assert layers == list(range(layers[0], layers[-1] + 1)), "needed layers must be contiguous"
            wanted = set(n for l in layers for n in need[l])
            names = [n for n in names if n in wanted]
            row_lo, row_hi = offsets[layers[0]], offsets[layers[-1] + 1]
            nf_nids = nf_nids[row_lo:row_hi]
            if out is not None:
                out = {n: out[n][row_lo:row_hi] for n in names}
        R = nf_nids.numel()
        stream = torch.cuda.current_stream(self.device)
        sp = L.stream_ptr(stream)
        with torch.autograd.profiler.record_function('cache-allocate'):
            if out is None:
                out = {name: torch.empty((R, self.dims[name]), dtype=torch.float32, device=self.device) for name in names}
            self._ensure_capacity(R)
            miss_pos, miss_fullid, miss_count = L.ptr(self._miss_pos), L.ptr(self._miss_fullid), L.ptr(self._miss_count)
            if self.miss_mode == "async":
                if slot is None:
                    raise L.PgError("miss_mode='async' needs fetch_data(..., slot=k)")
                miss_pos, miss_fullid, miss_count = self._missq_buffers(slot, R)
                self._order_after_tail(slot, sp)
        with torch.autograd.profiler.record_function('cache-gpu'):
            fields, nf = L.make_fields(
                (self.gpu_fix_cache.get(name), out[name], self.dims[name],
                 self.gpu_fix_cache[name].stride(0) if name in self.gpu_fix_cache else self.dims[name],
                 out[name].stride(0)) for name in names)
            timer = None
            if self.profile is not None:
                timer = L.vp()
                L.check(self.lib.pg_timer_create(ctypes.byref(timer)), "pg_timer_create")
            dd = None
            if self.miss_mode == "async":
                lay = sorted(need) if need is not None else list(range(nodeflow.num_layers))
                same = need is None or all(set(need[l]) == set(need[lay[0]]) for l in lay)
                dd = self._dedup_for(slot, [offsets[l] - row_lo for l in lay] + [offsets[lay[-1] + 1] - row_lo], lay[0],
                                     nodeflow.num_layers, same)
            ml = L.miss_list(miss_pos, miss_fullid, miss_count)
            L.check(self.lib.pg_gather_rows(L.ptr(nf_nids), R, L.ptr(self.slot_map), L.ptr(self.nid_map), fields, nf,
                                            ctypes.byref(ml), L.ptr(self._slots), L.ptr(self._stats) if self.log else None, timer,
                                            ctypes.byref(dd) if dd is not None else None, sp),
                    "pg_gather_rows")
            if timer is not None:
                self.profile.append([timer, R, None])
        with torch.autograd.profiler.record_function('cache-cpu'):
            if self.miss_mode == "async":
                optrs = (L.vp * L.PG_MAX_FIELDS)()
                ostr = (L.c_i32 * L.PG_MAX_FIELDS)()
                for f, name in enumerate(self.dims):          # queue fields are in self.dims order
                    if name in out and name in names:
                        optrs[f] = out[name].data_ptr()
                        ostr[f] = out[name].stride(0)
                L.check(self.lib.pg_missq_submit(self._missq, slot, optrs, ostr, None,
                                                       L.ptr(self._slots) if dd is not None else None, sp), "pg_missq_submit")
                self._missq_pending.add(slot)
                if self._missq_share < 256:
                    self._device_tail(slot, sp)
            elif self.miss_mode == "zerocopy":
                for name in names:
                    tab = _table(self.graph, name)
                    L.check(self.lib.pg_scatter_rows_from_host(
                        L.ptr(tab), tab.stride(0), L.ptr(self._miss_pos), L.ptr(self._miss_fullid), R,
                        L.ptr(self._miss_count), self.dims[name], L.ptr(out[name]), out[name].stride(0), sp),
                        "pg_scatter_rows_from_host")
            else:
                self._miss_count_h.copy_(self._miss_count, non_blocking=True)
                self._event.record(stream)
                self._event.synchronize()          # host needs the miss list: only this stream is waited on
                m = int(self._miss_count_h[0])
                if m > 0:
                    full = self._miss_fullid
                    for name in names:
                        tab = _table(self.graph, name)
                        dim = self.dims[name]
                        stg = self._staging[name]
                        L.check(self.lib.pg_host_gather_rows(L.ptr(tab), tab.stride(0), dim, L.ptr(full), m,
                                                             L.ptr(stg), self.host_threads), "pg_host_gather_rows")
                        dev = self._staged_dev[name]
                        dev[:m].copy_(stg[:m], non_blocking=True)       # pinned -> HBM, hipMemcpyAsync
                        L.check(self.lib.pg_scatter_rows(L.ptr(dev), L.ptr(self._miss_pos), m, None, dim,
                                                         L.ptr(out[name]), out[name].stride(0), sp), "pg_scatter_rows")
                    # the pinned staging buffers are reused next step: the copy must have left them
                    self._event.record(stream)
                    self._event.synchronize()
                if self.profile:
                    self.profile[-1][2] = m
        with torch.autograd.profiler.record_function('cache-asign'):
            for i in range(nodeflow.num_layers):
                if need is not None and i not in need:
                    nodeflow._node_frames[i] = {}
                    continue
                keep = names if need is None else [n for n in names if n in need[i]]
                nodeflow._node_frames[i] = {name: out[name][offsets[i] - row_lo:offsets[i + 1] - row_lo] for name in keep}

    def _fetch_data_virtual(self, nodeflow, out, need, slot, virtual):
        nf_nids = nodeflow._node_mapping.tousertensor().to(self.device, torch.int64)
        offsets = nodeflow._layer_offsets
        R = offsets[-1]
        names = list(self.dims) if need is None else [n for n in self.dims if any(n in v for v in need.values())]
        if out is None:
            out = {n: torch.empty((R, self.dims[n]), dtype=torch.float32, device=self.device) for n in names}
        plan = self.plan_fetch(offsets, out, need, virtual, slot=slot)
        if not plan.virtual:
            return self.fetch_data(nodeflow, out=out, need=need, slot=slot)
        self.fetch_planned(plan, nf_nids, torch.cuda.current_stream(self.device), slot=slot)
        lo = plan.row_lo + plan.dense_lo
        for i in range(nodeflow.num_layers):
            if need is not None and i not in need:
                nodeflow._node_frames[i] = {}
                continue
            keep = plan.names if need is None else [n for n in plan.names if n in need[i]]
            fr = {}
            for name in keep:
                rs = plan.row_sources.get((i, name))
                fr[name] = rs if rs is not None else plan.out[name][offsets[i] - lo:offsets[i + 1] - lo]
            nodeflow._node_frames[i] = fr
        nodeflow._fetch_plan = plan        # keeps the slot array alive as long as the NodeFlow

    # -- fixed-shape fast path (hipGraph pipelines) ---------------------------------------------
    def plan_fetch(self, layer_offsets, out, need=None, virtual=None, slot=None):
        """Everything fetch_data derives from (layer offsets, output frames, `need`) computed once, for callers
        that fetch the same shapes into the same frames every step (GraphedTrainer): the per-step call is
        then fetch_planned(plan, ...) = two or three C-ABI calls and no tensor slicing — at ~0.2 ms per
        step the launch thread is the bottleneck, not the GPU. Not for miss_mode 'staged' (which
        synchronises with the host anyway).
        `virtual` ({layer: [fields]}, a model's virtual_inputs()): fields of the FIRST needed layers that the model
        only aggregates. Their rows are not gathered: plan.row_sources[(layer, field)] is an ops.RowSource over the
        cache and the slot's staged miss block, which the aggregation kernel reads in place. Needs the
        async miss queue (`slot` = its slot index for this plan) or a full cache; silently ignored otherwise."""
        if self.miss_mode == "staged" and not self.full_cached:
            raise L.PgError("plan_fetch: miss_mode 'staged' has no asynchronous fast path")
        from ..ops import RowSource
        plan = _FetchPlan()
        names = list(self.dims)
        offsets = [int(x) for x in layer_offsets]
        lo, hi = offsets[0], offsets[-1]
        layers = list(range(len(offsets) - 1))
        if need is not None:
            layers = sorted(need)
            assert layers == list(range(layers[0], layers[-1] + 1)), "needed layers must be contiguous"
            wanted = set(n for l in layers for n in need[l])
            names = [n for n in names if n in wanted]
            lo, hi = offsets[layers[0]], offsets[layers[-1] + 1]
        plan.names, plan.row_lo, plan.rows = names, lo, hi - lo
        plan.layer_lo = [offsets[l] - lo for l in layers] + [hi - lo]
        plan.first_layer, plan.num_layers = layers[0], len(offsets) - 1
        plan.same_fields = need is None or all(set(need[l]) == set(need[layers[0]]) for l in layers)
        plan.dedup = False             # False = not looked at yet (needs the slot's queue buffers); None = no dedup
        # ---- which leading layers stay un-materialised -------------------------------------------------------
        vlayers = []
        if virtual and (self.full_cached or self.miss_mode == "async") and (self.full_cached or slot is not None):
            per_layer = [set(need[l]) if need is not None else set(names) for l in layers]
            same_everywhere = all(f == per_layer[0] for f in per_layer)
            for l in layers:
                want = per_layer[layers.index(l)]
                v = set(virtual.get(l, ()))
                # wide rows in whole 16-byte pieces: dim % 4 == 0, or (Reddit's 602) a fused cache row with room for the last
                # piece (the miss queue pads its staged rows the same way: pg_missq_staged_stride)
                wide = all(self.dims[n] >= 256 and (self.dims[n] % 4 == 0 or n not in self.gpu_fix_cache
                           or (self.gpu_fix_cache[n].stride(0) >= ((self.dims[n] + 3) & ~3)
                               and self.gpu_fix_cache[n].data_ptr() % 16 == 0)) for n in want)
                if want and want <= v and wide and l == layers[0] + len(vlayers) and (same_everywhere or len(layers) == 1):
                    vlayers.append(l)
                else:
                    break
        plan.virtual = bool(vlayers)
        plan.dense_lo = offsets[vlayers[-1] + 1] - lo if vlayers else 0
        plan.dense_rows = plan.rows - plan.dense_lo
        plan.slots = torch.empty(max(1, plan.rows), dtype=torch.int32, device=self.device) if vlayers else None
        plan.out = {n: out[n][lo + plan.dense_lo:hi] for n in names}
        plan.fields, plan.n_fields = L.make_fields(
            (self.gpu_fix_cache.get(name), plan.out[name], self.dims[name],
             self.gpu_fix_cache[name].stride(0) if name in self.gpu_fix_cache else self.dims[name],
             plan.out[name].stride(0)) for name in names)
        plan.optrs = (L.vp * L.PG_MAX_FIELDS)()
        plan.ostr = (L.c_i32 * L.PG_MAX_FIELDS)()
        plan.poslo = (L.c_i32 * L.PG_MAX_FIELDS)()
        for f, name in enumerate(self.dims):          # queue fields are in self.dims order
            if name in plan.out:
                plan.poslo[f] = plan.dense_lo
                if plan.dense_rows > 0:
                    plan.optrs[f] = plan.out[name].data_ptr()
                    plan.ostr[f] = plan.out[name].stride(0)
                else:
                    plan.optrs[f] = None
                    plan.ostr[f] = -1                 # every needed row is read in place: copy to the staged block only
        plan.row_sources = {}
        if vlayers:
            staged, sstride = {}, {}
            if not self.full_cached:
                self._missq_buffers(slot, plan.rows)  # creates the queue if need be
                for f, name in enumerate(self.dims):
                    if name in names:
                        sp_, st_ = L.vp(), L.c_i32(0)
                        L.check(self.lib.pg_missq_slot_staged(self._missq, slot, f, ctypes.byref(sp_)), "pg_missq_slot_staged")
                        L.check(self.lib.pg_missq_staged_stride(self._missq, f, ctypes.byref(st_)), "pg_missq_staged_stride")
                        staged[name], sstride[name] = sp_.value, int(st_.value)
            for l in vlayers:
                a, b = offsets[l] - lo, offsets[l + 1] - lo
                for name in (need[l] if need is not None else names):
                    plan.row_sources[(l, name)] = RowSource(plan.slots[a:b], self.gpu_fix_cache.get(name), staged.get(name, 0),
                                                            sstride.get(name, self.dims[name]), self.dims[name],
                                                            keep=(self, plan),
                                                            # (the self-timing ring is indexed by the step: ONE launch per
                                                            # step may stamp it — the first layer's, the dominant one)
                                                            prof=self.rows_prof if l == vlayers[0] else None)
        plan.cache_epoch = self._cache_epoch
        return plan

    def fetch_planned(self, plan, node_mapping, stream, slot=None):
        """fetch_data for a plan: node_mapping = the NodeFlow's id tensor (device int64), rows
        [plan.row_lo, plan.row_lo + plan.rows) of it are gathered into the plan's frames on `stream`."""
        if plan.cache_epoch != self._cache_epoch:
            raise L.PgError("fetch_planned: the cache changed after plan_fetch (re-plan after auto_cache)")
        R = plan.rows
        sp = ctypes.c_void_p(stream.cuda_stream)
        ids = ctypes.c_void_p(node_mapping.data_ptr() + 8 * plan.row_lo)
        if plan.virtual:
            return self._fetch_virtual(plan, ids, sp, slot, stream)
        if self.full_cached and not self.log:
            L.check(self.lib.pg_gather_rows_full(ids, R, plan.fields, plan.n_fields, sp), "pg_gather_rows_full")
            return
        self._ensure_capacity(R, stream)
        if self.miss_mode == "async" and not self.full_cached:
            if slot is None:
                raise L.PgError("miss_mode='async' needs fetch_planned(..., slot=k)")
            miss_pos, miss_fullid, miss_count = self._missq_buffers(slot, R)
            self._order_after_tail(slot, sp)
        else:
            miss_pos, miss_fullid, miss_count = L.ptr(self._miss_pos), L.ptr(self._miss_fullid), L.ptr(self._miss_count)
        timer = None
        if self.profile is not None:
            timer = L.vp()
            L.check(self.lib.pg_timer_create(ctypes.byref(timer)), "pg_timer_create")
        dd = self._plan_dedup(plan, slot) if self.miss_mode == "async" and not self.full_cached else None
        ml = L.miss_list(miss_pos, miss_fullid, miss_count)
        L.check(self.lib.pg_gather_rows(ids, R, L.ptr(self.slot_map), L.ptr(self.nid_map), plan.fields, plan.n_fields,
                                        ctypes.byref(ml), L.ptr(self._slots), L.ptr(self._stats) if self.log else None, timer,
                                        ctypes.byref(dd) if dd is not None else None, sp), "pg_gather_rows")
        if timer is not None:
            self.profile.append([timer, R, None])
        if self.full_cached:
            return                       # every row was a hit (the general kernel ran only for the hit counters)
        if self.miss_mode == "async":
            L.check(self.lib.pg_missq_submit(self._missq, slot, plan.optrs, plan.ostr, None,
                                                   L.ptr(self._slots) if dd is not None else None, sp), "pg_missq_submit")
            self._missq_pending.add(slot)
            if self._missq_share < 256:
                self._device_tail(slot, sp)
        else:
            for name in plan.names:
                tab = _table(self.graph, name)
                o = plan.out[name]
                L.check(self.lib.pg_scatter_rows_from_host(
                    L.ptr(tab), tab.stride(0), L.ptr(self._miss_pos), L.ptr(self._miss_fullid), R,
                    L.ptr(self._miss_count), self.dims[name], L.ptr(o), o.stride(0), sp), "pg_scatter_rows_from_host")

    def _fetch_virtual(self, plan, ids, sp, slot, stream=None):
        """split every needed row (slots + miss list), gather only the rows of the layers that are read row by row,
        hand the miss list to the queue: rows of the leading layers stay in the cache / the staged block"""
        R = plan.rows
        use_q = self.miss_mode == "async" and not self.full_cached
        if use_q:
            if slot is None:
                raise L.PgError("miss_mode='async' needs fetch_planned(..., slot=k)")
            miss_pos, miss_fullid, miss_count = self._missq_buffers(slot, R)
            self._order_after_tail(slot, sp)
        else:
            self._ensure_capacity(R, stream)
            miss_pos, miss_fullid, miss_count = L.ptr(self._miss_pos), L.ptr(self._miss_fullid), L.ptr(self._miss_count)
        dd = self._plan_dedup(plan, slot) if use_q else None
        if self.full_cached and not use_q:
            # nothing can miss: the slots alone, one launch (no miss counter to zero first)
            L.check(self.lib.pg_slots_full(ids, R, L.ptr(self.slot_map), L.ptr(plan.slots),
                                           L.ptr(self._stats) if self.log else None, sp), "pg_slots_full")
        else:
            ml = L.miss_list(miss_pos, miss_fullid, miss_count)
            L.check(self.lib.pg_split_rows(ids, R, L.ptr(self.slot_map), L.ptr(self.nid_map), ctypes.byref(ml), L.ptr(plan.slots),
                                           L.ptr(self._stats) if self.log else None,
                                           ctypes.byref(dd) if dd is not None else None, sp),
                    "pg_split_rows")
        if plan.dense_rows > 0:
            timer = None
            if self.profile is not None:
                timer = L.vp()
                L.check(self.lib.pg_timer_create(ctypes.byref(timer)), "pg_timer_create")
            L.check(self.lib.pg_gather_rows_presplit(ctypes.c_void_p(plan.slots.data_ptr() + 4 * plan.dense_lo),
                                                     plan.dense_rows, plan.fields, plan.n_fields, timer, sp),
                    "pg_gather_rows_presplit")
            if timer is not None:   # 4th item: share of the split rows this copy launch covers
                self.profile.append([timer, plan.dense_rows, None, plan.dense_rows / max(1, plan.rows)])
        if use_q:
            L.check(self.lib.pg_missq_submit(self._missq, slot, plan.optrs, plan.ostr, plan.poslo,
                                                   L.ptr(plan.slots) if dd is not None else None, sp),
                    "pg_missq_submit")
            self._missq_pending.add(slot)
            if self._missq_share < 256:      # the device reads the tail of the list into the staged block itself
                self._device_tail(slot, sp)

    def _plan_dedup(self, plan, slot):
        """the plan's pg_dedup_t (built at its first fetch: the slot's queue buffers exist by then), or None"""
        if plan.dedup is False:
            plan.dedup = self._dedup_for(slot, plan.layer_lo, plan.first_layer, plan.num_layers, plan.same_fields)
        return plan.dedup

    def _device_tail(self, slot, sp):
        self._missq_tails = True
        L.check(self.lib.pg_missq_device_tail(self._missq, slot, sp), "pg_missq_device_tail")

    def _order_after_tail(self, slot, sp):
        """cpu_share < 1: the split about to run rewrites the slot's miss list, which the previous submission's device
        tail may still be reading on the queue's stream"""
        if self._missq_tails:           # a device tail has been enqueued on this queue at some point
            L.check(self.lib.pg_missq_order_after_tail(self._missq, slot, sp), "pg_missq_order_after_tail")

    def _missq_buffers(self, slot, rows):
        hit = self._missq_bufs.get(slot)
        if hit is not None and rows <= self._missq_rows and slot < self._missq_nslots:
            return hit
        if self._missq is None or rows > self._missq_rows or slot >= self._missq_nslots:
            # (a consumer with a deeper ring than the one the queue was made for needs more slots)
            self._missq_bufs = {}
            self._missq_dup = {}
            recreated = self._missq is not None
            if self._missq is not None:
                # batches in flight on other slots still own the old queue's buffers: let the worker enqueue their
                # copies, let the device finish them, only then free (a growing NodeFlow in the eager trainer)
                L.check(self.lib.pg_missq_drain(self._missq), "pg_missq_drain")
                torch.cuda.synchronize(self.device)
                self._missq_pending.clear()
                L.check(self.lib.pg_missq_destroy(self._missq), "pg_missq_destroy")
            cap = max(int(rows * 1.25), 4096, self._missq_rows)
            arr = (L.PgMissqField * len(self.dims))()
            for f, name in enumerate(self.dims):
                tab = _table(self.graph, name)
                arr[f].table, arr[f].table_stride, arr[f].dim = tab.data_ptr(), tab.stride(0), self.dims[name]
            h = L.vp()
            L.check(self.lib.pg_missq_create(self.device.index, self.missq_slots, cap, arr, len(self.dims),
                                             self.host_threads, ctypes.byref(h)), "pg_missq_create")
            self._missq, self._missq_rows, self._missq_nslots = h, cap, self.missq_slots
            self._missq_share = None
            if recreated:
                self._cache_epoch += 1   # fetch plans hold pointers into the old queue's staging blocks
        share = max(0, min(256, int(round(self.cpu_share * 256))))
        pinned = getattr(self.graph, "pinned", None)
        if share < 256 and pinned is not None and not all(pinned.get(n, False) for n in self.dims):
            raise L.PgError("cpu_share < 1 lets the device read the tail of every miss list from the host table, "
                            "which needs page-locked tables")
        if share != self._missq_share:
            L.check(self.lib.pg_missq_set_cpu_share(self._missq, share), "pg_missq_set_cpu_share")
            self._missq_share = share
        pos, full, cnt = L.vp(), L.vp(), L.vp()
        L.check(self.lib.pg_missq_slot_buffers(self._missq, slot, ctypes.byref(pos), ctypes.byref(full),
                                               ctypes.byref(cnt)), "pg_missq_slot_buffers")
        self._missq_bufs[slot] = (pos, full, cnt)
        return pos, full, cnt

    def adapt_cpu_share(self, min_jobs=8, floor_GBps=None, quiet=False, apply=True):
        """Set `cpu_share` from what this rank's host can really do. The async queue moves a miss list
        in two legs that overlap across minibatches: the CPU row gather (latency bound, scales with the threads the
        process may use) and the copy over PCIe. On a host with few free cores (eight ranks sharing a CPU quota, a busy
        neighbour) the gather, not PCIe, bounds the step. The worker's counters give the gather rate of the last jobs;
        the rows it cannot gather within the list's PCIe time are handed to the device, which reads them from the
        pinned table itself (pg_missq_device_tail) — down to share 0, the pure zero-copy path. Shares >= 0.9 round up
        to 1 (a device-side PCIe read slows the concurrent compute kernels: not worth a 10 % shorter gather).
        apply=False only reports. Returns the dict it logged, or None when there is nothing to go by yet (no queue / fewer than `min_jobs` jobs
        since the last call / pageable tables)."""
        st = self.miss_queue_stats()
        if st is None:
            return None
        prev = getattr(self, "_adapt_prev", None)
        jobs = st["jobs"] - (prev["jobs"] if prev else 0)
        if jobs < min_jobs:
            return None
        rows = st["rows_per_job"] * st["jobs"] - (prev["rows_per_job"] * prev["jobs"] if prev else 0.0)
        gather_us = st["us_cpu_gather"] * st["jobs"] - (prev["us_cpu_gather"] * prev["jobs"] if prev else 0.0)
        self._adapt_prev = st
        pinned = getattr(self.graph, "pinned", None)
        if rows <= 0 or gather_us <= 0 or (pinned is not None and not all(pinned.get(n, False) for n in self.dims)):
            return None
        row_bytes = 4 * sum(self.dims.values())
        rate = floor_GBps
        if rate is None:
            eng = [v for b, v in st["sdma_engine_h2d_GBps"].items() if st["sdma_engine_mask"] >> b & 1]
            rate = eng[0] if eng else 50.0
        us_per_row_cpu = gather_us / rows                  # what the gather pool achieves, all its threads together
        us_per_row_pcie = row_bytes / (rate * 1e3)
        want = min(1.0, us_per_row_pcie / us_per_row_cpu)  # share of a list the CPU finishes within the list's PCIe time
        old = self.cpu_share
        # the measured rate belongs to the OLD share's list length; per-row time is roughly length-independent
        new = 1.0 if want >= 0.9 else (0.0 if want < 0.1 else round(want * 16) / 16)
        rec = {"us_per_row_cpu_gather": us_per_row_cpu, "us_per_row_pcie": us_per_row_pcie, "cpu_share_before": old,
               "cpu_share": new, "jobs_measured": int(jobs), "host_threads": self.host_threads}
        if new != old and apply:
            self.apply_cpu_share(new)
        if not quiet:
            print("GraphCacheServer: CPU gather {:.3f} us/row vs PCIe {:.3f} us/row -> cpu_share {} (was {})".format(
                us_per_row_cpu, us_per_row_pcie, new, old))
        return rec

    def apply_cpu_share(self, share):
        """set cpu_share between minibatches (takes effect at the next _missq_buffers call; fetch plans are rebuilt because
        the validity of their dedup depends on it)"""
        self.cpu_share = float(share)
        self._missq_bufs = {}
        self._cache_epoch += 1

    def _dedup_for(self, slot, offsets_rel, first_layer, num_layers, same_fields=True):
        """pg_dedup_t over the slot's dup buffers for a launch whose rows are the NodeFlow layers first_layer.. laid out at
        offsets_rel (0-based, len = layers + 1); None when the launch cannot repeat an id (one layer), the layers read
        different fields, or the queue splits its miss lists with the device (cpu_share < 1). Call after
        _missq_buffers(slot, ...)."""
        n = len(offsets_rel) - 1
        if not (self.dedup_misses and self.miss_mode == "async" and not self.full_cached and slot is not None
                and same_fields and 2 <= n <= L.PG_MAX_LAYERS and self._missq is not None and self._missq_share == 256):
            return None
        bufs = self._missq_dup.get(slot)
        if bufs is None:
            a, b, c = L.vp(), L.vp(), L.vp()
            L.check(self.lib.pg_missq_slot_dup_buffers(self._missq, slot, ctypes.byref(a), ctypes.byref(b), ctypes.byref(c)),
                    "pg_missq_slot_dup_buffers")
            bufs = self._missq_dup[slot] = (a.value, b.value, c.value)
        d = L.PgDedup()
        d.n_ranges = n
        for r in range(n + 1):
            d.lo[r] = int(offsets_rel[r])
        # sampler spec rule 5: every layer but the seeds' (the NodeFlow's last) ascends by id
        d.sorted_mask = sum(1 << r for r in range(n) if first_layer + r < num_layers - 1)
        d.dup_pos, d.dup_src, d.dup_count = bufs
        return d

    def wait_misses(self, slot, stream=None, host_blocking=False):
        """miss_mode == 'async': order `stream` (default: current) after the slot's miss rows. By default
        the wait happens on the GPU (a one-wave kernel sleeping on a flag) and the host returns at once;
        host_blocking=True waits for the worker on the CPU and then uses an event."""
        # (not keyed on miss_mode: a caller may switch paths between batches — bench.py probes both — and a batch
        # submitted to the queue must be waited for whatever the mode is by the time it is consumed)
        # decided per slot, not from full_cached: a batch submitted while the cache was still empty (GraphedTrainer
        # prepares its look-ahead batches before the first step's auto_cache) must be waited for even though every
        # later batch is a pure cache hit
        if self._missq is None or slot not in self._missq_pending:
            return
        self._missq_pending.discard(slot)
        st = stream if stream is not None else torch.cuda.current_stream(self.device)
        if host_blocking or self.host_wait:
            L.check(self.lib.pg_missq_wait(self._missq, slot, L.stream_ptr(st), None), "pg_missq_wait")
        else:
            L.check(self.lib.pg_missq_wait_device(self._missq, slot, L.stream_ptr(st)), "pg_missq_wait_device")

    def wait_worker(self, slot):
        """block the host until the async queue's worker has enqueued the copy of `slot`'s latest submission (no HIP
        call). The launch thread calls it before it enqueues, on ANY stream, a wait for something that happens after
        that submission's consumer (frames consumed, sampler ring slot free) — see pg_missq_wait_idle."""
        if self._missq is not None and slot is not None and 0 <= slot < self._missq_nslots:
            L.check(self.lib.pg_missq_wait_idle(self._missq, int(slot)), "pg_missq_wait_idle")

    def shutdown_miss_queue(self):
        """stop the async queue's worker and gather threads and free its buffers (every submitted batch must have
        been consumed: synchronise the device first)"""
        if self._missq is not None:
            L.check(self.lib.pg_missq_destroy(self._missq), "pg_missq_destroy")
            self._missq, self._missq_rows, self._missq_bufs, self._missq_share = None, 0, {}, None
            self._missq_nslots = 0
            self._missq_dup = {}
            self._missq_pending.clear()
            self._cache_epoch += 1       # fetch plans (and graphs captured over them) hold pointers into the queue's blocks

    def drain_misses(self):
        """block the host until the async queue's worker has enqueued the copy of every submitted batch (no HIP
        call). Call before a device-wide synchronise: see pg_missq_drain."""
        if self._missq is not None:
            L.check(self.lib.pg_missq_drain(self._missq), "pg_missq_drain")

    def miss_queue_stats(self):
        """async queue counters since its creation (None without a queue): jobs, rows, how the consumer was ordered
        after the rows (event vs spin kernel), mean per-job microseconds of the worker's phases"""
        if self._missq is None:
            return None
        st = L.PgMissqStats()
        L.check(self.lib.pg_missq_stats(self._missq, ctypes.byref(st), 0), "pg_missq_stats")
        return {"jobs": int(st.jobs), "rows_per_job": st.rows / max(1.0, st.jobs), "waits_by_event": int(st.waits_by_event),
                "rescued_chunks": int(st.rescued_chunks),  # overdue 32-row chunks of the CPU gather re-executed by the worker
                "spared_jobs": int(st.spared_jobs),        # jobs that took a spare staging buffer instead of waiting for a straggler
                "waits_by_spin_kernel": int(st.waits_by_spin_kernel), "us_submit_to_published": st.us_submit_to_published,
                "us_cpu_gather": st.us_cpu_gather, "us_enqueue": st.us_enqueue, "us_submit_to_done": st.us_submit_to_done,
                "sdma_engine_mask": int(st.sdma_engine_mask),      # 0 = hipMemcpyAsync (the runtime picks the engine)
                # which way the worker's copies go (csrc/pg_missq.hip): straight to one calibrated SDMA engine with the consumer
                # watching the completion signal (the default); the same engine but ordered through the copy stream
                # (PG_MISSQ_NO_DIRECT=1); or hipMemcpyAsync on the copy stream when ROCr's engine interface is not usable
                # (the probe failed, or PG_MISSQ_HSA_COPY=0) — the tested fallback
                "copy_path": ("hipMemcpyAsync on the copy stream (fallback)" if not st.sdma_engine_mask else
                              ("ROCr SDMA engine, ordered through the copy stream" if os.environ.get("PG_MISSQ_NO_DIRECT") == "1"
                               else "ROCr SDMA engine, direct (consumer watches the completion signal)")),
                "sdma_engine_h2d_GBps": {b: round(st.engine_GBps[b], 1) for b in range(16) if st.engine_GBps[b] > 0}}

    def miss_queue_longest(self, reset=False):
        """the longest single occurrence (us) of each of the worker's phases since the last reset — a stall of the miss
        path sits in exactly one of them: waiting for the device to publish the miss list, the CPU row gather, the copy
        submission, or the whole submit -> done span"""
        if self._missq is None:
            return None
        st = L.PgMissqStats()
        L.check(self.lib.pg_missq_stats(self._missq, ctypes.byref(st), 1 if reset else 0), "pg_missq_stats")
        return {"wait_published": round(st.max_us_wait_published, 1), "cpu_gather": round(st.max_us_cpu_gather, 1),
                "enqueue": round(st.max_us_enqueue, 1), "submit_to_done": round(st.max_us_submit_to_done, 1)}

    def miss_copy_log(self, cap=1 << 16):
        """(bytes, ms) of the worker's last host->device copies (needs PG_MISSQ_COPYLOG=1 in the environment)"""
        if self._missq is None:
            return []
        import numpy as np
        b = np.zeros(cap, np.int64)
        m = np.zeros(cap, np.float32)
        n = L.c_i64(0)
        L.check(self.lib.pg_missq_copy_log(self._missq, b.ctypes.data, m.ctypes.data, cap, ctypes.byref(n)),
                "pg_missq_copy_log")
        return list(zip(b[:n.value].tolist(), m[:n.value].tolist()))

    def misses_timed_out(self):
        if self._missq is None:
            return False
        v = ctypes.c_int(0)
        L.check(self.lib.pg_missq_timed_out(self._missq, ctypes.byref(v)), "pg_missq_timed_out")
        return bool(v.value)

    def check_misses(self):
        """raise if a device-side wait for miss rows ever gave up (the worker thread died or stalled > 3 s): the steps
        since then trained on rows that never landed. Synchronises the device; the trainers call it once per epoch."""
        if self.misses_timed_out():
            raise L.PgError("async miss queue: a device-side wait for miss rows timed out (worker thread dead or "
                            "stalled); feature rows of at least one minibatch never landed")

    def close(self):
        """deterministic teardown: wait for the device (kernels of the pipeline may still read the cache, the slot map and the
        miss queue's staged blocks), then stop the miss queue's threads and free its buffers. Idempotent."""
        waited = False
        try:
            if (L.del_waits_enabled() and torch.cuda.is_available() and getattr(self, "device", None) is not None
                    and not torch.cuda.is_current_stream_capturing()):
                torch.cuda.synchronize(self.device)
                waited = True
        except Exception:
            pass
        try:
            if getattr(self, "_missq", None):
                if waited or not torch.cuda.is_available():
                    self.lib.pg_missq_destroy(self._missq)
                else:
                    # The wait had to be skipped (a finalizer running inside a capture of this thread, or PG_NO_DEL_WAIT): a
                    # hipFree inside a capture invalidates it, and the staged blocks may still be read by kernels in flight
                    # The queue is parked and destroyed by the next close() of ANY cacher that could wait.
                    _DEFERRED_MISSQ.append((self.lib, self._missq, getattr(self, "device", None)))
                self._missq = None
            if waited:
                while _DEFERRED_MISSQ:
                    lib_, q_, dev_ = _DEFERRED_MISSQ.pop()
                    if dev_ is not None and dev_ != self.device:
                        torch.cuda.synchronize(dev_)
                    lib_.pg_missq_destroy(q_)
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()
        return False

    def __del__(self):
        # best-effort backstop (close() is the deterministic path). The torch buffers of this object that other streams touch
        # are recorded on those streams by the trainers (L.record_streams): their memory outlives kernels in flight whatever
        # drops the object; the miss queue's own blocks are freed by the library behind hipFree's device-wide wait
        try:
            self.close()
        except Exception:                # (interpreter shutdown: module globals may be gone already)
            pass

    # -- storage.py:207-216 ---------------------------------------------------
    def fetch_from_cache(self, nodeflow, out=None):
        with torch.autograd.profiler.record_function('cache-idxload'):
            nf_nids = nodeflow._node_mapping.tousertensor().to(self.device, torch.int64)
            offsets = nodeflow._layer_offsets
        R = nf_nids.numel()
        names = list(self.gpu_fix_cache)
        with torch.autograd.profiler.record_function('cache-gpu'):
            if out is None:
                out = {name: torch.empty((R, self.dims[name]), dtype=torch.float32, device=self.device) for name in names}
            fields, nf = L.make_fields((self.gpu_fix_cache[name], out[name], self.dims[name],
                                        self.gpu_fix_cache[name].stride(0), out[name].stride(0)) for name in names)
            L.check(self.lib.pg_gather_rows_full(L.ptr(nf_nids), R, fields, nf,
                                                 L.stream_ptr(torch.cuda.current_stream(self.device))),
                    "pg_gather_rows_full")
        for i in range(nodeflow.num_layers):
            nodeflow._node_frames[i] = {name: out[name][offsets[i]:offsets[i + 1]] for name in names}
        if self.log:
            self._stats[0] += int((nf_nids >= 0).sum()) if getattr(nodeflow, 'padded', False) else R

    # -- storage.py:219-227 ---------------------------------------------------
    def log_miss_rate(self, miss_num, total_num):
        self.try_num += total_num
        self.miss_num += miss_num

    def get_miss_rate(self):
        # the per-launch counters live on the device (pg_gather_rows `stats`): one sync here, none per step
        t, m = self._stats.tolist()
        self._stats.zero_()
        self.log_miss_rate(m, t)
        miss_rate = float(self.miss_num) / self.try_num
        self.miss_num = 0
        self.try_num = 0
        return miss_rate
