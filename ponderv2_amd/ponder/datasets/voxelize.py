"""Voxelisation transform that defines the voxel set the backbone sees.

Restates ``GridSample`` of ponder/datasets/transform.py:1078-1213 (train mode :1103-1145; the two
hash functions :1180-1213).  Integer work: the 64-bit hashes wrap mod 2^64 exactly as numpy's
uint64 arithmetic does in the reference, and the same ``np.argsort`` / ``np.random.randint`` calls
are made in the same order so identical seeds pick identical representatives.
"""
import os

import numpy as np

# a teacher's lists of a point (models/losses: TopLogitsDistillLoss), (N, k) each: whatever selects or reorders points takes
# them along where a sample has them
TEACHER_ARRAYS = ("teacher_index", "teacher_logits")

_FNV_OFFSET = np.uint64(14695981039346656037)
_FNV_PRIME = np.uint64(1099511628211)


def fnv_hash_vec(arr):
    """Per-coordinate FNV (multiply, then xor) over the columns of an int array, uint64."""
    assert arr.ndim == 2
    a = arr.astype(np.uint64)
    h = np.full(a.shape[0], _FNV_OFFSET, dtype=np.uint64)
    with np.errstate(over="ignore"):
        for j in range(a.shape[1]):
            h = h * _FNV_PRIME
            h = np.bitwise_xor(h, a[:, j])
    return h


def ravel_hash_vec(arr):
    """Row-major ravel of (coords - min) with per-axis extent max+1, uint64."""
    assert arr.ndim == 2
    a = (arr - arr.min(0)).astype(np.uint64)
    ext = a.max(0).astype(np.uint64) + np.uint64(1)
    keys = np.zeros(a.shape[0], dtype=np.uint64)
    for j in range(a.shape[1] - 1):
        keys += a[:, j]
        keys *= ext[j + 1]
    keys += a[:, -1]
    return keys


class GridSample:
    """One random point per occupied voxel (train mode) + integer grid coordinates."""

    def __init__(self, grid_size=0.05, hash_type="fnv", mode="train",
                 keys=("coord", "color", "normal", "segment"), return_grid_coord=False,
                 return_min_coord=False):
        assert mode == "train", "only the training mode is on the pre-training path"
        self.grid_size = grid_size
        self.hash = fnv_hash_vec if hash_type == "fnv" else ravel_hash_vec
        self.keys = keys
        self.return_grid_coord, self.return_min_coord = return_grid_coord, return_min_coord

    def __call__(self, data_dict):
        scaled = data_dict["coord"] / np.array(self.grid_size)
        grid_coord = np.floor(scaled).astype(int)
        min_coord = grid_coord.min(0) * np.array(self.grid_size)
        grid_coord -= grid_coord.min(0)
        key = self.hash(grid_coord)
        idx_sort = np.argsort(key)
        _, count = np.unique(key[idx_sort], return_counts=True)
        first = np.cumsum(np.insert(count, 0, 0)[0:-1])
        pick = first + np.random.randint(0, count.max(), count.size) % count
        idx_unique = idx_sort[pick]
        if self.return_grid_coord:
            data_dict["grid_coord"] = grid_coord[idx_unique]
        if self.return_min_coord:
            data_dict["min_coord"] = min_coord.reshape([1, 3])
        for k in (*self.keys, *(t for t in TEACHER_ARRAYS if t in data_dict and t not in self.keys)):
            data_dict[k] = data_dict[k][idx_unique]
        return data_dict


# ---------------------------------------------------------------------------------------------
# Device-side voxelisation: the same transform on torch tensors, so it
# can run on the GPU after the raw cloud has been uploaded instead of in a DataLoader worker.
# ---------------------------------------------------------------------------------------------
_SIGN = -(1 << 63)
_KERNELS = __import__("os").environ.get("PV2_VOXELIZE_KERNELS", "1") != "0"


def _as_i64(u):
    u = int(u)
    return u - (1 << 64) if u >= (1 << 63) else u


def fnv_hash_torch(grid):
    """``fnv_hash_vec`` on an integer tensor: int64 arithmetic wraps mod 2^64 exactly like the
    uint64 arithmetic of the numpy version, so the BIT PATTERNS of the keys are identical."""
    import torch

    h = torch.full((grid.shape[0],), _as_i64(_FNV_OFFSET), dtype=torch.int64, device=grid.device)
    prime = _as_i64(_FNV_PRIME)
    for j in range(grid.shape[1]):
        h = (h * prime) ^ grid[:, j].to(torch.int64)
    return h


def ravel_hash_torch(grid):
    import torch

    a = (grid - grid.amin(0)).to(torch.int64)
    ext = a.amax(0) + 1
    keys = torch.zeros(a.shape[0], dtype=torch.int64, device=grid.device)
    for j in range(a.shape[1] - 1):
        keys = (keys + a[:, j]) * ext[j + 1]
    return keys + a[:, -1]


def grid_sample_torch(coord, grid_size, hash_type="fnv", pick=None):
    """Train-mode ``GridSample`` on tensors (any device): -> (idx_unique, grid_coord) with
    ``idx_unique`` one point index per occupied voxel, voxels in ascending UNSIGNED key order (the
    order numpy's argsort on uint64 keys produces) and ``grid_coord`` their integer coordinates.

    ``pick`` (n_voxels,) integers plays the role of the reference's
    ``np.random.randint(0, count.max(), n_voxels)``: the representative of a voxel is its
    ``pick % count``-th member in point-index order (a stable sort; numpy's unstable argsort may
    order the members of a voxel differently, so representatives - not voxels - can differ from the
    host transform even for equal draws).  ``None`` draws them on the tensor's device."""
    import torch

    scaled = coord.double() / grid_size  # the host transform divides by a float64 array
    grid = torch.floor(scaled).to(torch.int64)
    grid = grid - grid.amin(0)
    key = fnv_hash_torch(grid) if hash_type == "fnv" else ravel_hash_torch(grid)
    order = torch.sort(key ^ _SIGN, stable=True).indices  # signed order of key^2^63 == unsigned order
    skey = key[order]
    first = torch.ones_like(skey, dtype=torch.bool)
    first[1:] = skey[1:] != skey[:-1]
    start = torch.nonzero(first).flatten()
    count = torch.diff(start, append=start.new_tensor([skey.numel()]))
    if pick is None:
        pick = torch.randint(0, int(count.max()), (count.numel(),), device=coord.device)
    # (draws are reduced modulo the LARGEST member count first - a no-op for the reference's own draws,
    # ``randint(0, count.max())`` - and then modulo the voxel's: exactly what the device kernel does with
    # caller-supplied or raw 31-bit draws, so the two paths pick the same point for ANY draw)
    idx_unique = order[start + (pick.to(start.device) % count.max()) % count]
    return idx_unique, grid[idx_unique]


def grid_sample_device(coord, grid_size, hash_type="fnv", pick=None):
    """``grid_sample_torch`` on the hand-written kernels of csrc/voxelize.hip (device tensors only): the
    raw points are de-duplicated through a hash table keyed by the reference's own 64-bit key and only
    the unique keys are sorted - instead of two 64-bit sorts of every raw point.  Same voxel set, same
    order, same representatives for equal draws; one device -> host read (the voxel count)."""
    import torch

    from ponderv2_amd import _lib
    from ponderv2_amd.kernels import _ptr, _stream

    assert coord.is_cuda and coord.dim() == 2 and coord.shape[1] == 3
    if coord.dtype not in (torch.float32, torch.float64):
        coord = coord.float()
    coord = coord.contiguous()
    dev, n = coord.device, coord.shape[0]
    L, st = _lib.lib(), _stream(coord)
    table = 1 << max(int(2 * n - 1).bit_length(), 4)
    i32 = dict(dtype=torch.int32, device=dev)
    tkeys = torch.full((table,), -1, dtype=torch.int64, device=dev)          # 0xff..ff = empty
    ints = torch.zeros(table + 2, **i32)                                    # table counts | n_vox | max count
    tcount, n_vox_dev, max_count = ints[:table], ints[table:table + 1], ints[table + 1:]
    grid, slot_of = torch.empty((n, 3), **i32), torch.empty(n, **i32)
    ukeys, uslot = torch.empty(n, dtype=torch.int64, device=dev), torch.empty(n, **i32)
    minmax = torch.empty(6, dtype=torch.int64, device=dev)
    _lib.check(L.pv2_voxelize_stage1(
        _ptr(coord), int(coord.dtype == torch.float64), n, float(grid_size), int(hash_type != "fnv"),
        _ptr(minmax), _ptr(tkeys), _ptr(tcount), table, _ptr(grid), _ptr(slot_of), _ptr(ukeys), _ptr(uslot),
        _ptr(n_vox_dev), st), "pv2_voxelize_stage1")
    n_vox = int(n_vox_dev.item())                                           # the one host read
    if pick is None:   # raw draws; the kernel reduces them modulo the largest member count, then the voxel's
        pick = torch.randint(0, 2 ** 31 - 1, (n_vox,), device=dev)
    pick = pick.to(dev, torch.int64).contiguous()
    assert pick.numel() == n_vox, (pick.numel(), n_vox)
    skeys, sslot = torch.empty(n_vox, dtype=torch.int64, device=dev), torch.empty(n_vox, **i32)
    rank = torch.empty(table, **i32)
    per_vox = torch.zeros(3 * n_vox, **i32)                                 # count | start | cursor (zeroed)
    members = torch.empty(n, **i32)
    ws_bytes = int(L.pv2_voxelize_workspace_bytes(n_vox))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    idx_unique = torch.empty(n_vox, dtype=torch.int64, device=dev)
    grid_coord = torch.empty((n_vox, 3), dtype=torch.int64, device=dev)
    _lib.check(L.pv2_voxelize_stage2(
        n, n_vox, _ptr(ukeys), _ptr(uslot), _ptr(tcount), _ptr(slot_of), _ptr(grid), _ptr(pick), _ptr(skeys),
        _ptr(sslot), _ptr(rank), _ptr(per_vox[:n_vox]), _ptr(per_vox[n_vox:2 * n_vox]),
        _ptr(per_vox[2 * n_vox:]), _ptr(members), _ptr(max_count), _ptr(ws), ws_bytes, _ptr(idx_unique),
        _ptr(grid_coord), st), "pv2_voxelize_stage2")
    return idx_unique, grid_coord


_INPUT_STREAMS = {}


class input_stream:
    """``with input_stream(device): ...`` - the device half of the input pipeline (upload, GridSample) on
    its OWN stream.  The transform reads the voxel count back to the host; on the training stream that
    read waits for everything the trainer has queued (the whole previous step: the host then runs in
    lock-step with the GPU, +6 ms per step measured); on a stream that carries only the batch's own
    work it returns in microseconds.  On exit the training stream is made to wait for the input
    stream, and the tensors handed over (``adopt``) are marked as used by it."""

    def __init__(self, device):
        import torch

        self.device = torch.device(device)
        self.on = self.device.type == "cuda"
        if self.on:
            key = self.device.index if self.device.index is not None else torch.cuda.current_device()
            if key not in _INPUT_STREAMS:
                # (high priority: short kernels whose result the host waits for)
                _INPUT_STREAMS[key] = torch.cuda.Stream(
                    device=self.device, priority=int(os.environ.get("PV2_INPUT_PRIORITY", "-1")))
            self.side = _INPUT_STREAMS[key]

    def __enter__(self):
        import torch

        if self.on:
            self.cur = torch.cuda.current_stream(self.device)
            self.ctx = torch.cuda.stream(self.side)
            self.ctx.__enter__()
        return self

    def __exit__(self, *exc):
        if self.on:
            self.ctx.__exit__(*exc)
            self.cur.wait_stream(self.side)
        return False

    def adopt(self, batch):
        """The batch's tensors were allocated on the input stream and will be read (and later freed)
        under the training stream."""
        import torch

        if self.on:
            # (tensors, and what a model's prefetch hook added: nested dicts / tuples / rulebooks)
            from ponderv2_amd.kernels import _record_stream

            _record_stream(batch, self.cur)
        return batch


def device_grid_sample(batch, grid_size=0.02, hash_type="fnv", keys=("coord", "feat", "segment"),
                       picks=None):
    """Train-mode GridSample of a collated batch of RAW points on whatever device the batch lives
    on (the GPU, after the trainer's host->device copy): per scene - the rows between consecutive
    ``offset`` entries - one representative per occupied voxel, in the host transform's voxel order
    (``grid_sample_torch``).  Rewrites ``keys``, a teacher's lists and ``offset`` and adds
    ``grid_coord``; every other entry (images, poses, ...) passes through.  This is the device half of SURVEY 8(f) F3: the
    loader workers then only stream raw points (``voxelize=False`` on the synthetic datasets).
    ``picks``: optional list of per-scene tensors standing in for the transform's random draws."""
    import torch

    ends = batch.get("offset_host") or batch["offset"].tolist()   # one read of B small numbers
    out = {k: [] for k in (*keys, *TEACHER_ARRAYS) if k in batch}
    grids, new_ends, start = [], [], 0
    for b, end in enumerate(ends):
        # device tensors: the HIP hash-insert / segmented-pick kernels (csrc/voxelize.hip); host
        # tensors (tests, CPU-only boxes): the same transform composed of torch ops
        sample = grid_sample_device if (batch["coord"].is_cuda and _KERNELS) else grid_sample_torch
        idx, grid = sample(batch["coord"][start:end], grid_size, hash_type,
                           None if picks is None else picks[b])
        for k in out:
            out[k].append(batch[k][start:end][idx])
        grids.append(grid)
        new_ends.append((new_ends[-1] if new_ends else 0) + int(idx.numel()))
        start = end
    res = dict(batch)
    for k, parts in out.items():
        res[k] = torch.cat(parts)
    res["grid_coord"] = torch.cat(grids)
    # the backbone's spatial shape (max grid coordinate + 96, spconv_unet_v1m1_base.py:248 of the
    # reference) read here, where the voxel counts are read anyway: the model then needs no
    # device->host read of its own and the geometry can be prefetched a batch ahead
    res["sparse_shape"] = torch.add(res["grid_coord"].amax(0), 96).tolist()
    res["offset"] = torch.tensor(new_ends, dtype=batch["offset"].dtype).to(batch["offset"].device)
    if "offset_host" in batch:
        res["offset_host"] = list(new_ends)
    return res
