"""SlabExtractor over gloo when its grid lives on a device: gloo must see host tensors only (its collectives on device
tensors have hung when several ranks shared one GPU).  On the CPU the device is played by a tensor subclass that reports
`is_cuda`; the GPU form runs the device path of extract() itself.  Both wrap torch.distributed's calls and compare the
merged mesh with the oracle's mesh of the whole grid."""
import os
import sys
from pathlib import Path

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))

from oracle import canonical_mesh, oracle_extract  # noqa: E402
from tests import test_gpu_slab_dist, test_slab_gloo  # noqa: E402


class DeviceTensor(torch.Tensor):
    """A CPU tensor that says it is on a GPU; `cpu()` is the way off it."""
    is_cuda = property(lambda self: True)

    def cpu(self):
        return self.as_subclass(torch.Tensor).clone()


class DeviceBackend(test_slab_gloo.OracleBackend):
    """The oracle's stand-in backend with its exchanged records on that device."""

    def count_and_vertices(self, grid, *args):
        out = super().count_and_vertices(grid.as_subclass(torch.Tensor), *args)
        self.plane0, self.halo = (t.as_subclass(DeviceTensor) for t in (self.plane0, self.halo))
        return out

    def faces(self, *bases):
        self.halo = self.halo.as_subclass(torch.Tensor)
        return super().faces(*bases)


def _host_only(seen):
    """Wraps every torch.distributed call that extract() makes with tensors."""
    def check(*tensors):
        for t in tensors:
            for u in t if isinstance(t, (list, tuple)) else [t]:
                assert not u.is_cuda, "gloo was handed a device tensor"
        seen.append(len(tensors))

    p2p, gather, gather_into = dist.P2POp, dist.all_gather, dist.all_gather_into_tensor
    dist.P2POp = lambda op, tensor, peer: (check(tensor), p2p(op, tensor, peer))[1]
    dist.all_gather = lambda out, t, **k: (check(out, t), gather(out, t, **k))[1]
    dist.all_gather_into_tensor = lambda out, t, **k: (check(out, t), gather_into(out, t, **k))[1]


def _cpu_worker(rank, world, port, out_dir, shape, thresh, lower, upper):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    from primitive3d_amd.fields import perlin_grid
    from primitive3d_amd.slab import SlabExtractor
    seen = []
    _host_only(seen)
    torch.cuda.synchronize = lambda *a: None
    ex = SlabExtractor(shape, rank, world, torch.device("cpu"), backend=DeviceBackend())
    ex.grid = ex.grid.as_subclass(DeviceTensor)
    ex.fill_local(lambda x0, x1: perlin_grid(shape, period=10, seed=2, x0=x0, x1=x1))
    res = ex.extract(thresh, lower, upper)
    assert len(seen) >= 3   # a plane, its records, the counts
    k = ex.backend.keys[ex.backend.local_id >= 0]
    ry, rz = shape[1], shape[2]
    gk = (k // 3 + ex.x0 * ry * rz) * 3 + k % 3
    np.savez(Path(out_dir) / f"r{rank}.npz", v=res.vertices.numpy(), f=res.faces.numpy(), k=gk)
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 3])
def test_gloo_sees_host_tensors_only(tmp_path, world, built):
    from primitive3d_amd.fields import perlin_grid
    shape, thresh, lower, upper = (13, 9, 20), 0.03, [0.0, 1.0, -2.0], [2.0, 3.0, 4.0]
    port = 33600 + (os.getpid() % 2000) + world
    mp.spawn(_cpu_worker, args=(world, port, str(tmp_path), shape, thresh, lower, upper), nprocs=world, join=True)
    parts = [np.load(tmp_path / f"r{r}.npz") for r in range(world)]
    got = canonical_mesh(*(np.concatenate([p[n] for p in parts]) for n in ("v", "f", "k")))
    ref = canonical_mesh(*oracle_extract(perlin_grid(shape, period=10, seed=2).numpy(), thresh, lower, upper))
    assert all(np.array_equal(a, b) for a, b in zip(got, ref))


def _gpu_worker(*args):
    seen = []
    _host_only(seen)
    test_gpu_slab_dist._worker(*args)
    assert len(seen) >= 6   # two calls of extract(): a plane, its records, the counts


@pytest.mark.gpu
def test_gloo_sees_host_tensors_only_on_the_device_path(tmp_path, gpu, built, monkeypatch):
    monkeypatch.setattr(test_gpu_slab_dist, "_worker", _gpu_worker)   # (in this process: what it spawns)
    test_gpu_slab_dist._run_and_compare(tmp_path, 2, (61, 21, 150), "gloo")
