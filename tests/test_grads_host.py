"""Gradient clipping without a GPU: refusals, and the ranks' powers over gloo."""
import ctypes
import os
import socket
from array import array

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _norm_worker(rank, world, port, out_dir):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    from object_detection_amd.dist import all_reduce_norm_power
    inf, nan = float("inf"), float("nan")
    out = {}
    for name, p, values in (("two", 2.0, (3.0, 4.0)), ("one", 1.0, (3.0, nan)), ("max", inf, (2.0, 7.0)), ("max_inf", inf, (inf, 1.0)),
                            ("max_nan_first", inf, (nan, 1.0)), ("max_nan_second", inf, (5.0, nan)), ("max_nan_inf", inf, (inf, nan))):
        mine = torch.tensor([values[rank]], dtype=torch.float64)
        out[name] = all_reduce_norm_power(mine, p)
        assert torch.equal(torch.nan_to_num(mine), torch.nan_to_num(torch.tensor([values[rank]], dtype=torch.float64)))
    torch.save(out, os.path.join(out_dir, f"n{rank}.pt"))
    dist.barrier()
    dist.destroy_process_group()


def test_two_rank_norm_power(tmp_path):
    mp.spawn(_norm_worker, args=(2, _free_port(), str(tmp_path)), nprocs=2, join=True)
    for k in range(2):
        r = torch.load(tmp_path / f"n{k}.pt")
        assert float(r["two"]) == 7.0 and float(r["max"]) == 7.0 and float(r["max_inf"]) == float("inf")
        assert all(bool(torch.isnan(r[n]).all()) for n in ("one", "max_nan_first", "max_nan_second", "max_nan_inf"))
        assert all(v.dtype == torch.float64 and v.shape == (1,) for v in r.values())


def test_no_process_group_leaves_the_power():
    from object_detection_amd.dist import all_reduce_norm_power
    p = torch.tensor([2.5], dtype=torch.float64)
    got = all_reduce_norm_power(p, 2.0)
    assert torch.equal(got, p) and got.data_ptr() != p.data_ptr()


def test_no_cpu_path():
    from object_detection_amd.grads import clip_grad_norm_, clip_grads, total_grad_norm
    g = torch.ones(4)
    for call in (lambda: total_grad_norm([g]), lambda: clip_grads([g], 1.0)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    q = torch.nn.Parameter(torch.zeros(4))
    q.grad = g
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        clip_grad_norm_([q], 1.0)
    with pytest.raises(TypeError):
        clip_grads([None], 1.0)
    with pytest.raises(ValueError):
        clip_grads([g], 1.0, norm_type=0.5)
    with pytest.raises(ValueError):
        clip_grads([g], -1.0)


def test_entries_refuse_bad_arguments():
    """Argument errors come back before anything is launched (addresses are never read)."""
    from object_detection_amd import _lib as L
    lib = L.lib()
    at = lambda a: a.buffer_info()[0]
    n, p = array("q", [10000, 0, 5]), array("Q", [4096, 0, 8192])
    assert lib.dh_grad_parts(at(n), 3) == 3 and lib.dh_grad_parts(at(n), 0) == 0
    assert lib.dh_grad_parts(at(array("q", [-1])), 1) == 0
    many = array("q", [1 << 30] * 130)
    assert lib.dh_grad_parts(at(many), 130) == 1024
    many = array("q", [1 << 30] * 300)
    assert lib.dh_grad_parts(at(many), 300) == 2 * 1024
    assert lib.dh_grad_parts(at(array("q", [1 << 39] * 17)), 17) == 0          # more chunks than an int counts
    power = lambda grads=at(p), n=at(n), count=3, dtype=0, norm=2, partial=4096, parts=3: lib.dh_grad_power(grads, n, count, dtype, norm, partial, parts, None)
    assert power(count=-1) == -1 and power(grads=None) == -1 and power(n=None) == -1
    assert power(dtype=3) == -1 and power(norm=3) == -1 and power(partial=None) == -1 and power(parts=2) == -4
    assert power(grads=at(array("Q", [4098, 0, 8192]))) == -3 and power(grads=at(array("Q", [0, 0, 8192]))) == -1
    assert lib.dh_grad_norm(None, 1, 2, None, None, 4096, None) == -1
    assert lib.dh_grad_norm(4096, 1, 2, None, None, None, None) == -1
    assert lib.dh_grad_norm(4096, 1, 7, None, None, 4096, None) == -1

    def clip(out=at(p), dtype=0, out_dtype=0, norm=2, limit=1.0, parts=3):
        return lib.dh_grad_clip(at(p), out, at(n), 3, dtype, out_dtype, norm, 4096, parts, None, ctypes.c_double(limit), 4096, None)
    assert clip(limit=-1.0) == -1 and clip(limit=float("nan")) == -1 and clip(out=None) == -1
    assert clip(dtype=0, out_dtype=1) == -1 and clip(dtype=1, out_dtype=2) == -1 and clip(norm=-1) == -1 and clip(parts=-1) == -1
    assert clip(out=at(array("Q", [4097, 0, 8192]))) == -3
