"""
Which process groups make a capture hold only its own thread to the capture rules (pygho_amd/graphs.py): every one with RCCL, not only a default
group that was asked for by that name.  CPU only.
"""
import pytest


@pytest.mark.parametrize("default,configs,mode", [
    ("undefined", ["cpu:gloo,cuda:nccl"], "thread_local"),      # init_process_group() without a backend on a machine with GPUs
    ("undefined", ["cpu:gloo"], "global"),                      # and on one without
    ("gloo", ["cpu:gloo", "cuda:nccl"], "thread_local"),        # a second group by new_group(backend="nccl")
    ("gloo", ["cpu:gloo", "cpu:gloo"], "global"),
    ("nccl", ["cuda:nccl"], "thread_local"),
])
def test_capture_mode_looks_at_every_group(monkeypatch, default, configs, mode):
    import torch.distributed as dist
    from pygho_amd import graphs
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_backend", lambda *a: default)
    monkeypatch.setattr(dist, "get_backend_config", lambda group=None: configs[int(group)])
    for i in range(len(configs)):
        monkeypatch.setitem(dist.distributed_c10d._world.pg_map, str(i), None)
    assert graphs._capture_mode() == mode


def test_capture_mode_of_real_groups(tmp_path):
    """groups of one CPU process: the backend that torch picks by itself, and a second group"""
    import torch.distributed as dist
    from pygho_amd import graphs
    assert not dist.is_initialized()
    dist.init_process_group(init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        dist.new_group([0], backend="gloo")
        want = "thread_local" if "nccl" in str(dist.get_backend_config()) else "global"
        assert graphs._capture_mode() == want
    finally:
        dist.destroy_process_group()
    assert graphs._capture_mode() == "global"
