"""CPU: the sharded call_freq (call_mods_freq.DeviceSiteFrequency) over several ranks, from its blocks to rank 0's table: the collectives
on gloo with host tensors, the kernels (csrc/dsp_freq_dev.hip) through the interpreter of tests/native/emu.  And which aggregator
call_mods takes where ranks share a GPU."""
import contextlib
import ctypes
import faulthandler
import os
import socket
import types

import numpy as np
import pytest

from tests.helpers import GOLDEN, ROOT, cached_build
from tests.test_call_freq import CALLS, _rows_from_calls

CLANG = "/opt/rocm/lib/llvm/bin/clang++"
EMU = os.path.join(ROOT, "tests", "native", "emu")
CSRC = os.path.join(ROOT, "deepsignal_plant_amd", "csrc")
NAME, OTHER = b"chr", b"c\xff\xe9"     # no UTF-8
RUNS = (("tsv", {}), ("bed_sorted", dict(bed=True, sort=True)), ("tsv_cf0", dict(prob_cf=0.0)), ("bed_cf02", dict(bed=True, prob_cf=0.2)))


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _join(rank, world, port):
    import torch.distributed as dist
    faulthandler.dump_traceback_later(100, exit=True)   # a rank that waits for ever says where
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    return dist


class _Library(object):
    """the product library's host functions, the interpreter's kernels"""

    def __init__(self, host, kernels):
        self.host, self.kernels = host, kernels

    def __getattr__(self, name):
        fn = getattr(self.host, name)
        if not name.startswith("dsp_freq_dev_"):
            return fn
        k = getattr(self.kernels, name)
        k.restype, k.argtypes = fn.restype, fn.argtypes
        return k


def _on_the_host(so):
    """the aggregator's device is the host: streams and devices mean nothing"""
    import torch
    from deepsignal_plant_amd import _native as nat
    lib = _Library(nat.lib(), ctypes.CDLL(so))
    nat.lib = lambda: lib
    nothing = lambda *a, **k: contextlib.nullcontext()
    torch.cuda.device = torch.cuda.stream = nothing
    torch.cuda.set_device = lambda d: None
    torch.cuda.current_stream = lambda d=None: types.SimpleNamespace(cuda_stream=None)
    torch.Tensor.record_stream = lambda self, s: None
    os.environ["DSP_FREQ_DEV_MAX_BYTES"] = str(1 << 30)


def _shard(rank, world, port, so, outdir):
    dist = _join(rank, world, port)
    _on_the_host(so)
    import torch
    from deepsignal_plant_amd import call_mods_freq as cf
    r, probs, labels = _rows_from_calls(open(CALLS).read().splitlines())
    r.text = np.frombuffer(r.text.tobytes().replace(NAME, OTHER), np.uint8)
    shares = [1, 0, 3, 2, 0, 5, 1, 1][:world] if world > 2 else [1] * world   # ranks without a row among them
    cuts = (np.cumsum([0] + shares) * r.n // sum(shares)).tolist()
    a, b = cuts[rank], cuts[rank + 1]
    for tag, kw in RUNS:     # one after the other in one process group, as a launch of several call_mods is
        agg = cf.DeviceSiteFrequency(kw.get("prob_cf", 0.5), "cpu", nthreads=2)
        for at in range(a, b, 700):
            to = min(b, at + 700)
            agg.add_block(r, torch.from_numpy(probs[at:to]), torch.from_numpy(labels[at:to]), at, at, to)
        assert agg.can_finish(world)
        table = agg.finish(rank, world)
        assert (table is None) == (rank != 0)
        if rank == 0:
            open(os.path.join(outdir, tag), "wb").write(table.format(kw.get("sort", False), kw.get("bed", False)))
            open(os.path.join(outdir, tag + ".n"), "w").write("%d" % table.counts()[0])
        dist.barrier()
    dist.destroy_process_group()
    faulthandler.cancel_dump_traceback_later()


@pytest.mark.skipif(not os.path.exists(CLANG), reason="the image's clang++ builds the interpreter")
@pytest.mark.parametrize("world", [2, 3, 8])
def test_the_shards_tables_are_the_references_bytes_whatever_the_names(tmp_path, world):
    """four runs in one launch; chromosome names that are not UTF-8, other ones in every shard, shards without a row"""
    import torch.multiprocessing as mp
    so = cached_build([CLANG, "-std=c++17", "-O2", "-Wno-psabi", "-fPIC", "-shared", "-DDSP_EMU", "-ffp-contract=off", "-Wno-unused-value", "-I", EMU, "-I",
                       os.path.join(ROOT, "include"), "-I", CSRC, os.path.join(EMU, "last_error.cpp"), os.path.join(EMU, "hip_emu.cpp"), "-x", "c++",
                       os.path.join(CSRC, "dsp_freq_dev.hip"), "-pthread"], "libdsp_freq_ranks.so")
    mp.start_processes(_shard, args=(world, _free_port(), so, str(tmp_path)), nprocs=world, join=True, start_method="spawn")
    for tag, _ in RUNS:
        want = open(os.path.join(GOLDEN, "f5_freq_%s.txt" % tag), "rb").read()
        assert NAME in want and (tmp_path / tag).read_bytes() == want.replace(NAME, OTHER), tag
        assert int((tmp_path / (tag + ".n")).read_text()) == sum(1 for _ in open(CALLS))


def _choice(rank, world, port, outdir):
    dist = _join(rank, world, port)
    import torch
    from deepsignal_plant_amd import call_modifications as cm
    args = types.SimpleNamespace(freq_file="x", freq_on="device", prob_cf=0.5)
    assert cm._make_freq(args, torch.device("cuda", 0), world, 1) == (None, None)
    assert args._freq_from_file is True
    assert cm._make_freq(types.SimpleNamespace(freq_file=None), torch.device("cuda", 0), world, 1) == (None, None)
    cm._finish_freq(args, None, None, rank, world)
    open(os.path.join(outdir, "ok%d" % rank), "w").close()
    dist.destroy_process_group()
    faulthandler.cancel_dump_traceback_later()


def test_ranks_that_share_a_gpu_take_the_host_table(tmp_path, capfd):
    """gloo under call_mods means fewer GPUs than ranks: the frequencies come from the merged per-read file, and rank 0 says so"""
    import torch.multiprocessing as mp
    mp.start_processes(_choice, args=(2, _free_port(), str(tmp_path)), nprocs=2, join=True, start_method="spawn")
    assert sorted(os.listdir(str(tmp_path))) == ["ok0", "ok1"]
    assert capfd.readouterr().err.count("[call_freq] 2 ranks share") == 1
