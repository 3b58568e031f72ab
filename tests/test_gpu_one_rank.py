"""GPU: `call_mods --freq_file` by one rank, end to end: every input form and both parsers under the slot canary, the frequencies fused
into the run against `call_freq` on its result, the fall-back past the device budget, inputs of no row and of one.  (The tests of the
same paths that go on to several ranks on one GPU do not run, tests/conftest.py; what they say of one rank is said here.)"""
import gzip
import os
import socket
import subprocess
import sys

import pytest

from tests.helpers import GOLDEN, ROOT, run_cli_jobs
from tests.test_gpu_canary import _inputs
from tests.test_gpu_cli import _ckpt, _folded_rows, _run_cli

pytestmark = pytest.mark.gpu


def _bytes(path, gz=False):
    return gzip.open(path + ".gz", "rb").read() if gz else open(path, "rb").read()


def _run(tmp_path, jobs, tag="jobs"):
    res = run_cli_jobs(tmp_path, jobs, world=1, tag=tag)
    assert len(res) == len(jobs), (res.proc.stdout[-2000:], res.proc.stderr[-4000:])
    return res


def test_every_input_form_and_parser_under_the_slot_canary(tmp_path):
    ck = _ckpt(tmp_path)
    paths = _inputs(tmp_path, _folded_rows(n_rep=6))     # 1,200 rows, 23 sites
    common = ["-m", ck, "--seed", "31", "--prob_cf", "0.02"]

    def job(tag, fmt, env, *extra):
        out = str(tmp_path / (tag + ".tsv"))
        return {"argv": ["call_mods", "-i", paths[fmt], "-o", out, "--freq_file", out + ".freq"] + common + list(extra), "env": env, "out": out, "gz": "--gzip" in extra}
    jobs = [{"argv": ["pack_features", "-i", paths["plain"], "-o", paths["dspf"]], "env": {}}, job("ref", "plain", {})]
    forms = [(f, p) for f in ("plain", "bgzf", "foreign_gz", "dspf") for p in ("device", "host") if (f, p) != ("dspf", "host")]
    for i, (fmt, parse) in enumerate(forms):   # blocks of a few rows up to the whole file, a writer slower than the GPU or not
        size, delay = [(20000, 0), (61000, 3), (150000, 0), (33000, 11), (400000, 1), (97000, 0), (10_000_000, 0)][i]
        jobs.append(job("c%d" % i, fmt, {"DSP_SLOT_CANARY": "1", "DSP_BLOCK_BYTES": str(size), "DSP_WRITER_DELAY_MS": str(delay)}, "--parse_on", parse,
                        *(["--gzip"] if i % 3 == 2 else [])))
    for j, r in zip(jobs, _run(tmp_path, jobs)):
        assert r["rc"] == 0, (j["argv"], r["stderr"][-3000:])
    calls, freq = _bytes(jobs[1]["out"]), _bytes(jobs[1]["out"] + ".freq")
    assert calls.count(b"\n") == 1200 and len(freq) > 0
    for j in jobs[2:]:
        assert _bytes(j["out"], j["gz"]) == calls and _bytes(j["out"] + ".freq", j["gz"]) == freq, j["argv"]


def test_fused_frequencies_equal_call_freq_on_the_result(tmp_path):
    """on the device and through the host table, tsv and sorted bedMethyl"""
    ck = _ckpt(tmp_path)
    inp = str(tmp_path / "folded.tsv")
    open(inp, "wb").write(_folded_rows(n_rep=6))
    T = lambda name: str(tmp_path / name)
    jobs = []
    for tag, flags, cf_flags in (("tsv", [], []), ("bed", ["--freq_bed", "--freq_sort"], ["--bed", "--sort"])):
        cm = ["call_mods", "-i", inp, "-m", ck, "--prob_cf", "0.02"]
        jobs.append({"argv": cm + ["-o", T(tag + ".calls"), "--freq_file", T(tag + ".fused")] + flags})
        jobs.append({"argv": ["call_freq", "-i", T(tag + ".calls"), "-o", T(tag + ".two_step"), "--prob_cf", "0.02"] + cf_flags})
        jobs.append({"argv": cm + ["-o", T(tag + ".host_calls"), "--freq_file", T(tag + ".host"), "--freq_on", "host"] + flags})
    assert all(r["rc"] == 0 for r in _run(tmp_path, jobs))
    for tag in ("tsv", "bed"):
        want = _bytes(T(tag + ".two_step"))
        assert len(want) > 0 and _bytes(T(tag + ".fused")) == want == _bytes(T(tag + ".host"))
        assert _bytes(T(tag + ".host_calls")) == _bytes(T(tag + ".calls"))


@pytest.mark.parametrize("gz", [False, True])
def test_a_foreign_gz_in_many_blocks(tmp_path, gz):
    ck = _ckpt(tmp_path)
    inp, out = str(tmp_path / "foreign.tsv.gz"), str(tmp_path / "calls.tsv")
    open(inp, "wb").write(gzip.compress(_folded_rows(n_rep=10), 1))
    flags = ["--gzip"] if gz else []
    jobs = [{"argv": ["call_mods", "-i", inp, "-m", ck, "-o", out, "--freq_file", out + ".freq", "--prob_cf", "0.02"] + flags, "env": {"DSP_BLOCK_BYTES": "200000"}},
            {"argv": ["call_freq", "-i", out + (".gz" if gz else ""), "-o", out + ".two_step", "--prob_cf", "0.02"]}]
    for r in _run(tmp_path, jobs):
        assert r["rc"] == 0, r["stderr"][-3000:]
    assert _bytes(out, gz).count(b"\n") == 2000 and _bytes(out + ".freq", gz) == _bytes(out + ".two_step")


def test_past_the_device_budget_the_host_table_gives_the_same_bytes(tmp_path):
    ck = _ckpt(tmp_path)
    inp, out = str(tmp_path / "folded.tsv"), [str(tmp_path / ("calls%d.tsv" % i)) for i in range(2)]
    open(inp, "wb").write(_folded_rows())
    for o, env in zip(out, (None, {"DSP_FREQ_DEV_MAX_BYTES": "10000", "DSP_BLOCK_BYTES": "300000"})):
        r = _run_cli(["-i", inp, "-m", ck, "-o", o, "--freq_file", o + ".freq", "--prob_cf", "0.02", "--seed", "8"], env=env)
        assert r.returncode == 0 and ("exceed the device budget" in r.stderr) == (env is not None), r.stderr[-3000:]
    assert _bytes(out[0]) == _bytes(out[1]) and _bytes(out[0] + ".freq") == _bytes(out[1] + ".freq") != b""


def test_both_parsers_on_odd_rows_and_on_bad_ones(tmp_path):
    """odd but legal spellings take the host parser for their block; a malformed row and an unknown base end the run alike"""
    ck = _ckpt(tmp_path)
    lines = _folded_rows(n_rep=6).split(b"\n")
    w = lines[700].split(b"\t")
    w[7], w[8] = b"+" + w[7], w[8].replace(b",", b",0000000000000000000", 1)
    lines[700] = b" " + b"\t".join(w)
    w = lines[333].split(b"\t")
    w[7] = b",".join([b"-1_0.2_5" if i == 2 else v for i, v in enumerate(w[7].split(b","))])
    lines[333] = b"\t".join(w)
    number, base = lines[:], lines[:]
    w = number[300].split(b"\t")
    w[7] = w[7].replace(b",", b";", 1)
    number[300] = b"\t".join(w)
    w = base[10].split(b"\t")
    w[6] = w[6][:5] + b"X" + w[6][6:]
    base[10] = b"\t".join(w)
    paths = _inputs(tmp_path, b"\n".join(lines))
    jobs = []
    for name, rows in (("number", number), ("base", base)):
        paths[name] = str(tmp_path / name)
        open(paths[name], "wb").write(b"\n".join(rows))
    for fmt in ("plain", "bgzf", "foreign_gz", "number", "base"):
        for parse in ("host", "device"):
            out = str(tmp_path / (fmt + parse))
            jobs.append({"argv": ["call_mods", "-i", paths[fmt], "-m", ck, "-o", out, "--seed", "3", "--freq_file", out + ".freq", "--prob_cf", "0.02", "--parse_on", parse],
                         "env": {"DSP_BLOCK_BYTES": "120000"}, "out": out})
    res = _run(tmp_path, jobs)
    got = []
    for j, r in zip(jobs[:6], res):
        assert r["rc"] == 0, (j["argv"], r["stderr"][-3000:])
        got.append((_bytes(j["out"]), _bytes(j["out"] + ".freq")))
    assert got[0][0].count(b"\n") == 1200 and all(g == got[0] for g in got)
    for r in res[6:8]:
        assert r["rc"] != 0 and "malformed feature row" in r["stderr"] and "signal_means" in r["stderr"]
    for r in res[8:]:
        assert r["rc"] != 0 and "KeyError: 'X'" in r["stderr"]


def test_no_row_one_row_and_two_ranks_on_three(tmp_path):
    ck = _ckpt(tmp_path)
    rows = open(os.path.join(GOLDEN, "f2_rows.tsv"), "rb").read().split(b"\n")[:3]
    T = lambda name: str(tmp_path / name)
    for name, data in (("none", b""), ("one", rows[0]), ("three", b"\n".join(rows) + b"\n")):
        open(T(name), "wb").write(data)
    jobs = [{"argv": ["call_mods", "-i", T(n), "-m", ck, "-o", T(n + ".calls"), "--seed", "3"] + more}
            for n, more in (("none", []), ("one", []), ("three", ["--freq_file", T("three.freq"), "--prob_cf", "0"]))]
    for r in _run(tmp_path, jobs):
        assert r["rc"] == 0, r["stderr"][-2000:]
    assert [_bytes(T(n + ".calls")).count(b"\n") for n in ("none", "one", "three")] == [0, 1, 3] and _bytes(T("three.freq")).count(b"\n") == 3
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", "2", "--master-addr", "127.0.0.1", "--master-port", str(port), "-m",
           "deepsignal_plant_amd.deepsignal_plant", "call_mods", "-i", T("three"), "-m", ck, "-o", T("two_ranks"), "--seed", "3"]
    r = subprocess.run(cmd, cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr[-3000:]
    assert _bytes(T("two_ranks")) == _bytes(T("three.calls"))
