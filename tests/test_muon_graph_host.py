"""What a recorded Muon step's graph reads, on the CPU: its launches are stubbed, the tables are
the real ones (built for the host), and a graph's reads are the addresses that the recorded launch
was given."""
import ctypes
import gc
import weakref

import numpy as np
import pytest
import torch

import mi_adamw
from mi_adamw import _lib
from mi_adamw import muon as M

CPU = torch.device("cpu")


class Library:
    """The library with the two launches of a step taken down instead of made."""

    def __init__(self):
        self.real = _lib.load()
        self.steps = []

    def __getattr__(self, name):
        return getattr(self.real, name)

    def mi_adamw_muon_step(self, rows, matrices, tables, hyper, options, flags, ws, stream):
        t = _lib.MuonTables.from_address(tables)
        self.steps.append({"rows": rows, "matrices": matrices, "stream": stream,
                           "items": [p for p in t.items if p]})
        return _lib.OK

    def mi_adamw_set_grads(self, rows, n_rows, n, index, grads, vec, stream):
        at = np.frombuffer((ctypes.c_byte * (n_rows * M._ROW_DTYPE.itemsize)).from_address(rows),
                           dtype=M._ROW_DTYPE)
        idx = np.ctypeslib.as_array((ctypes.c_int32 * n).from_address(index))
        at["grad"][idx] = np.ctypeslib.as_array((ctypes.c_uint64 * n).from_address(grads))
        return _lib.OK


class Machine:
    def __init__(self):
        self.stream, self.capturing = 0, False


@pytest.fixture
def machine(monkeypatch):
    m = Machine()
    m.lib = Library()
    monkeypatch.setattr(_lib, "load", lambda *a: m.lib)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: m.stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: m.capturing)
    return m


def optimizer(**options):
    params = [torch.nn.Parameter(torch.randn(s)) for s in ((70, 90), (200, 300), (150, 40))]
    opt = mi_adamw.Muon(params, **options)
    for p in params:
        p.grad = torch.randn(p.shape)
        opt.state[p]["momentum_buffer"] = torch.zeros_like(p)
    return opt, params


def step(opt):
    groups = [[(p, p.grad, opt.state[p]["momentum_buffer"]) for p in g["params"]
               if p.grad is not None] for g in opt.param_groups]
    with torch.no_grad():
        opt._launch(groups, CPU)


def capture(opt, machine):
    """The launches that a graph takes down, and weak references to all that they read."""
    machine.capturing = True
    before = len(machine.lib.steps)
    try:
        step(opt)
    finally:
        machine.capturing = False
    read = {}
    for b in (b for batches in opt._batches for b in batches):
        for t in (b.rows, b.matrices, *(i for i in b.items if i is not None)):
            read[t.data_ptr()] = weakref.ref(t)
        for p in b.params:
            for t in (p.grad, opt.state[p]["momentum_buffer"]):
                read[t.data_ptr()] = weakref.ref(t)
    for launch in machine.lib.steps[before:]:
        assert {launch["rows"], launch["matrices"], *launch["items"]} <= read.keys()
    return read


def alive(read):
    gc.collect()
    return all(r() is not None and r().data_ptr() == at for at, r in read.items())


def move(params):
    for p in params:
        p.grad = torch.randn(p.shape)


def rebuild_by_options(opt, params):
    opt.param_groups[0]["ns_steps"] = 4


def rebuild_by_a_missing_gradient(opt, params):
    params[1].grad = None


def rebuild_by_loading(opt, params):
    opt.load_state_dict({"state": {k: {"momentum_buffer": torch.ones_like(p)}
                                   for k, p in enumerate(params)},
                         "param_groups": opt.state_dict()["param_groups"]})


@pytest.mark.parametrize("moved", [False, True])
@pytest.mark.parametrize("rebuild", [rebuild_by_options, rebuild_by_a_missing_gradient,
                                     rebuild_by_loading])
def test_a_graph_keeps_what_it_reads(machine, moved, rebuild):
    opt, params = optimizer()
    step(opt)
    read = capture(opt, machine)
    rows = {a: r().clone() for a, r in read.items() if r().dtype == torch.uint8}
    if moved:
        move(params)
        step(opt)                   # new rows beside the recorded ones
        move(params)
        step(opt)                   # these may change
    rebuild(opt, params)
    step(opt)
    move([p for p in params if p.grad is not None])
    step(opt)
    assert alive(read)
    assert all(torch.equal(read[a](), t) for a, t in rows.items())


def test_two_graphs_of_one_set_of_tables(machine):
    opt, params = optimizer(bf16_copy=True)
    step(opt)
    first = capture(opt, machine)
    move(params)
    step(opt)
    second = capture(opt, machine)
    move(params)
    step(opt)
    rebuild_by_options(opt, params)
    step(opt)
    assert alive(first) and alive(second)


def test_tables_that_no_graph_reads_end(machine):
    opt, params = optimizer()
    step(opt)
    tables = [weakref.ref(b.matrices) for batches in opt._batches for b in batches]
    rebuild_by_options(opt, params)
    step(opt)
    gc.collect()
    assert all(t() is None for t in tables) and not opt._kept


def batches(opt):
    return [b for of_group in opt._batches for b in of_group]


def test_a_capture_on_another_stream(machine):
    """torch.cuda.graph() captures on a stream of its own."""
    opt, params = optimizer(bf16_copy=True)
    step(opt)
    built = batches(opt)
    machine.stream = 7
    read = capture(opt, machine)
    assert batches(opt) == built and {s["stream"] for s in machine.lib.steps} == {0, 7}
    machine.stream = 0
    move(params)
    step(opt)
    assert batches(opt) == built and alive(read)


def test_streams_in_turn_build_nothing(machine):
    opt, params = optimizer()
    step(opt)
    built = batches(opt)
    for machine.stream in (1, 0, 2, 1):
        step(opt)
        move(params)
    assert batches(opt) == built


def test_a_refused_capture_leaves_the_tables(machine):
    opt, params = optimizer()
    step(opt)
    built = batches(opt)
    kept = [p.grad for p in params]
    params[0].grad = torch.randn(params[0].shape)
    before = len(machine.lib.steps)
    with pytest.raises(RuntimeError, match="under graph capture"):
        capture(opt, machine)
    opt.param_groups[0]["ns_steps"] = 3
    with pytest.raises(RuntimeError, match="under graph capture"):
        capture(opt, machine)
    opt.param_groups[0]["ns_steps"] = 5
    assert len(machine.lib.steps) == before and not any(b.kept for b in built)
    params[0].grad = kept[0]
    step(opt)
    assert batches(opt) == built


def test_a_capture_without_its_copies_is_refused(machine):
    opt, params = optimizer(bf16_copy=True)
    step(opt)
    opt._copies.clear()
    with pytest.raises(RuntimeError, match="under graph capture"):
        capture(opt, machine)
    assert not opt._copies


def test_a_step_raises_the_versions_of_all_it_writes(machine):
    opt, params = optimizer(bf16_copy=True)
    written = [t for p in params
               for t in (p, opt.state[p]["momentum_buffer"], opt.bf16_param(p))]
    for _ in range(2):
        before = [t._version for t in written]
        step(opt)
        assert all(t._version > v for t, v in zip(written, before))
    params[0].grad = None
    before = params[0]._version
    step(opt)
    assert params[0]._version == before
