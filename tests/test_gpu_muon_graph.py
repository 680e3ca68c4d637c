"""Muon steps recorded into HIP graphs, replayed between eager steps that move gradients and rebuild
tables: every replay equals an eager step of a twin with the recorded gradients, bit for bit."""
import copy

import pytest
import torch

import mi_adamw

pytestmark = pytest.mark.gpu

DEV = "cuda"
SHAPES = [(96, 64), (300, 180), (200, 200), (64, 520)]


def make(seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.nn.Parameter(0.02 * torch.randn(s, device=DEV, generator=g)) for s in SHAPES]


def set_grads(params, seed):
    g = torch.Generator(device=DEV).manual_seed(100 + seed)
    for p in params:
        p.grad = 1e-3 * torch.randn(p.shape, device=DEV, generator=g)


def twin_of(opt, params, **options):
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    twin = mi_adamw.Muon(twins, **options)
    twin.load_state_dict(copy.deepcopy(opt.state_dict()))
    return twin, twins


def eager(opt, params, grads):
    for p, g in zip(params, grads):
        p.grad = None if g is None else g.clone()
    opt.step()


def occupy():
    """Memory that was freed is taken and written over."""
    junk = [torch.full((n,), 0x7b, dtype=torch.uint8, device=DEV)
            for n in (512, 512, 2048, 4096, 1 << 16) * 20]
    torch.cuda.synchronize()
    return junk


def same(params, twins):
    return all(torch.equal(p, q) for p, q in zip(params, twins))


def test_replays_after_moved_gradients_and_rebuilt_tables():
    options = dict(lr=0.02)
    params = make()
    opt = mi_adamw.Muon(params, **options)
    set_grads(params, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            opt.step()
        recorded = [p.grad.clone() for p in params]
        twin, twins = twin_of(opt, params, **options)
        for k in range(3):
            set_grads(params, 2 * k + 1)                # moved
            grads = [p.grad for p in params]
            opt.step()
            eager(twin, twins, grads)
            set_grads(params, 2 * k + 2)
            params[k].grad = None                       # other tables
            grads = [p.grad for p in params]
            opt.step()
            eager(twin, twins, grads)
            assert same(params, twins)
            junk = occupy()
            graph.replay()
            eager(twin, twins, recorded)
            torch.cuda.synchronize()
            assert same(params, twins)
            del junk
    torch.cuda.current_stream().wait_stream(side)


def test_plain_capture_after_eager_steps_on_the_default_stream():
    """The usual order: eager steps on the current stream, then torch.cuda.graph(), which captures
    on a stream of its own."""
    options = dict(lr=0.02, bf16_copy=True)
    params = make(1)
    opt = mi_adamw.Muon(params, **options)
    set_grads(params, 0)
    opt.step()
    twin, twins = twin_of(opt, params, **options)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(4):
        for p in params:
            p.grad.mul_(-0.5)
        graph.replay()
        eager(twin, twins, [p.grad for p in params])
        torch.cuda.synchronize()
        assert same(params, twins)
        assert all(torch.equal(opt.bf16_param(p), p.detach().bfloat16()) for p in params)


def test_streams_in_turn():
    options = dict(lr=0.02)
    params = make(2)
    opt = mi_adamw.Muon(params, **options)
    twin, twins = twin_of(opt, params, **options)
    streams = [torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(7):
        stream, last = streams[k % 3], streams[(k - 1) % 3]
        stream.wait_stream(last)
        with torch.cuda.stream(stream):
            set_grads(params, k)
            if k == 4:
                params[1].grad = None                   # other tables, the old ones still queued
            opt.step()
            junk = occupy() if k == 5 else None
    torch.cuda.synchronize()
    for k in range(7):
        set_grads(twins, k)
        if k == 4:
            twins[1].grad = None
        twin.step()
    assert same(params, twins)


def test_a_backward_through_stepped_copies_raises():
    """The forward of bf16_weights saves the copies that the step writes."""
    model = torch.nn.Sequential(torch.nn.Linear(64, 96, bias=False),
                                torch.nn.Linear(96, 64, bias=False)).to(DEV)
    opt = mi_adamw.Muon(model.parameters(), lr=0.02, bf16_copy=True)
    x = torch.randn(8, 64, device=DEV)

    def forward():
        with torch.autocast("cuda", dtype=torch.bfloat16), mi_adamw.bf16_weights(opt, model):
            return model(x).float().square().mean()

    forward().backward()
    late = forward()
    opt.step()
    with pytest.raises(RuntimeError, match="modified (by an )?inplace"):
        late.backward()
    opt.zero_grad()
    forward().backward()
    opt.step()


@pytest.mark.parametrize("optimizer", [mi_adamw.Muon, mi_adamw.FusedAdamW])
def test_a_context_held_open_over_steps(optimizer):
    """The copies are rewritten in place: the forward after a step takes the new weights."""
    def run(held):
        torch.manual_seed(0)
        model = torch.nn.Sequential(torch.nn.Linear(64, 96, bias=False),
                                    torch.nn.Linear(96, 64, bias=False)).to(DEV)
        opt = optimizer(model.parameters(), lr=0.02, bf16_copy=True)
        x = torch.randn(8, 64, device=DEV)
        losses = []

        def step():
            opt.zero_grad()
            loss = model(x).float().square().mean()
            loss.backward()
            opt.step()
            losses.append(loss.item())

        with torch.autocast("cuda", dtype=torch.bfloat16):
            if held:
                with mi_adamw.bf16_weights(opt, model):
                    for _ in range(3):
                        step()
            else:
                for _ in range(3):
                    with mi_adamw.bf16_weights(opt, model):
                        step()
        return losses

    assert run(True) == run(False)


@pytest.mark.parametrize("seed", range(6))
def test_random_sequences(seed):
    """Eager steps with moved, missing and in-place gradients, options, loaded states and streams
    that change, replays of graphs recorded along the way: each equals the step of an optimizer built
    for it alone."""
    import random
    rng = random.Random(seed)
    half = rng.random() < 0.5
    options = dict(lr=0.02, ns_precision="half" if half else "single")
    params = make(seed)
    groups = [{"params": params[:2]}, {"params": params[2:], "nesterov": False}]
    opt = mi_adamw.Muon(groups, **options)
    set_grads(params, 0)
    streams = [torch.cuda.current_stream(), torch.cuda.Stream()]
    at, graphs = 0, []

    def check(run, grads, settings):
        # an optimizer of its own, on copies: new tables
        twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
        twin = mi_adamw.Muon([{"params": twins[:2]}, {"params": twins[2:], "nesterov": False}],
                             **options)
        twin.load_state_dict(copy.deepcopy(opt.state_dict()))
        for group, setting in zip(twin.param_groups, settings):
            group.update(setting)
        run()
        eager(twin, twins, grads)
        torch.cuda.synchronize()
        assert same(params, twins)
        for p, q in zip(params, twins):
            a, b = (o.state.get(t, {}).get("momentum_buffer") for o, t in ((opt, p), (twin, q)))
            assert (a is None) == (b is None) and (a is None or torch.equal(a, b))

    def settings_now():
        return [{k: g[k] for k in ("lr", "ns_steps", "weight_decay", "nesterov", "momentum")}
                for g in opt.param_groups]

    for k in range(25):
        event = rng.choice(["same", "same", "move", "move", "missing", "options", "load", "stream",
                            "capture", "replay", "replay"])
        if event == "stream":
            at ^= 1
            streams[at].wait_stream(streams[at ^ 1])
        with torch.cuda.stream(streams[at]):
            if event == "move" or any(p.grad is None for p in params):
                set_grads(params, rng.randrange(1000))
            if event == "missing":
                params[rng.randrange(len(params))].grad = None
            if event == "options":
                group = rng.choice(opt.param_groups)
                group["ns_steps"] = rng.choice([3, 5])
                group["lr"] = rng.choice([0.01, 0.02])
                group["weight_decay"] = rng.choice([0.0, 0.1])
            if event == "load":
                opt.load_state_dict(copy.deepcopy(opt.state_dict()))
            if event == "replay" and graphs:
                # a graph steps the momentum it was recorded with
                graph, grads, settings, moments = rng.choice(graphs)
                if all(opt.state[p]["momentum_buffer"] is m for p, m in zip(params, moments)):
                    junk = occupy()
                    check(graph.replay, grads, settings)
                    del junk
                continue
            check(opt.step, [p.grad for p in params], settings_now())
            if event == "capture" and all(p.grad is not None for p in params):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    opt.step()
                graphs.append((graph, [p.grad for p in params], settings_now(),
                               [opt.state[p]["momentum_buffer"] for p in params]))
