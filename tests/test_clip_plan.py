"""The order of table calls in a step that clips: parameters are given back as soon as a layer's backward pass has ended, as in a step
that does not; only the updates wait for the norm of all gradients."""
import pytest

from geeps_b200.models.net import Net
from geeps_b200.ops.layers import Input, Linear
from geeps_b200.parallel.ps_module import PSModule


class FakePS:
    """Records the virtual iteration."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name,) + args)
            return len(self.calls) - 1
        return call


class Table:
    def __init__(self, i, rows):
        self.table_id, self.rows = i, rows


def declared(clip, managed=(), rows=(4, 4, 4, 4)):
    mod = PSModule.__new__(PSModule)
    mod.ps, mod.slack, mod.clip_gradients = FakePS(), 0, clip
    tables = [Table(i, n) for i, n in enumerate(rows)]
    mod.groups = [(object(), tables[:1]), (object(), []), (object(), tables[1:3]), (object(), tables[3:])]
    mod.managed = {i: {"rows": range(8)} for i in managed}
    mod._declare()
    return mod.ps.calls


def names(calls):
    return [c[0].replace("virtual_", "") for c in calls]


@pytest.mark.parametrize("managed", [(), (0, 2)])
def test_parameters_are_given_back_layer_by_layer(managed):
    plain, clipped = declared(None, managed), declared(1.0, managed)
    # the same calls, of which only the updates stand elsewhere: in the same order behind all else
    def bare(calls):
        return [n for n in names(calls) if n != "update"]
    assert bare(plain) == bare(clipped) and names(plain).count("update") == names(clipped).count("update") == 4
    assert names(clipped)[-6:] == ["update"] * 4 + ["clock", "finish_iteration"]
    # every table's read is given back before the next layer asks for its update buffers
    reads = {i for i, c in enumerate(clipped) if c[0] == "virtual_read"}
    held, most = set(reads), []
    for c in clipped:
        if c[0] == "virtual_post_read":
            held.discard(c[1])
        elif c[0] == "virtual_pre_update":
            most.append(len(held))
    assert most == [4, 3, 3, 1] and not held


def peak(calls, rows):
    """Rows of staged buffers at once in the plan of these calls, on a GPU that has no room for a copy of the parameters."""
    from test_core_cpu import CLOCK, POST_READ, PRE_UPDATE, READ, UPDATE, Planner
    p = Planner(tables=len(rows))
    handle = {}
    for i, c in enumerate(calls):
        name = c[0].replace("virtual_", "")
        if name == "read":
            handle[i] = p.rec(READ, c[1], list(c[2]), slack=c[3])
        elif name == "pre_update":
            handle[i] = p.rec(PRE_UPDATE, c[1], list(c[2]))
        elif name in ("post_read", "update"):
            p.rec(POST_READ if name == "post_read" else UPDATE, prestep=handle[c[1]])
        elif name == "clock":
            p.rec(CLOCK)
    plan = p.compile()
    assert plan["ok"]
    return plan["peak_staging_rows"]


@pytest.mark.parametrize("rows", [(4, 4, 4, 4), (100, 3, 50, 7), (1, 2, 3, 400)])
def test_staged_buffers_at_once(rows):
    """A step reads all tables, so these are held when the backward pass starts.  A layer then takes update buffers, and gives its
    parameters back; clipping keeps the update buffers, a plain step does not."""
    groups = [sum(rows[3:]), sum(rows[1:3]), rows[0]]       # in the order of the backward pass
    for clip in (None, 1.0):
        held, most = sum(rows), 0
        for g in groups:
            most = max(most, held + g)
            held -= g if clip is None else 0
        assert peak(declared(clip, rows=rows), rows) == most


@pytest.mark.gpu
def test_a_clipped_step_trains_under_a_budget():
    """Parameters that leave the GPU (host transport).  The tables have 1026, 514, 514, 514 and 33 rows: a step that clips has them
    and one layer's update buffers staged at once, 0.70 of two copies of all, and some gaps between; with the parameters held to the
    end it had two copies of all, for which no fraction below 1 has room."""
    import torch

    from geeps_b200.utils.config import TRANSPORT_TCP
    from test_gpu_residual import cfg, same_training

    def run(**kw):
        net = Net("n", Input(cpad=8), [Linear(f"f{i}", 256, relu=True, std=0.05) for i in range(4)] + [Linear("fc", 16, std=0.1, fp32_out=True)])
        mod = PSModule(net, (16, 3, 8, 8), cfg(TRANSPORT_TCP), device="cuda:0", seed=3, **kw)
        gen = torch.Generator(device="cuda:0").manual_seed(1)
        x, y = torch.randn(16, 3, 8, 8, generator=gen, device="cuda:0"), torch.randint(0, 16, (16,), generator=gen, device="cuda:0")
        out = [mod.step(x, y).item() for _ in range(4)]
        mod.close()
        return out
    plain = run()
    same_training([plain, run(clip_gradients=float("inf")), run(clip_gradients=float("inf"), cache_fraction=0.9)])


def test_layouts_are_kept_for_the_phases_of_the_update_ring_only(monkeypatch):
    """A step's gradients come in the buffers of its phase of the ring, so a phase's layout serves again (a recorded step finds the same
    arguments); buffers that do not come back are not held."""
    import torch

    import geeps_b200.parallel.ps_module as pm

    class List:
        def __init__(self, tensors):
            self.tensors = list(tensors)

        def work_size(self):
            return 4
    used = []
    monkeypatch.setattr(pm.F, "GradList", List)
    monkeypatch.setattr(pm.F, "clip_gradients", lambda grads, bound, result, work: used.append(grads))

    class Layer:
        pass
    mod = PSModule.__new__(PSModule)
    mod.device, mod.clip_gradients, mod.clip_result, mod._clip_lists, mod._clip_work = torch.device("cpu"), 1.0, None, {}, None
    mod._period, mod.tables = 2, []
    for i in range(3):
        t = Table(i, 1)
        t.layer = Layer()
        mod.tables.append(t)
    ring = [[torch.zeros(5) for _ in mod.tables] for _ in range(2)]

    def step(i, buffers):
        mod.steps = i
        for t, b in zip(mod.tables, buffers):
            t.layer.g32 = {"w": b}
        mod._clip()
        assert [t.data_ptr() for t in used[-1].tensors] == [b.data_ptr() for b in buffers]
    for i in range(8):
        step(i, ring[i % 2])
    assert len({id(u) for u in used}) == 2 and used[0] is used[2] and used[1] is used[3]
    other = [[torch.zeros(5) for _ in mod.tables] for _ in range(10)]        # all alive, so all at addresses of their own
    for i in range(10):
        step(8 + i, other[i])
    assert len(mod._clip_lists) == 2
