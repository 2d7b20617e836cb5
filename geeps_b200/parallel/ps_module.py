"""PSModule: trains a Net through the parameter server.

Every parameterised layer owns one table (its parameters packed row after row, each padded to
whole 128-float rows).  One fwd/bwd is declared to the runtime as a virtual iteration:
    Read(table_l) before layer l's forward ... then, walking the layers backwards,
    PreUpdate(table_l) -> layer l's backward writes its gradients straight into that buffer ->
    PostRead(table_l) -> Update(table_l) ... Clock.
Because a layer's Update is the last write of its table in the clock, the runtime signals that
table's clock immediately and the push of layer l overlaps the backward pass of layers < l
(the per-table clocks of the reference exist for exactly this: src/client/clientlib-viter.cpp:773-797).

Stands in for the solver glue of the reference's (absent) Caffe application.
"""
from __future__ import annotations

import os
import warnings
from dataclasses import replace

import torch

from ..ops import _lib as L
from ..ops import functional as F
from ..ops.layers import BF
from ..utils.config import TABLE_ADDITIVE, TRANSPORT_NVLINK, GeePsConfig
from ..utils.trace import NullTrace
from .ps import ROW_FLOATS, GeePs


def _rows_for(numel: int) -> int:
    return (numel + ROW_FLOATS - 1) // ROW_FLOATS


class _Table:
    def __init__(self, table_id, layer):
        self.table_id = table_id
        self.layer = layer
        self.specs = layer.param_specs()
        self.offsets = []
        off = 0
        for sp in self.specs:
            self.offsets.append(off)
            off += _rows_for(sp.numel) * ROW_FLOATS
        self.rows = off // ROW_FLOATS
        self.h_read = self.h_post = self.h_pre = self.h_upd = -1
        self.p16_buf = None

    def views(self, buf: torch.Tensor) -> dict:
        flat = buf.view(-1)
        return {sp.name: flat[o:o + sp.numel].view(sp.shape) for sp, o in zip(self.specs, self.offsets)}


class _AdamW:
    """The AdamW step of a module's tables: gradients in the update buffers become the updates."""
    _KEPT = ("m", "v", "exponents", "steps")

    def __init__(self, device, world, learning_rate, weight_decay, betas=(0.9, 0.999), eps: float = 1e-8, bits: int = 32, seed: int | None = None,
                 rank: int = 0):
        self.betas, self.eps, self.bits, self.weight_decay, self.world = betas, eps, bits, weight_decay, world
        # each worker rounds with bits of its own, so that what their roundings add to the sum of their steps averages out
        self.seed = None if seed is None else seed + (rank << 32)
        self.lr = torch.tensor([learning_rate / world], device=device)
        self.state, self._lists, self._resumed, self._rate = None, {}, None, None

    def save(self, directory: str, rank: int) -> None:
        """Nothing before the first step; after a resume what it brought back."""
        kept = self._resumed if self.state is None else {k: getattr(self.state, k) for k in self._KEPT}
        if kept is not None:
            if self.lr.is_cuda:
                torch.cuda.synchronize(self.lr.device)      # the last step may be on its way on another stream than this call's
            os.makedirs(directory, exist_ok=True)
            torch.save(kept, os.path.join(directory, f"adamw.{rank}"))

    def resume(self, directory: str, rank: int) -> None:
        """A rank that the saved job did not have goes on with rank 0's states; a snapshot without any begins anew."""
        with open(os.path.join(directory, "LATEST")) as f:
            at = os.path.join(directory, f"snapshot.{int(f.read())}")
        for r in (rank, 0):
            if os.path.exists(os.path.join(at, f"adamw.{r}")):
                self._resumed = torch.load(os.path.join(at, f"adamw.{r}"), map_location=self.lr.device)
                return
        warnings.warn(f"{at} has no AdamW states: moments and steps begin anew")

    def set(self, learning_rate=None, weight_decay=None) -> bool:
        """Whether a recorded step carries an old value."""
        if learning_rate is not None:
            self._rate = learning_rate / self.world
        changed = weight_decay is not None and weight_decay != self.weight_decay
        if changed:
            self.weight_decay = weight_decay
        return changed

    def begin(self) -> None:
        """In front of a step and on its stream: steps that are still on their way there keep the rate that they were called with."""
        if self._rate is not None:
            self.lr.fill_(self._rate)
            self._rate = None

    def step(self, mod) -> None:
        names = [(t.layer, sp) for t in mod.tables for sp in t.specs]
        params, grads = [l.p32[sp.name] for l, sp in names], [l.g32[sp.name] for l, sp in names]
        # laid out once for each phase of the update ring, so that a recorded step finds the same arguments again
        at = [x.data_ptr() for x in params] + [x.data_ptr() for x in grads]
        lists = self._lists.get(mod.steps % mod._period)
        if lists is None or lists[0] != at:
            lists = self._lists[mod.steps % mod._period] = (at, F.GradList(params), F.GradList(grads))
        _, params, grads = lists
        if self.state is None:
            self.state = F.AdamWState(params, self.bits, [sp.decay for _, sp in names])
            if self._resumed is not None:
                for k in self._KEPT:
                    setattr(self.state, k, self._resumed[k])
                self._resumed = None
        clip = None
        if mod.clip_gradients is not None:
            if mod._clip_work is None:
                mod._clip_work = torch.empty(grads.work_size(), dtype=torch.float64, device=mod.device)
            F.clip_gradients(grads, float("inf"), mod.clip_result, work=mod._clip_work)
            clip = (mod.clip_result, mod.clip_gradients)
        F.adamw_step(params, grads, self.state, self.lr, betas=self.betas, eps=self.eps, weight_decay=self.weight_decay, out=grads, clip=clip,
                     seed=self.seed)


class PSModule:
    adamw = None

    def __init__(self, net, in_shape, ps_config: GeePsConfig, rank: int = 0, world: int = 1, device="cuda:0",
                 slack: int = 0, seed: int = 0, keep_init: bool = False, trace=None, manage_activations: bool = False,
                 cache_fraction: float | None = None, use_tape: bool = False, bf16_weights_only: bool = False,
                 use_graph: bool = False, pull_fc: bool = False, uncached=(), resume_from: str | None = None,
                 clip_gradients: float | None = None, adamw: dict | None = None):
        """bf16_weights_only: with the NVLINK transport and the bf16 compute cache, weight rows are published to
        the workers' bf16 caches only (the layers never read weights in fp32; biases, BatchNorm scale / shift and
        the shard's master rows stay fp32).  The fp32 views of weights (`params_fp32`) then keep their initial
        values.
        use_graph: (NVLINK transport, implies use_tape) once a step's native calls are known to repeat, capture
        them in a CUDA graph per (input buffer, label buffer, update-ring phase) and replay the graph: one launch
        per step instead of one per kernel.  The runtime then keeps its clock in a device word (stamps relative
        to it, dropout seeds derived from it), so nothing in the captured launches changes from step to step.
        pull_fc: (NVLINK transport with the bf16 compute cache) the tables of the fully-connected layers become
        uncached tables: the shards do not publish them, and each layer's forward GEMM pulls the weight rows from
        the owning shards while it computes (ops.functional.pull_gemm), leaving a local bf16 copy for the backward
        pass; the bias rows arrive through the table's fp32 tail.
        uncached: names of further layers whose tables are kept uncached (no worker-side copy; every Read fetches
        the whole table from the shards into the staging pool) - the device-side form of a parameter cache that
        does not fit the GPU budget.
        resume_from: directory of table snapshots (`save_snapshot`): the tables (master rows, momentum, clocks) come
        from its latest snapshot instead of the initial values, and training goes on at the snapshot's clock.  The
        world size may differ from the one that wrote it.  Layer-local state (BatchNorm running statistics) is not
        part of a table snapshot.
        clip_gradients: scale the worker's gradients by clip_gradients / norm where the norm of all of them exceeds it
        (Caffe's solver parameter; every worker clips its own batch's).  No table is then pushed before the backward pass has
        ended, and the update buffers of all tables are held until then.  `clip_result` holds the last step's {norm, factor};
        inf only measures.
        adamw: the worker computes the updates of all tables with one AdamW step (F.adamw_step) at the end of the backward pass and the
        shards add them (tables must be TABLE_ADDITIVE): a dict of betas, eps, bits (32, or 8 for states in 8 bits) and seed (of
        stochastic rounding, to which the rank is added; None: to the nearest), each optional.  The rate is ps_config.learning_rate (set_hyper_params changes it
        without a new capture), the decay ps_config.weight_decay, for the parameters that decay.  Of several workers each takes 1 /
        world of its own step.  With clip_gradients the gradients are scaled on their way into the step and `clip_result` holds {norm, 1}.
        Parameters are given back when the step has read them.  The states (`adamw.state`) are the worker's own; save_snapshot and
        the snapshots of ps_config.snapshot_interval write and resume_from reads them."""
        self.net, self.rank, self.world, self.slack = net, rank, world, slack
        self.device = torch.device(device)
        self.trace = trace or NullTrace()
        net.setup(in_shape, self.device)
        self.tables = [_Table(i, l) for i, l in enumerate(net.param_layers())]
        by_layer = {id(t.layer): t for t in self.tables}
        # tables grouped by top-level layer (a Concat module holds several parameterised layers)
        self.groups = []
        for l in net.layers:
            subs = list(l.sublayers()) if hasattr(l, "sublayers") else [l]
            self.groups.append((l, [by_layer[id(s)] for s in subs if id(s) in by_layer]))
        ps_config.num_tables = len(self.tables)
        # Activations managed by the runtime's memory plan: the output of every large top-level layer becomes a
        # worker-local row batch (produced in forward: no fetch / keep; consumed in backward: fetch / discard), so
        # that under a GPU budget the plan decides which of them stay resident and which are swapped to pinned
        # host memory through the staging pool.
        self.managed = {}
        if manage_activations:
            from ..ops.layers import Dropout, Linear
            for i, (l, _) in enumerate(self.groups):
                nbytes = l.out_numel() * 2
                if isinstance(l, (Linear, Dropout)) or nbytes < (1 << 20):
                    continue
                nrows = (nbytes + 511) // 512
                for sub in (l.sublayers() if hasattr(l, "sublayers") else [l]):
                    sub.hold_no_extras()
                self.managed[i] = {"rows": range(1_000_000 * (i + 1), 1_000_000 * (i + 1) + nrows), "nrows": nrows}
        direct16 = ps_config.transport == TRANSPORT_NVLINK and ps_config.bf16_compute_cache
        # uncached (pull) tables
        nv = ps_config.transport == TRANSPORT_NVLINK and torch.cuda.is_available()
        from ..ops.layers import Linear as _Linear
        for t in self.tables:
            t.pull = t.fused_pull = False
            l = t.layer
            if not nv:
                continue
            if (pull_fc and isinstance(l, _Linear) and direct16 and l.B <= 256 and l.ld % ROW_FLOATS == 0
                    and len(t.specs) == 2):
                t.pull = t.fused_pull = True
                ps_config.table_partition_align[t.table_id] = l.ld // ROW_FLOATS    # whole weight rows per shard
                ps_config.table_fp32_from_row[t.table_id] = t.offsets[1] // ROW_FLOATS  # the bias rows are the tail
            elif getattr(l, "name", None) in uncached:
                t.pull = True
                ps_config.table_fp32_from_row.pop(t.table_id, None)
            if t.pull:
                ps_config.table_pull[t.table_id] = 1
        self.param_rows = sum(t.rows for t in self.tables)
        self.managed_rows = sum(m["nrows"] for m in self.managed.values())
        if cache_fraction is not None:
            ring = slack + 1 if ps_config.transport == TRANSPORT_NVLINK else 1 + int(bool(ps_config.read_my_writes))
            # rows of parameter state that stay in GPU memory: the update ring of every table, plus the worker's copy
            # of every table that is not uncached
            param_state = sum(t.rows * (ring + (0 if t.pull else 1)) for t in self.tables)
            if ps_config.transport == TRANSPORT_NVLINK:
                # peers read and write the parameter cache and the update ring in place, so that state stays
                # device resident; the cap applies to the activation working set, but never goes below what
                # one forward step needs at once (a layer's input and output)
                sizes = [self.managed.get(i, {"nrows": 0})["nrows"] for i in range(len(self.groups))]
                pair = max([a + b for a, b in zip(sizes, sizes[1:])] + sizes + [0])
                budget_rows = param_state + max(int(cache_fraction * self.managed_rows), int(pair * 1.02) + 16)
            else:
                budget_rows = int(cache_fraction * (param_state + self.managed_rows))
            self.budget_rows = budget_rows
            self.working_set_rows = param_state + self.managed_rows
            ps_config.gpu_memory_capacity = budget_rows * 512
            ps_config.mm_warning_level = 0
        self.direct16 = direct16
        if bf16_weights_only and self.direct16:
            for t in self.tables:
                if t.specs and t.specs[0].name == "weight" and not t.pull:
                    ps_config.table_fp32_from_row[t.table_id] = (t.offsets[1] // ROW_FLOATS) if len(t.specs) > 1 else t.rows
        # the runtime's periodic snapshots are taken inside a clock and know nothing of AdamW's states: the module takes them instead
        self._snapshot_every = ps_config.snapshot_interval if adamw is not None and ps_config.snapshot_dir else 0
        self._snapshot_dir = ps_config.snapshot_dir
        self.ps = GeePs(rank, replace(ps_config, snapshot_interval=0) if self._snapshot_every else ps_config)
        # tape replay: record two consecutive steps; if they issued identical native calls (static pointers),
        # later steps walk the tape instead of re-running the Python layer code
        self.use_graph = (use_graph and not manage_activations and ps_config.transport == TRANSPORT_NVLINK
                          and torch.cuda.is_available())
        self.use_tape = (use_tape or self.use_graph) and not manage_activations
        self._graphs, self._graph_failed = {}, False
        self._period = (slack + 1) if (slack + 1) % 2 == 0 else 2 * (slack + 1)
        self._tapes, self._tape_sigs, self._tape_tries = {}, {}, {}     # keyed by _step_key()
        self.tape_mismatch = None
        # diagnostics: set to [] to collect CUDA events (step start, forward end, backward end, clock end) per step
        self.phase_events = None
        # diagnostics: set to [] to collect (tag, CUDA event) at every layer boundary; the markers are part of a
        # recorded tape, so they also fire during tape replay
        self.layer_marks = None
        self.initial_params = {} if keep_init else None
        self.captured = None
        if clip_gradients is not None and not (clip_gradients >= 0 and self.device.type == "cuda"):
            raise ValueError(f"clip_gradients needs a bound from 0 up and a GPU, got {clip_gradients} on {self.device}")
        self.clip_gradients = clip_gradients
        self.clip_result = None if clip_gradients is None else torch.zeros(2, device=self.device)
        self._clip_lists, self._clip_work = {}, None
        if adamw is not None:
            if self.device.type != "cuda" or ps_config.table_mode != TABLE_ADDITIVE or pull_fc or bf16_weights_only:
                raise ValueError("adamw needs a GPU, additive tables and fp32 parameters of the worker (neither pull_fc nor bf16_weights_only)")
            self.adamw = _AdamW(self.device, world, ps_config.learning_rate, ps_config.weight_decay, rank=rank, **adamw)
        self._declare()
        if resume_from is not None:
            if not self.ps.load_snapshot(resume_from):
                raise RuntimeError(f"resume from {resume_from}: {self.ps.last_error_string()}")
            if self.adamw is not None:
                self.adamw.resume(resume_from, rank)
        else:
            self._bootstrap(seed)
        self.ps.start_iterations()
        self.steps = max(0, self.ps.clock_value - 1)      # clock 0 is the bootstrap clock
        if self.use_graph:
            ref = self.ps.enable_device_clock()
            for l in net.all_layers():
                if hasattr(l, "step_ref"):
                    l.step_ref = ref

    # one virtual iteration = the exact call sequence of step()
    def _declare(self):
        ps, M = self.ps, self.managed
        n = len(self.groups)
        for i, (_, tabs) in enumerate(self.groups):
            for t in tabs:
                t.h_read = ps.virtual_read(t.table_id, range(t.rows), self.slack)
            if i in M:
                M[i]["f"] = ps.virtual_local_access(M[i]["rows"], False)
            if i - 1 in M:      # the previous output was this layer's input: release (and keep) it now
                M[i - 1]["pf"] = ps.virtual_post_local_access(M[i - 1]["f"], True)
        if n - 1 in M:
            M[n - 1]["pf"] = ps.virtual_post_local_access(M[n - 1]["f"], True)
            M[n - 1]["b"] = ps.virtual_local_access(M[n - 1]["rows"], True)
        for i, (_, tabs) in reversed(list(enumerate(self.groups))):
            if i - 1 in M:
                M[i - 1]["b"] = ps.virtual_local_access(M[i - 1]["rows"], True)
            for t in reversed(tabs):
                t.h_pre = ps.virtual_pre_update(t.table_id, range(t.rows))
            for t in reversed(tabs):
                if self.adamw is None:
                    t.h_post = ps.virtual_post_read(t.h_read)
                if not self._updates_late():
                    t.h_upd = ps.virtual_update(t.h_pre)
            if i in M:
                M[i]["pb"] = ps.virtual_post_local_access(M[i]["b"], False)
        if self._updates_late():       # the updates wait for all gradients, with AdamW the parameters, too
            for _, tabs in reversed(self.groups):
                for t in reversed(tabs):
                    if self.adamw is not None:
                        t.h_post = ps.virtual_post_read(t.h_read)
                    t.h_upd = ps.virtual_update(t.h_pre)
        ps.virtual_clock()
        ps.finish_virtual_iteration()

    def _updates_late(self) -> bool:
        return self.clip_gradients is not None or self.adamw is not None

    def _update(self, name, tabs, post_read, update):
        if tabs:
            with self.trace.span(f"{'update' if update else 'post_read'}:{name}", "ps"):
                for t in reversed(tabs):
                    if post_read:
                        self.ps.post_read(t.h_post)
                    if update:
                        self.ps.update(t.h_upd)

    def _clip(self):
        """Clip the gradients where they are, in the tables' update buffers.  Their layout is made once for each phase of the update
        ring, so that a recorded step finds the same arguments again, and anew when a phase has other buffers."""
        buffers = [g for t in self.tables for g in t.layer.g32.values()]
        phase = self.steps % self._period
        grads = self._clip_lists.get(phase)
        if grads is None or [g.data_ptr() for g in grads.tensors] != [g.data_ptr() for g in buffers]:
            grads = self._clip_lists[phase] = F.GradList(buffers)
        if self._clip_work is None:
            self._clip_work = torch.empty(grads.work_size(), dtype=torch.float64, device=self.device)
        F.clip_gradients(grads, self.clip_gradients, self.clip_result, work=self._clip_work)

    def _bootstrap(self, seed):
        # the bootstrap update carries the initial values; updates add up over workers, so only rank 0
        # sends non-zero values
        gen = torch.Generator().manual_seed(seed)
        for t in [t for _, tabs in reversed(self.groups) for t in reversed(tabs)]:
            buf = self.ps.pre_update(t.h_pre)
            buf.zero_()
            views = t.views(buf)
            for sp in t.specs:
                init = sp.initial(gen)
                if self.rank == 0:
                    views[sp.name].copy_(init.to(buf.device))
                if self.initial_params is not None:
                    self.initial_params[f"{t.layer.name}.{sp.name}"] = init.clone()
            self.ps.update(t.h_upd)
        self.ps.clock()
        self._periodic_snapshot()

    def _bind_read_pull(self, t):
        """Fully-connected layer on an uncached table: no copy of the weights is made here - the layer's forward
        GEMM reads them from the shards (and leaves a bf16 copy in p16 for its backward)."""
        info = self.ps.read_pull(t.h_read)
        l = t.layer
        rpw = l.ld // ROW_FLOATS                       # table rows per weight row
        wrows = t.offsets[1] // ROW_FLOATS
        shards, n_start = [], []
        for s in range(info.num_shards):
            if info.row_count[s] == 0 or info.row_start[s] >= wrows:
                break
            shards.append(int(info.shard_bf16[s]))
            n_start.append(int(info.row_start[s]) // rpw)
        l.pull = (shards, n_start)
        if t.p16_buf is None:
            t.p16_buf = torch.zeros(t.rows, ROW_FLOATS, dtype=BF, device=self.device)
        l.p16 = t.views(t.p16_buf)
        tail = info.tail_tensor.view(-1)
        l.p32 = {"bias": tail[:t.specs[1].numel].view(t.specs[1].shape)}
        if self.captured is not None:
            self.captured[f"{l.name}.bias"] = l.p32["bias"].clone()

    def _bind_read(self, t):
        if t.fused_pull:
            return self._bind_read_pull(t)
        buf = self.ps.read(t.h_read)
        t.layer.p32 = t.views(buf)
        b16 = self.ps.read_bf16(t.h_read) if self.direct16 else None
        if b16 is None:
            if t.p16_buf is None:
                t.p16_buf = torch.empty(t.rows, ROW_FLOATS, dtype=BF, device=self.device)
            F.f32_to_bf16(buf, t.p16_buf)
            b16 = t.p16_buf
        t.layer.p16 = t.views(b16)
        if self.captured is not None:
            # stream-ordered copy of what this clock's Read delivered (tests)
            for name, v in t.layer.p32.items():
                self.captured[f"{t.layer.name}.{name}"] = v.clone()

    def _step_key(self, x, labels):
        """What a recorded step depends on.  The update ring has slack + 1 slots and staged buffers alternate between two
        copies, so the pointers a step uses repeat with the least common multiple of the two; its launches name the stream."""
        stream = torch.cuda.current_stream(self.device).cuda_stream if x.is_cuda else None
        return (x.data_ptr(), labels.data_ptr(), self.steps % self._period, stream)

    def step(self, x: torch.Tensor, labels: torch.Tensor, capture: bool = False) -> torch.Tensor:
        """One clock: forward, backward, push.  Returns the mean loss as a 1-element device tensor.
        capture=True keeps clones of the parameters this clock read in `self.captured`."""
        if self.adamw is not None:
            self.adamw.begin()
        loss = self._step(x, labels, capture)
        self._periodic_snapshot()
        return loss

    def _step(self, x, labels, capture):
        net, tr = self.net, self.trace
        key = self._step_key(x, labels)
        graph = self._graphs.get(key) if self.use_graph and not capture else None
        if graph is not None:
            graph.launch()
            self.ps.advance_replayed_clock()
            self.ps.check()
            self.steps += 1
            return net.loss_layer.loss
        tape = self._tapes.get(key) if self.use_tape and not capture else None
        if tape is not None and self.use_graph and not self._graph_failed:
            # capture this step (the host-side bookkeeping of the iteration happens now, during the capture),
            # then run it by launching the graph once
            try:
                graph = L.StepGraph(tape, torch.cuda.current_stream(self.device))
            except RuntimeError as e:
                self._graph_failed = True
                raise RuntimeError(f"step capture failed: {e}") from e
            self._graphs[key] = graph
            graph.launch()
            self.ps.check()
            self.steps += 1
            return net.loss_layer.loss
        if tape is not None:
            for arg, offset in tape.dropouts:      # the only arguments that change from step to step
                arg.value = offset + self.steps
            tape.replay()
            self.ps.check()
            self.steps += 1
            for l in tape.stepped_layers:
                l.step += 1
            return net.loss_layer.loss
        recording = (self.use_tape and not capture and self.steps >= 2 and self._tape_tries.get(key, 0) < 4
                     and (key in self._tape_tries or len(self._tape_tries) < 24))
        if recording:
            L.start_recording()
        self.captured = {} if capture else None
        ev = self.phase_events
        if ev is not None:
            ev.append([torch.cuda.Event(enable_timing=True) for _ in range(4)])
            ev[-1][0].record()
        self._mark("start")
        with tr.span("input", "fwd"):
            h = net.input_layer.forward(x)
        self._mark("f:input")
        M, n = self.managed, len(self.groups)

        def local(handle):
            return self.ps.local_access(handle).view(BF).view(-1)

        for i, (l, tabs) in enumerate(self.groups):
            name = getattr(l, "name", type(l).__name__)
            if tabs:
                with tr.span(f"read:{name}", "ps"):
                    for t in tabs:
                        self._bind_read(t)
            if i in M:
                l.set_output(local(M[i]["f"]))
            with tr.span(f"fwd:{name}", "fwd"):
                h = l.forward(h)
            self._mark("f:" + name)
            if i - 1 in M:
                self.ps.post_local_access(M[i - 1]["pf"])
        if n - 1 in M:
            self.ps.post_local_access(M[n - 1]["pf"])
            held = local(M[n - 1]["b"])
            self.groups[n - 1][0].set_output(held)
        with tr.span("loss", "fwd"):
            loss = net.loss_layer.forward(h, labels)
            g = net.loss_layer.backward()
        self._mark("loss")
        if ev is not None:
            ev[-1][1].record()
        for i, (l, tabs) in reversed(list(enumerate(self.groups))):
            name = getattr(l, "name", type(l).__name__)
            if i - 1 in M:
                # this layer's input was evicted after forward: fetch it back; it is also the previous
                # layer's output, which that layer's backward (ReLU / BN / LRN) reads
                buf = local(M[i - 1]["b"])
                l.set_input(buf[:self.groups[i - 1][0].out_numel()])
                self.groups[i - 1][0].set_output(buf)
            for t in reversed(tabs):
                t.layer.g32 = t.views(self.ps.pre_update(t.h_pre))
            with tr.span(f"bwd:{name}", "bwd"):
                g = l.backward(g)
            self._update(name, tabs, post_read=self.adamw is None, update=not self._updates_late())
            if i in M:
                self.ps.post_local_access(M[i]["pb"])
            self._mark("b:" + name)
        if self._updates_late():
            if self.adamw is not None:
                with tr.span("adamw", "bwd"):
                    self.adamw.step(self)
                self._mark("adamw")
            else:
                with tr.span("clip", "bwd"):
                    self._clip()
                self._mark("clip")
            for l, tabs in reversed(self.groups):
                self._update(getattr(l, "name", type(l).__name__), tabs, post_read=self.adamw is not None, update=True)
        if ev is not None:
            ev[-1][2].record()
        with tr.span("clock", "ps", clock=self.steps):
            self.ps.clock()
        if ev is not None:
            ev[-1][3].record()
        if recording:
            self._finish_recording(L.stop_recording(), key)
        self.steps += 1
        return loss

    def _periodic_snapshot(self) -> None:
        if self._snapshot_every and self.ps.clock_value % self._snapshot_every == 0:
            self.save_snapshot(self._snapshot_dir)

    def is_steady(self, x: torch.Tensor, labels: torch.Tensor) -> bool:
        """True when the next step with these buffers replays a captured graph (or, without graphs, a recorded
        tape): the Python layer code and the capture work are behind us."""
        key = self._step_key(x, labels)
        if self.use_graph and not self._graph_failed:
            return key in self._graphs
        return (not self.use_tape) or key in self._tapes

    def save_snapshot(self, directory: str) -> None:
        """Write every table (master rows, momentum, clocks) under directory/snapshot.<clock>; every rank calls it
        before the same step.  AdamW's states go beside them, a file for each rank."""
        if self.adamw is not None:          # first: what LATEST names is complete
            self.adamw.save(os.path.join(directory, f"snapshot.{self.ps.clock_value}"), self.rank)
        if not self.ps.save_snapshot(directory):
            raise RuntimeError(f"snapshot to {directory}: {self.ps.last_error_string()}")

    def set_hyper_params(self, learning_rate=None, momentum=None, weight_decay=None) -> None:
        """Change the optimizer's learning rate / momentum / weight decay from the next step on (every rank makes the
        same call before the same step).  Recorded and captured steps carry the old values in their push launches, so
        they are dropped when a value changes: the next few steps run through the layer code and are captured again.
        With AdamW the rate is read from the device and only another decay drops them; there is no momentum to change."""
        if self.adamw is not None:
            if self.adamw.set(learning_rate, weight_decay):
                if self.use_graph:
                    torch.cuda.synchronize(self.device)
                self.invalidate_tapes()
            return
        old = self.ps.hyper_params()
        self.ps.set_hyper_params(learning_rate, momentum, weight_decay)
        if self.ps.hyper_params() != old:
            if self.use_graph:
                torch.cuda.synchronize(self.device)      # no replay in flight when its graph is destroyed
            self.invalidate_tapes()

    def invalidate_tapes(self) -> None:
        """Forget the recorded steps (call after anything that changes what a step launches: switching layers
        between training and inference mode, rebinding buffers, changing hyper-parameters baked into arguments)."""
        self._tapes.clear()
        self._tape_sigs.clear()
        self._tape_tries.clear()
        for g in self._graphs.values():
            g.close()
        self._graphs.clear()

    def _mark(self, tag):
        if self.layer_marks is None:
            return

        def fire():
            e = torch.cuda.Event(enable_timing=True)
            e.record()
            self.layer_marks.append((tag, e))
            return 0
        L.record_call(fire, "mark:" + tag)

    def _finish_recording(self, tape, key):
        """Keep the tape for this (input, label) buffer pair once two recordings of it issued the same native
        calls with the same arguments (dropout seeds aside, which are re-derived from the step count)."""
        import ctypes
        self._tape_tries[key] = self._tape_tries.get(key, 0) + 1
        tape.dropouts = [(a, a.value - self.steps) for fn, args, label in tape.ops if label == "dropout"
                         for a in args if isinstance(a, ctypes.c_ulonglong)]
        tape.stepped_layers = [l for l in self.net.all_layers() if hasattr(l, "seed") and hasattr(l, "step")]
        sig = [row for row in tape.signature() if row[0] != "dropout"]
        prev = self._tape_sigs.get(key)
        if prev == sig:
            self._tapes[key] = tape
        elif prev is not None:
            # keep the first difference for diagnostics (why a step does not repeat)
            i = next((i for i, (a, b) in enumerate(zip(prev, sig)) if a != b), min(len(prev), len(sig)))
            self.tape_mismatch = (key[2], i, prev[i][0] if i < len(prev) else None, sig[i][0] if i < len(sig) else None,
                                  len(prev), len(sig))
        self._tape_sigs[key] = sig

    def params_fp32(self) -> dict:
        """Current parameter values as seen by this worker's last Read (for tests)."""
        out = {}
        for t in self.tables:
            for name, v in t.layer.p32.items():
                out[f"{t.layer.name}.{name}"] = v
        return out

    def close(self):
        torch.cuda.synchronize(self.device) if self.use_graph else None
        for g in self._graphs.values():
            g.close()
        self._graphs.clear()
        self.ps.shutdown()
        self.ps.close()
