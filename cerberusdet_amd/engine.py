"""Plan compiler: CerberusDet block DAG  ->  static launch list of gfx950 kernels (forward, and backward for training).

The reference walks its DAG in Python on every call and dispatches ~600 torch ops per task pass
(cerberusdet/models/cerberus.py:804-882, models/yolo.py:172-203). Here the walk happens ONCE per
(task set, input shape, mode): every activation, gradient and workspace buffer is allocated up front, every kernel
descriptor is pre-built, and a step is a flat loop over (C function, argument tuple) pairs on one HIP stream --
capturable into a hipGraph, no allocator traffic, no host syncs.

Dataflow conventions
  * activations are NHWC `View`s (channel slices of buffers); Concat / chunk never copy more than once;
  * train mode keeps, per Conv: z (raw conv output, bf16), batch mean / invstd, and the activation y;
  * the backward list is generated by walking the forward ops in reverse with a static "already written" tracker per
    gradient buffer, which selects overwrite vs accumulate variants at compile time (no zero-fills at run time);
  * parameter gradients accumulate into persistent fp32 `.grad` tensors (the reference accumulates across the per-task
    passes of one iteration as well, trainers/averaging.py:142-168).
"""
from __future__ import annotations

import ctypes as C
import os
from typing import Dict, List, Optional, Sequence

import torch
import torch.nn as nn

from . import _lib as L
from .models.common import BN_EPS, BN_MOMENTUM, C2f, Concat, Conv, SPPF, Upsample
from .ops import View, conv_desc, dt

_PAD8 = lambda v: (v + 7) // 8 * 8  # noqa: E731


class _Deferred:
    """Output of an Upsample block that has not been materialised: the following Concat writes it straight into its slice."""

    def __init__(self, src: View):
        self.src = src
        self.C, self.N, self.H, self.W = src.C, src.N, 2 * src.H, 2 * src.W


class _VirtualCat:
    """Output of a Concat block in an eval plan that has not been materialised: the 1x1 convolution behind it (a C2f's cv1) walks the
    parts itself (cdet_conv2d_tiled_cat). parts: [(View, upsampled: bool)]; an upsampled part is half the size."""

    def __init__(self, parts):
        self.parts = parts
        v0, up0 = parts[0]
        self.N, self.H, self.W = v0.N, v0.H * (2 if up0 else 1), v0.W * (2 if up0 else 1)
        self.C = sum(v.C for v, _ in parts)


class _Written:
    """Static tracker of which channel ranges of each gradient buffer have been written during the backward walk."""

    def __init__(self):
        self.iv: Dict[int, List[tuple]] = {}

    def query(self, v: View) -> bool:
        lo, hi = v.coff, v.coff + v.C
        cov = [r for r in self.iv.get(id(v.buf), []) if r[0] < hi and r[1] > lo]
        if not cov:
            return False
        pos = lo
        for a, b in sorted(cov):
            if a > pos:
                raise RuntimeError("partially written gradient range (unsupported graph)")
            pos = max(pos, b)
        if pos < hi:
            raise RuntimeError("partially written gradient range (unsupported graph)")
        return True

    def mark(self, v: View):
        self.iv.setdefault(id(v.buf), []).append((v.coff, v.coff + v.C))


_LANE_STREAMS: Dict[tuple, "torch.cuda.Stream"] = {}


def lane_stream(device, lane: int) -> "torch.cuda.Stream":
    """Side-lane streams are created ONCE per device and shared by every plan. The HIP runtime multiplexes streams onto a few
    hardware queues in creation order; a fresh set of streams per plan made the forward time depend on how many streams the
    process had created before (two lanes landing on one queue serialise: 14.0 / 15.3 / 17.0 ms for the same plan,
    profiles/r02_placement_probe.txt)."""
    dev = torch.device(device)
    di = dev.index if dev.index is not None else torch.cuda.current_device()
    if (di, lane) not in _LANE_STREAMS:
        for ln in range(1, lane + 1):  # always created in lane order: lane k is the k-th stream this package makes on the device
            if (di, ln) not in _LANE_STREAMS:
                # (stream priorities per lane were measured without effect on the step: 900.7 / 904.1 default, 898.3 / 895.5 with either task stream
                #  at high priority, 902.4 with both -- round 5, one box)
                st = _LANE_STREAMS[(di, ln)] = torch.cuda.Stream(device=torch.device("cuda", di))
                # ... and FIRST USED in lane order: the runtime binds a stream to a hardware queue at its first submission, not at its creation.
                # Round 5: the trainer used lanes 1, 2, 4 before any eval plan touched lane 3 -- lane 3 then shared a queue with another lane and
                # the 2-task forward took 15.0 instead of 12.6 ms (tools/debug/ns_regress.py: use124 vs use1234). One marker per new stream.
                torch.cuda.Event().record(st)
    return _LANE_STREAMS[(di, lane)]


_TASK_STREAMS: Dict[tuple, "torch.cuda.Stream"] = {}


def task_stream(device, k: int, n: int) -> "torch.cuda.Stream":
    """Stream of the k-th of n concurrent task passes of a training iteration (Averaging._run_tasks_on_streams).
    Default: the process-wide lane streams. CDET_TASK_CU_SPLIT=<mode> gives every task pass a stream restricted to its own share of the
    compute units (hipExtStreamCreateWithCUMask): kernels of two unrestricted streams only overlap at their tails -- a convolution grid owns
    every VGPR of every CU it runs on, so the other pass's BatchNorm kernels wait for it instead of running beside it
    (profiles/r04_step_timeline.txt). Modes: "even" (CU bit i -> pass i % n), "block" (the mask split into n contiguous runs)."""
    mode = os.environ.get("CDET_TASK_CU_SPLIT", "0")
    if mode in ("0", "") or n < 2:
        return lane_stream(device, k + 1)
    dev = torch.device(device)
    di = dev.index if dev.index is not None else torch.cuda.current_device()
    key = (di, k, n, mode)
    if key not in _TASK_STREAMS:
        import ctypes as _C

        ncu = torch.cuda.get_device_properties(di).multi_processor_count
        words = (ncu + 31) // 32
        bits = [0] * words
        for i in range(ncu):
            mine = (i % n == k) if mode == "even" else (min(i * n // ncu, n - 1) == k)  # "block": n contiguous runs of the mask
            if mine:
                bits[i // 32] |= 1 << (i % 32)
        hip = _C.CDLL("libamdhip64.so")
        st = _C.c_void_p()
        arr = (_C.c_uint32 * words)(*bits)
        with torch.cuda.device(di):
            rc = hip.hipExtStreamCreateWithCUMask(_C.byref(st), _C.c_uint32(words), arr)
        if rc != 0 or not st.value:
            raise RuntimeError(f"hipExtStreamCreateWithCUMask failed ({rc})")
        _TASK_STREAMS[key] = torch.cuda.ExternalStream(st.value, device=torch.device("cuda", di))
    return _TASK_STREAMS[key]


class Plan:
    def __init__(self, model, tasks: Sequence[str], N: int, H: int, W: int, training: bool, dtype: torch.dtype,
                 img_dtype: torch.dtype, device, frozen=()):
        self.lib = L.load()
        self.model, self.tasks, self.training, self.dtype, self.device = model, list(tasks), training, dtype, device
        self.N, self.H, self.W, self.img_dtype = N, H, W, img_dtype
        self.fwd: List[tuple] = []
        self.bwd_groups: List[tuple] = []  # (block_idx, [calls]) in FORWARD order; executed reversed
        self.fwd_marks: List[tuple] = []   # (block_idx, end index into self.fwd) per executed block
        self.block_sync = None             # optional BlockSync: cross-stream ordering of the blocks this task shares with others
        self.deferred_stats: Dict[int, List[tuple]] = {}  # block -> running-statistics updates that follow the block (later task of a shared block)
        # trainer-managed model with per-task gradient buckets on shared blocks (_alt_grad): this pass shares no read-modify-write state with
        # the other tasks' passes -- no cross-stream waits except in front of its deferred running-statistics updates
        self.decoupled = bool(getattr(model, "_pgrad_alt", None)) and training and len(tasks) == 1
        self._cur_bwd: Optional[List[tuple]] = None
        self.keep: List[object] = []
        self._registered: List[tuple] = []     # (module's _plan_slots list, entry) pairs this plan added (release())
        self.convs: List[nn.Module] = []       # Conv modules on this plan's path (weight packing)
        self.biased: List[nn.Module] = []      # head nn.Conv2d(1x1, bias)
        self.img_slots: List[list] = []        # argument lists whose [0] is the image pointer
        self.grad_bufs: Dict[int, torch.Tensor] = {}
        self.written = _Written()
        self._dz_elems = self._part_elems = self._wgrad_elems = 0
        # round 5: CDET_BN_FOLD=1 reduces the BatchNorm partial sums inside the launches that produce them (csrc/bn_fold.h): no bn_finalize /
        # bn_bwd_sums launches in the per-GPU training plans, bit-identical to the separate kernels (both forms add in the same fixed tree order).
        # MEASURED AND NOT THE DEFAULT: 884.8 against 908.0 images/s on the same box (72.3 vs 70.5 ms; profiles/r05_bn_fold_ab.txt). The in-launch
        # hand-off is a chain of ~6 dependent cross-XCD round trips behind the last workgroup (drain the write-through row, ticket, read the
        # cluster's rows, drain, ticket, read the cluster sums: 15-30 us), longer than the launch boundary + 5 us kernel it replaces, and it sits on
        # the same dependent chain conv -> statistics -> normalisation.
        # Round 6: the fold's kernels are compiled into -DCDET_EXPERIMENTS builds of the library only (make -C cerberusdet_amd/csrc EXTRA=-DCDET_EXPERIMENTS).
        self._bn_fold = os.environ.get("CDET_BN_FOLD", "0") == "1"
        if self._bn_fold and not self.lib.cdet_has_experiments():
            raise RuntimeError("CDET_BN_FOLD=1 needs an experiments build of libcerberus_hip.so (make EXTRA=-DCDET_EXPERIMENTS); the product build "
                               "does not carry the in-launch BatchNorm fold (measured slower, profiles/r05_bn_fold_ab.txt)")
        self._fold_cl_doubles = 0
        self._fold_descs: List[tuple] = []     # (BnFold host struct, device byte tensor, fill(desc, part) -> None)
        self._deferred_items: Dict[int, List[tuple]] = {}  # block -> [(totals, bn, 1 / count, unbias)] of the later task's running-statistics updates
        self.n_folded = [0, 0]                 # forward / backward reductions folded into their producers
        self._wg_pending: List[dict] = []      # weight gradients of the block being compiled that wait for the grouped launch
        self._wg_group = os.environ.get("CDET_WGRAD_GROUP", "1") != "0"
        self._late: List = []                  # closures that bind scratch buffers once their size is known
        self.feats: Dict[str, List[torch.Tensor]] = {}
        self._out_ptr_slots: List[tuple] = []  # every launch argument that holds a pointer to a head map / `y` (fresh_outputs)
        self._home_outputs = None
        self.head_chains: Dict[str, List[tuple]] = {}  # task -> [(level, branch, first call, end call)]
        self.sched = None                      # eval plans: launch-list segments per stream lane (see _build_lanes)
        self.dfeats: Dict[str, List[torch.Tensor]] = {}
        self.y: Dict[str, torch.Tensor] = {}
        self.block_of_param: Dict[int, int] = {}
        self.early_blocks: frozenset = frozenset()  # trainer: blocks whose weights are re-packed before the task streams fork (the shared trunk)
        self.tail_event = None                 # trainer: event behind the optimizer's tail (the other blocks' update): awaited in front of the late re-pack
        self.hooks = {}                        # block idx | (0, backbone row) -> callable, run right after that block's / row's backward launches
        self.bwd_sub: Dict[int, List[tuple]] = {}  # block 0: [(row, end index into the block's backward calls)] -- where each backbone row's gradients are complete
        self._sub_marks: List[tuple] = []
        self._sbn_fwd = None                   # SyncBatchNorm: open group of INDEPENDENT layers whose statistics travel in one all-reduce
        self._sbn_bwd = None
        self.trace: List[dict] = []            # one record per compiled unit (module, views, launch-list positions): what each launch reads / writes
        self._params_seen: Dict[int, torch.nn.Parameter] = {}
        # frozen blocks (all their parameters have requires_grad False, reference cerberus.py:885-905): train-form forward with batch
        # statistics but no running-statistic update (see _conv_unit), no backward launches, no gradient sent into them
        self.frozen = frozenset(frozen) if training else frozenset()
        self.dead = set()
        self.frozen_convs: List[nn.Module] = []
        self._train_here = training
        self._nograd = set()
        import torch.distributed as dist
        self.world = dist.get_world_size() if (dist.is_available() and dist.is_initialized()) else 1
        self.sync_bn = bool(getattr(model, "sync_bn", False)) and training and dist.is_available() and dist.is_initialized()
        self._build()

    # ------------------------------------------------------------------------------------------------ helpers
    def _new(self, N, H, W, Cn, dtype=None, zero=False, row_align=0) -> View:
        """row_align (elements): pitch of a pixel row rounded up to it. A concat buffer of 800 (400) channels has 1600 (800)-byte pixel rows,
        12.5 (6.25) cache lines: the 1x1 convolution over it ran 13 % slower than the 832-channel one (tools/conv_tiled_bench.py --shape);
        the pad channels are never written or read."""
        ld = Cn if not row_align or os.environ.get("CDET_LD_ALIGN", "1") == "0" else -(-Cn // row_align) * row_align
        t = self._alloc((N, H, W, ld), dtype or self.dtype, zero)
        if self.training and not self._train_here:
            self._nograd.add(id(t))
        return View(t, 0, Cn)

    def _out(self, N, H, W, Cn) -> View:
        """Output buffer of the layer / block being compiled. When a later Concat consumes it (the pre-pass of _build found the
        pair) the output IS its channel slice of that Concat's buffer: the producer writes it there and the copy -- and the
        gradient copy back -- disappear (the reference's torch.cat materialises every input, models/common.py:288-295)."""
        pl = self._cur_place
        self._cur_place = None  # one output per layer: inner temporaries of a C2f / SPPF allocate normally
        if pl is None:
            return self._new(N, H, W, Cn)
        cidx, off, ctot = pl
        cat = self._cat_bufs.get(cidx)
        if cat is None:
            cat = self._cat_bufs[cidx] = self._new(N, H, W, ctot, row_align=64)
        assert (cat.N, cat.H, cat.W) == (N, H, W)
        return cat.slice(off, Cn)

    def _alloc(self, shape, dtype, zero=False) -> torch.Tensor:
        t = (torch.zeros if zero else torch.empty)(tuple(shape), dtype=dtype, device=self.device)
        self.keep.append(t)
        return t

    def _vec(self, n, dtype=torch.float32, zero=False):
        return self._alloc((n,), dtype, zero)

    def grad(self, v: View) -> View:
        g = self.grad_bufs.get(id(v.buf))
        if g is None:
            g = self._alloc(tuple(v.buf.shape), v.buf.dtype)
            self.grad_bufs[id(v.buf)] = g
        return View(g, v.coff, v.C)

    def _allreduce_call(self, t: torch.Tensor, key=None):
        """A launch-list entry that SUM-all-reduces `t` on the plan's stream (RCCL orders itself behind the preceding kernels).
        key: (direction, BatchNorm layer(s)) of the exchange -- with the plan's task set it names the peer-exchange slot, so that recompiled
        plans of the same tasks (frozen / unfrozen trunk, another batch shape) reuse their slots (peer_exchange.PeerExchange.make_call)."""
        import torch.distributed as dist

        from .trainers.averaging import comm_span, on_group

        model = self.model
        px = getattr(self.model, "_peer_xchg", None)
        if px is not None:  # round 4: one peer-write kernel instead of an RCCL collective (peer_exchange.py)
            inner = px.make_call(t, key=None if key is None else (tuple(self.tasks),) + tuple(key))

            def pcall(st):
                with comm_span(model, "syncbn"):  # (bench.py --gpus N: comm_exposed_ms; a no-op without a timer)
                    inner(st)

            pcall.__name__ = inner.__name__
            return pcall

        def call(st, t=t):
            with comm_span(model, "syncbn"):
                on_group(dist.all_reduce, t, op=dist.ReduceOp.SUM)

        call.__name__ = "all_reduce"
        return call

    def _flush_wgrads(self):
        """Emit one cdet_conv2d_wgrad_grouped launch per geometry for the weight gradients deferred during this block's backward."""
        lib = self.lib
        groups: Dict[tuple, List[dict]] = {}
        for r in self._wg_pending:
            groups.setdefault(r["key"], []).append(r)
        self._wg_pending = []
        for recs in groups.values():
            d0 = recs[0]["desc"]
            d = L.ConvDesc.from_buffer_copy(bytes(d0))
            d.src_ld = max(r["x"].ld for r in recs)  # the 32-bit DMA-offset bound is checked against the widest source view
            tab = (L.WgradItem * len(recs))()
            for i, r in enumerate(recs):
                tab[i].x, tab[i].dy, tab[i].dw = r["x"].buf.data_ptr(), r["dz"].data_ptr(), r["dw"].data_ptr()
                tab[i].src_ld, tab[i].src_coff = r["x"].ld, r["x"].coff
            tab_dev = torch.frombuffer(bytearray(bytes(tab)), dtype=torch.uint8).to(self.device)
            n_ws = lib.cdet_conv2d_wgrad_grouped_ws_elems(C.byref(d), len(recs))
            assert n_ws > 0, "grouped weight gradient refused a geometry cdet_conv2d_wgrad_groupable accepted"
            self._wgrad_elems = max(self._wgrad_elems, n_ws)
            self.keep += [d, tab_dev]
            call = [C.byref(d), tab_dev.data_ptr(), len(recs), None, 1]
            self._cur_bwd.append((lib.cdet_conv2d_wgrad_grouped, call))

            def bind(dz, part, ws, call=call):
                call[3] = ws.data_ptr()

            self._late.append(bind)

    def _fold_desc(self, nrows: int, Cn: int, fill):
        """A cdet_bn_fold descriptor in device memory (the producing kernel reads it at its very end). `fill(desc, part)` sets the layer's
        pointers; tickets / cluster scratch are the plan's (bound in _bind_folds once their sizes are known)."""
        d = L.BnFold()
        d.nrows, d.C, d.ncl = nrows, Cn, -(-nrows // 32)
        dev = torch.zeros(C.sizeof(L.BnFold), dtype=torch.uint8, device=self.device)
        self._fold_cl_doubles = max(self._fold_cl_doubles, int(self.lib.cdet_bn_fold_cl_doubles(nrows, Cn)))
        self._fold_descs.append((d, dev, fill))
        self.keep.append(dev)
        return dev

    def _bind_deferred_items(self):
        """One cdet_bn_running_update launch per shared block for the later task's running-statistics updates (from the fp32 totals the folded
        finalize left): same arithmetic and order as the per-layer cdet_bn_finalize(nblk = 1) launches, 3 launches instead of 26."""
        for blk, items in self._deferred_items.items():
            tab = (L.BnRunningItem * len(items))()
            for it, (totals, bn, inv_count, unbias) in zip(tab, items):
                it.totals, it.running_mean, it.running_var = totals.data_ptr(), bn.running_mean.data_ptr(), bn.running_var.data_ptr()
                it.inv_count, it.unbias, it.momentum, it.C = inv_count, unbias, float(bn.momentum), totals.numel() // 2
            tab_dev = torch.frombuffer(bytearray(bytes(tab)), dtype=torch.uint8).to(self.device)
            self.keep.append(tab_dev)
            self.deferred_stats.setdefault(blk, []).append(
                (self.lib.cdet_bn_running_update, [tab_dev.data_ptr(), len(items), max(it.C for it in tab)]))
        self._deferred_items = {}

    def _bind_folds(self, part):
        if not self._fold_descs:
            return
        tickets = self._alloc((L.BN_FOLD_TICKET_WORDS,), torch.int32, zero=True)  # zeroed once; the last arrivers reset what they used
        cl = self._alloc((max(self._fold_cl_doubles, 1),), torch.float64)
        for d, dev, fill in self._fold_descs:
            d.tickets, d.cl_sums = tickets.data_ptr(), cl.data_ptr()
            fill(d, part)
            dev.copy_(torch.frombuffer(bytearray(bytes(d)), dtype=torch.uint8))
        self._fold_descs = []

    def _f(self, fn, *args):
        self.fwd.append((fn, list(args)))

    def _b(self, fn, *args):
        self._cur_bwd.append((fn, list(args)))

    def _reg(self, m, kind, slot, attr="_plan_slots"):
        """Register an argument list whose weight pointers are (re)bound when the module's weights are packed."""
        lst = getattr(m, attr, None)
        if lst is None:
            lst = []
            setattr(m, attr, lst)
        entry = (kind, slot)
        lst.append(entry)
        self._registered.append((lst, entry))
        m._pack_key = None

    def release(self):
        """The model drops this plan (eval-plan eviction, models/cerberus.py::get_plan): take its argument lists off the modules' re-bind lists,
        which would otherwise grow by one dead entry per evicted plan and module (rectangular validation: a plan per frame shape)."""
        for lst, entry in self._registered:
            for i, e in enumerate(lst):
                if e is entry:
                    del lst[i]
                    break
        self._registered = []

    def _ensure_grad(self, p):
        """Model-owned persistent fp32 gradient buffer of parameter p (shared by all plans of the model)."""
        g = self.model._grad_buffer(p)
        if id(p) not in self._params_seen:
            self._params_seen[id(p)] = p
        a = self._alt_grad(p)
        return g if a is None else a

    def _alt_grad(self, p):
        """Trainer-managed models (Averaging): on a block that several tasks serve, every task but the first accumulates into a gradient bucket
        of its own (model._pgrad_alt, folded into the block's bucket in task order by model._merge_alt_grads) -- the task passes of an iteration
        then share no read-modify-write state and run as independent launch streams."""
        alt = getattr(self.model, "_pgrad_alt", None)
        if not alt or not self.training or len(self.tasks) != 1:
            return None
        return alt.get((id(p), self.tasks[0]))

    # ------------------------------------------------------------------------------------------------ conv units
    def _conv_unit(self, m: Conv, x: View, y: View, res: Optional[View] = None, bwd_ops: Optional[list] = None, need_dx_default=True,
                   stem: bool = False, shortcut: Optional[View] = None):
        """SiLU(BN(conv(x))) (+res) -> y. Appends forward calls; pushes a backward closure onto bwd_ops.
        shortcut: the other addend of y = shortcut + SiLU(BN(conv(x))) (Bottleneck, reference common.py:107-117): the unit's backward pass over
        grad(y) also accumulates it into grad(shortcut) (cdet_bn_silu_bwd_apply_add) instead of a separate add launch."""
        lib = self.lib
        k, s = m.k, m.s
        # A frozen block inside a training plan (--freeze-shared-till-epoch): the reference's freeze sets m.eval() +
        # track_running_stats = False (cerberus.py:885-905) and then calls model.train() (trainers/averaging.py:106), which leaves the
        # frozen BatchNorms normalising with BATCH statistics while their running statistics stay untouched. So: train-form forward
        # (statistics from the conv epilogue, no running-stat update), no backward, no gradient into the block.
        frozen_here = self.training and not self._train_here
        self.convs.append(m)
        if frozen_here:
            self.frozen_convs.append(m)
        if not self.training and stem:
            # first backbone row: direct MFMA stem kernel on the NCHW image (csrc/stem_mfma.hip), BN folded into scale / bias
            slot = [None, dt(self.img_dtype), None, None, None, y.buf.data_ptr(), y.N, self.H, self.W, m.c2, dt(self.dtype), L.ACT_SILU, None]
            self.img_slots.append(slot)
            self._reg(m, "stem_eval", slot)
            self.fwd.append((lib.cdet_stem_conv, slot))
            self.trace.append(dict(kind="econv", m=m, x=None, y=y, res=None, block=self._cur_block, fwd_hi=len(self.fwd)))
            return
        if not self.training and isinstance(x, _VirtualCat):
            from .ops import cat_desc, cat_srcs
            arr, _ = cat_srcs(x.parts)
            d = cat_desc(x.parts, y, L.ACT_SILU, res)
            if k == 1 and s == 1 and os.environ.get("CDET_CONV_TILED", "1") != "0" and lib.cdet_conv2d_tiled_cat_ok(C.byref(d), arr, len(x.parts)):
                slot = [C.byref(d), arr, len(x.parts), None, None, None, res.buf.data_ptr() if res else None, y.buf.data_ptr()]
                self.keep += [d, arr]
                self._reg(m, "eval_tc", slot)
                self.fwd.append((lib.cdet_conv2d_tiled_cat, slot))
                self.trace.append(dict(kind="econv", m=m, x=x, y=y, res=res, block=self._cur_block, fwd_hi=len(self.fwd)))
                return
            x = self._materialize(x)
        if not self.training:
            d = conv_desc(x, y, k, s, L.CONV_FWD, L.ACT_SILU, res)
            tiled = _use_tiled(lib, d)  # tap-resident kernel (csrc/conv_halo.hip) where the geometry allows
            s2t = not tiled and _use_tiled_s2(lib, d)  # 3x3 stride 2: the parity-plane kernel (csrc/conv_vt.hip)
            slot = [C.byref(d), x.buf.data_ptr(), None, None, None, res.buf.data_ptr() if res else None, y.buf.data_ptr(), None]
            self.keep.append(d)
            self._reg(m, "eval_t" if (tiled or s2t) else "eval", slot)
            self.fwd.append((lib.cdet_conv2d_tiled if tiled else (lib.cdet_conv2d_s2_tiled if s2t else lib.cdet_conv2d), slot))
            # eval plans leave a trace too (round 5): one record per unit naming what its launch reads and writes -- what the teacher-forced
            # full-size parity test of the EVAL plan walks (tests/teacher.py::check_eval_forward)
            self.trace.append(dict(kind="econv", m=m, x=x, y=y, res=res, block=self._cur_block, fwd_hi=len(self.fwd)))
            return
        if m.fused:
            raise RuntimeError("training needs un-fused Conv modules (BatchNorm present)")
        z = self._new(y.N, y.H, y.W, m.c2)
        dz_need = z.M * m.c2
        self._dz_elems = max(self._dz_elems, dz_need)
        d = conv_desc(x, z, k, s) if x is not None else None
        fold_fwd = False
        if stem:  # raw convolution + BN partial sums straight from the NCHW image (x = the 8-channel copy only feeds the weight gradient)
            nblk = lib.cdet_stem_conv_stat_blocks(self.N, self.H, self.W)
            stats = self._vec(nblk * 2 * m.c2)
            slot = [None, dt(self.img_dtype), None, None, None, z.buf.data_ptr(), self.N, self.H, self.W, m.c2, dt(self.dtype), L.ACT_NONE,
                    stats.data_ptr()]
            self.img_slots.append(slot)
            self._reg(m, "stem_train", slot)
            self.fwd.append((lib.cdet_stem_conv, slot))
        else:
            tiled = _use_tiled(lib, d)
            s2t = not tiled and _use_tiled_s2(lib, d)
            nblk = (lib.cdet_conv2d_tiled_stat_blocks if tiled else (lib.cdet_conv2d_s2_tiled_stat_blocks if s2t else lib.cdet_conv2d_stat_blocks))(C.byref(d))
            stats = self._vec(nblk * 2 * m.c2)
            fold_fwd = bool(self._bn_fold and not self.sync_bn and ((tiled and lib.cdet_conv2d_tiled_bn_ok(C.byref(d))) or
                                                                      (s2t and lib.cdet_conv2d_s2_tiled_bn_ok(C.byref(d)))))
            if fold_fwd:
                # train form with the statistics finished in the launch: [desc, x, w, z, stats, fold descriptor (bound below)]
                slot = [C.byref(d), x.buf.data_ptr(), None, z.buf.data_ptr(), stats.data_ptr(), None]
                self._reg(m, "train_fwd_t", slot)
                self.fwd.append((lib.cdet_conv2d_tiled_bn if tiled else lib.cdet_conv2d_s2_tiled_bn, slot))
            else:
                slot = [C.byref(d), x.buf.data_ptr(), None, None, None, None, z.buf.data_ptr(), stats.data_ptr()]
                self._reg(m, "train_fwd_t" if (tiled or s2t) else "train_fwd", slot)
                self.fwd.append((lib.cdet_conv2d_tiled if tiled else (lib.cdet_conv2d_s2_tiled if s2t else lib.cdet_conv2d), slot))
        mean, invstd = self._vec(m.c2), self._vec(m.c2)
        if d is not None:
            self.keep.append(d)
        bn = m.bn
        sync = self.sync_bn
        silu_call = (lib.cdet_bn_silu_fwd, [z.buf.data_ptr(), z.ld, z.coff, mean.data_ptr(), invstd.data_ptr(), bn.weight.data_ptr(), bn.bias.data_ptr(),
                                            res.buf.data_ptr() if res else None, res.ld if res else 0, res.coff if res else 0, y.buf.data_ptr(), y.ld, y.coff,
                                            z.M, m.c2, dt(self.dtype)])
        if sync:
            # SyncBatchNorm (reference train.py:140-143): per-layer [sum, sumsq] all-reduced over the ranks between two kernels. Inside a
            # group of independent layers (_sbn_group: the six parallel chains of a Detect head) the vectors of all layers sit in ONE
            # buffer and travel in ONE all-reduce; finalize + activation of the group follow it.
            grp = self._sbn_fwd
            fsum = grp["take"](2 * m.c2) if grp is not None else self._vec(2 * m.c2)
            self._f(lib.cdet_bn_bwd_sums, stats.data_ptr(), nblk, m.c2, fsum.data_ptr(), None, None, 0)
            defer = (not frozen_here) and self._alt_grad(bn.weight) is not None
            upd = not (frozen_here or defer)
            fin = (lib.cdet_bn_finalize, [fsum.data_ptr(), 1, m.c2, z.M * self.world, float(bn.eps), float(bn.momentum),
                                          bn.running_mean.data_ptr() if upd else None, bn.running_var.data_ptr() if upd else None,
                                          mean.data_ptr(), invstd.data_ptr()])
            if defer:  # (as in the per-GPU list below: the running statistics of a shared block are updated behind the block, in task order)
                if grp is not None:  # the group's buffer is recycled by the next group: keep this layer's all-reduced sums
                    raise NotImplementedError("grouped SyncBatchNorm statistics on a block shared by several tasks")
                sm_, si_ = self._vec(m.c2), self._vec(m.c2)
                self.deferred_stats.setdefault(self._cur_block, []).append(
                    (lib.cdet_bn_finalize, [fsum.data_ptr(), 1, m.c2, z.M * self.world, float(bn.eps), float(bn.momentum),
                                            bn.running_mean.data_ptr(), bn.running_var.data_ptr(), sm_.data_ptr(), si_.data_ptr()]))
            if grp is not None:
                grp["deferred"] += [fin, silu_call]
            else:
                self.fwd.append((self._allreduce_call(fsum, ("f", id(bn))), []))
                self.fwd += [fin, silu_call]
        else:
            # A later task of a shared block (see _alt_grad) must not touch the running statistics before the earlier task has: its finalize
            # leaves them alone, and the SAME kernel runs once more -- on the same partial sums, into scratch outputs -- behind the block,
            # ordered after the earlier task's update (iter_forward): same arithmetic in the same order as the sequential schedule.
            defer = (not frozen_here) and self._alt_grad(bn.weight) is not None
            upd = not (frozen_here or defer)
            count = z.M
            unbias = count / (count - 1) if count > 1 else 1.0
            if fold_fwd:
                totals = self._vec(2 * m.c2) if defer else None  # the fp32 [sum, sumsq] totals: what the deferred update below reads

                def fill(fd, part, totals=totals, upd=upd):
                    fd.totals = totals.data_ptr() if totals is not None else None
                    fd.mean, fd.invstd = mean.data_ptr(), invstd.data_ptr()
                    fd.running_mean = bn.running_mean.data_ptr() if upd else None
                    fd.running_var = bn.running_var.data_ptr() if upd else None
                    fd.inv_count, fd.unbias, fd.eps, fd.momentum = 1.0 / count, unbias, float(bn.eps), float(bn.momentum)

                slot[5] = self._fold_desc(nblk, m.c2, fill).data_ptr()
                self.n_folded[0] += 1
                if defer:  # the later task's running-statistics updates of a block travel in ONE launch behind it (cdet_bn_running_update)
                    self._deferred_items.setdefault(self._cur_block, []).append((totals, bn, 1.0 / count, unbias))
            else:
                self._f(lib.cdet_bn_finalize, stats.data_ptr(), nblk, m.c2, z.M, float(bn.eps), float(bn.momentum),
                        bn.running_mean.data_ptr() if upd else None, bn.running_var.data_ptr() if upd else None, mean.data_ptr(),
                        invstd.data_ptr())
                if defer:
                    sm_, si_ = self._vec(m.c2), self._vec(m.c2)
                    self.deferred_stats.setdefault(self._cur_block, []).append(
                        (lib.cdet_bn_finalize, [stats.data_ptr(), nblk, m.c2, z.M, float(bn.eps), float(bn.momentum), bn.running_mean.data_ptr(),
                                                bn.running_var.data_ptr(), sm_.data_ptr(), si_.data_ptr()]))
            self.fwd.append(silu_call)
        if frozen_here:
            return  # no backward for a frozen block, and num_batches_tracked does not advance
        bn._nbt_pending = getattr(bn, "_nbt_pending", 0)
        self._bn_seen.append(bn)
        rec = dict(kind="conv", m=m, x=x, z=z, y=y, res=res, mean=mean, invstd=invstd, stem=stem, block=self._cur_block, fwd_hi=len(self.fwd))
        self.trace.append(rec)

        def backward(need_dx=need_dx_default):
            gy = self.grad(y)
            assert self.written.query(gy), "gradient of a conv output was never produced"
            rec.update(gy=gy, gx=None, gx_acc=False, bwd_group=len(self.bwd_groups), bwd_lo=len(self._cur_bwd), grouped=False)
            nb = lib.cdet_bn_bwd_blocks(z.M)
            self._part_elems = max(self._part_elems, nb * 2 * m.c2 + 2 * m.c2)
            gw, gb = self._ensure_grad(bn.weight), self._ensure_grad(bn.bias)
            cw = self._ensure_grad(m.conv.weight)
            stem8 = getattr(m, "_stem8", False)
            red = [gy.buf.data_ptr(), gy.ld, gy.coff, z.buf.data_ptr(), z.ld, z.coff, mean.data_ptr(), invstd.data_ptr(), bn.weight.data_ptr(),
                   bn.bias.data_ptr(), None, z.M, m.c2, dt(self.dtype)]
            small = lambda v: v.M * v.ld * 2 < (1 << 31) - 65536  # noqa: E731 -- (the lean kernels' 32-bit addressing, csrc/elementwise.hip::bn_small)
            fold_bwd = self._bn_fold and not sync and small(gy) and small(z) and m.c2 % 8 == 0
            if fold_bwd:
                red.append(None)  # [14] the fold descriptor
                self._cur_bwd.append((lib.cdet_bn_silu_bwd_reduce_fold, red))
                self.n_folded[1] += 1
            else:
                self._cur_bwd.append((lib.cdet_bn_silu_bwd_reduce, red))
            bgrp = self._sbn_bwd if sync else None
            if sync:
                bsum = bgrp["take"](2 * m.c2) if bgrp is not None else self._vec(2 * m.c2)
                sm = [None, nb, m.c2, bsum.data_ptr(), gw.data_ptr(), gb.data_ptr(), 1]  # local dgamma/dbeta, like torch's SyncBatchNorm
                self._cur_bwd.append((lib.cdet_bn_bwd_sums, sm))
                if bgrp is None:
                    self._cur_bwd.append((self._allreduce_call(bsum, ("b", id(bn))), []))
                app = [gy.buf.data_ptr(), gy.ld, gy.coff, z.buf.data_ptr(), z.ld, z.coff, mean.data_ptr(), invstd.data_ptr(), bn.weight.data_ptr(),
                       bn.bias.data_ptr(), bsum.data_ptr(), 0, None, None, 1, None, m.c2, 0, z.M, m.c2, dt(self.dtype), z.M * self.world]
            else:
                sm = None
                app = [gy.buf.data_ptr(), gy.ld, gy.coff, z.buf.data_ptr(), z.ld, z.coff, mean.data_ptr(), invstd.data_ptr(), bn.weight.data_ptr(),
                       bn.bias.data_ptr(), None, 0 if fold_bwd else nb, gw.data_ptr(), gb.data_ptr(), 1, None, m.c2, 0, z.M, m.c2, dt(self.dtype), 0]
                if fold_bwd:  # the reduce launch leaves the sums [2C] behind the partial rows and writes dgamma / dbeta itself (nblk = 0 form)
                    def fill_b(fd, part):
                        fd.totals = part.data_ptr() + nb * 2 * m.c2 * 4
                        fd.dgamma, fd.dbeta, fd.accumulate = gw.data_ptr(), gb.data_ptr(), 1

                    red[14] = self._fold_desc(nb, m.c2, fill_b).data_ptr()
            if bgrp is not None:  # everything behind the group's all-reduce is emitted when the group closes (same relative order)
                emit_to, self._cur_bwd = self._cur_bwd, bgrp["deferred"]
            if shortcut is not None:
                gs = self.grad(shortcut)
                assert self.written.query(gs), "the shortcut's gradient slice must have a first writer before the residual sum reaches it"
                rec["also"] = gs
                app += [gs.buf.data_ptr(), gs.ld, gs.coff]
                self._cur_bwd.append((lib.cdet_bn_silu_bwd_apply_add, app))
            else:
                self._cur_bwd.append((lib.cdet_bn_silu_bwd_apply, app))
            dzd = None
            if x is not None:
                dzd = conv_desc(x, z, k, s)  # wgrad descriptor: forward geometry, dy = dz scratch [M, c2]
                dzd.dst_ld, dzd.dst_coff = m.c2, 0
                self._wgrad_elems = max(self._wgrad_elems, lib.cdet_conv2d_wgrad_ws_elems(C.byref(dzd)))
            dg_slot = None
            if need_dx and id(x.buf) not in self._nograd:
                gx = self.grad(x)
                acc = self.written.query(gx)
                dd = L.ConvDesc()
                dd.N, dd.Hs, dd.Ws, dd.Cs = z.N, z.H, z.W, m.c2
                dd.Hd, dd.Wd, dd.Cd = x.H, x.W, x.C
                dd.kh = dd.kw = k
                dd.stride, dd.pad, dd.mode = s, k // 2, L.CONV_DGRAD
                dd.dtype, dd.out_dtype, dd.act = dt(self.dtype), dt(self.dtype), L.ACT_NONE
                dd.src_ld, dd.src_coff, dd.dst_ld, dd.dst_coff = m.c2, 0, gx.ld, gx.coff
                dd.res_ld, dd.res_coff = (gx.ld, gx.coff) if acc else (0, 0)
                dd.accumulate = 0
                # stride-1 data gradient = forward convolution of dz with the tap-flipped, transposed (DGRAD) tiled operand
                dd.mode = L.CONV_FWD
                dg_tiled = s == 1 and _use_tiled(lib, dd)
                if not dg_tiled:
                    dd.mode = L.CONV_DGRAD
                # stride 2: the four parity classes of dX as stride-1 convolutions of dz with taps of the same DGRAD operand (csrc/conv_vt.hip)
                dg_s2 = not dg_tiled and s == 2 and _use_tiled_s2(lib, dd)
                self.keep.append(dd)
                dg_slot = [C.byref(dd), None, None, None, None, gx.buf.data_ptr() if acc else None, gx.buf.data_ptr(), None]
                self._reg(m, "dgrad_t" if (dg_tiled or dg_s2) else "dgrad", dg_slot)
                self._cur_bwd.append((lib.cdet_conv2d_tiled_dgrad if dg_tiled else (lib.cdet_conv2d_s2_tiled_dgrad if dg_s2 else lib.cdet_conv2d), dg_slot))
                self.written.mark(gx)
                rec.update(gx=gx, gx_acc=acc)
            self.keep.append(dzd)
            own_dz = None
            stem_wg = None
            if x is None:
                # direct stem: weight gradient straight from the NCHW image (csrc/stem_wgrad.hip); [0] = the image pointer of the run
                assert stem
                sws = self._vec(lib.cdet_stem_conv_wgrad_ws_elems(self.N, self.H, self.W))
                wg = None
                stem_wg = [None, dt(self.img_dtype), None, m.c2, dt(self.dtype), cw.data_ptr(), self.N, self.H, self.W, m.c2, 1, sws.data_ptr()]
                self.img_slots.append(stem_wg)
                self._cur_bwd.append((lib.cdet_stem_conv_wgrad, stem_wg))
            elif self._wg_group and not stem8 and lib.cdet_conv2d_wgrad_groupable(C.byref(dzd)):
                # same-geometry 3x3 layers of a block (the Bottleneck convolutions of a C2f) share ONE weight-gradient launch at the
                # end of the block's backward (_flush_wgrads): their dz must outlive the shared scratch, so each gets its own buffer
                own_dz = self._alloc((z.M, m.c2), self.dtype)
                self._wg_pending.append(dict(desc=dzd, x=x, dz=own_dz, dw=cw,
                                             key=(z.N, z.H, z.W, x.C, m.c2, dzd.dst_ld, dzd.dst_coff, dzd.dtype)))
                wg = None
                rec["grouped"] = True
            elif stem8:  # weight gradient lands in the channel-padded scratch, then its first 3 input channels are accumulated into dW
                wg = [C.byref(dzd), x.buf.data_ptr(), None, m._gw8.data_ptr(), None, 0]
                self._cur_bwd.append((lib.cdet_conv2d_wgrad, wg))
                O_, c_in, kh_, kw_ = m.conv.weight.shape
                self._cur_bwd.append((lib.cdet_fold_padded_wgrad, [m._gw8.data_ptr(), cw.data_ptr(), O_, m._gw8.shape[1], c_in, kh_ * kw_, 1]))
            else:
                wg = [C.byref(dzd), x.buf.data_ptr(), None, cw.data_ptr(), None, 1]
                self._cur_bwd.append((lib.cdet_conv2d_wgrad, wg))

            if bgrp is not None:
                self._cur_bwd = emit_to
            rec["bwd_hi"] = len(self._cur_bwd)

            def bind(dz, part, ws):
                rec["dz"] = own_dz if own_dz is not None else dz
                red[10] = part.data_ptr()
                if sm is not None:
                    sm[0] = part.data_ptr()
                else:
                    app[10] = part.data_ptr() + (nb * 2 * m.c2 * 4 if fold_bwd else 0)
                dzp = (own_dz if own_dz is not None else dz).data_ptr()
                app[15] = dzp
                if dg_slot is not None:
                    dg_slot[1] = dzp
                if wg is not None:
                    wg[2] = dzp
                    wg[4] = ws.data_ptr()
                if stem_wg is not None:
                    stem_wg[2] = dzp

            self._late.append(bind)

        if bwd_ops is not None:
            bwd_ops.append(backward)

    def _stem_unit(self, m: Conv, y: View, bwd_ops):
        """First backbone row (Cin = 3, 3x3 stride 2): forward through the direct MFMA stem kernel on the NCHW image (uint8 * 1/255 or
        float; csrc/stem_mfma.hip), weight gradient from the same image (csrc/stem_wgrad.hip). A stem of any other geometry repacks the image to
        NHWC with channels padded to 8 and runs on the generic kernels."""
        lib = self.lib
        if m.c1 > 8:
            raise NotImplementedError("stem with more than 8 input channels")
        N, H, W = self.N, self.H, self.W
        direct = m.k == 3 and m.s == 2 and m.c2 % 8 == 0 and m.c2 <= 96 and H % 2 == 0 and W % 2 == 0
        if direct and (m.c2 <= 80 or not self._train_here):  # (the weight-gradient kernel's tile is 80 couts wide)
            # forward AND weight gradient read the NCHW image itself (stem_mfma.hip, stem_wgrad.hip): no 8-channel copy of it at all
            self._conv_unit(m, None, y, None, bwd_ops, need_dx_default=False, stem=True)
            return
        x8 = self._new(N, H, W, 8)
        slot = [None, dt(self.img_dtype), x8.buf.data_ptr(), N, H, W, dt(self.dtype)]
        self.img_slots.append(slot)
        self.fwd.append((lib.cdet_image_to_nhwc8, slot))
        if getattr(m, "_w8", None) is None or m._w8.device != self.device:
            m._w8 = torch.zeros((m.c2, 8, m.k, m.k), dtype=torch.float32, device=self.device)
            m._gw8 = torch.zeros_like(m._w8)
        m._stem8 = True
        self._conv_unit(m, x8, y, None, bwd_ops, need_dx_default=False, stem=direct)

    def _stem_conv1_fusable(self, blk, place) -> bool:
        """Eval plans: backbone rows 0 and 1 -- Conv(3, c1, 3, 2) and Conv(c1, c2, 3, 2) -- run as ONE kernel that keeps the stem's map in LDS
        (csrc/stem_conv1.hip) when nothing else reads row 0 and the geometry fits. CDET_STEM_FUSE=0 switches it off (A/B timing, tests)."""
        if self.training or os.environ.get("CDET_STEM_FUSE", "1") == "0" or len(blk.model) < 2:
            return False
        m0, m1 = blk.model[0], blk.model[1]
        if not (isinstance(m0, Conv) and isinstance(m1, Conv) and m1.f == -1):
            return False
        if not (m0.k == 3 and m0.s == 2 and m0.c1 == 3 and m1.k == 3 and m1.s == 2 and m1.c1 == m0.c2):
            return False
        if m0.conv.groups != 1 or m1.conv.groups != 1:
            return False
        for li, layer in enumerate(blk.model):  # another reader of row 0 (a skip connection, a neck tap)?
            f = layer.f
            for j in ([f] if isinstance(f, int) else list(f)):
                if j == 0 or (j < -1 and li + j == 0):
                    return False
        if any(kind == "bb" and j == 0 for ins in self.model._inputs.values() for kind, j in ins):
            return False
        pl = place.get(("bb", 1))
        ld, coff = (m1.c2, 0)
        if pl is not None:
            ld, coff = -(-pl[2] // 64) * 64, pl[1]
        return bool(self.lib.cdet_stem_conv1_ok(self.N, self.H, self.W, m0.c2, m1.c2, dt(self.img_dtype), dt(self.dtype), ld, coff))

    def _stem_conv1_unit(self, m0: Conv, m1: Conv, y: View):
        lib = self.lib
        self.convs += [m0, m1]
        ok = lib.cdet_stem_conv1_ok(self.N, self.H, self.W, m0.c2, m1.c2, dt(self.img_dtype), dt(self.dtype), y.ld, y.coff)
        assert ok, "stem + second-row fusion refused a geometry _stem_conv1_fusable accepted"
        slot = [None, dt(self.img_dtype), None, None, None, None, None, None, y.buf.data_ptr(), self.N, self.H, self.W, m0.c2, m1.c2,
                dt(self.dtype), y.ld, y.coff, L.ACT_SILU]
        self.img_slots.append(slot)
        self._reg(m0, "stemc1", slot)      # [2] packed stem operand, [3] / [4] the stem's folded scale / bias
        self._reg(m1, "stemc1_w1", slot)   # [5] tiled forward operand of the second row, [6] / [7] its folded scale / bias
        self.fwd.append((lib.cdet_stem_conv1, slot))
        self.trace.append(dict(kind="stemc1", m0=m0, m1=m1, y=y, block=self._cur_block, fwd_hi=len(self.fwd)))

    def _bias_unit(self, m: nn.Conv2d, x: View, feat: View, dfeat: Optional[View], bwd_ops):
        """Head projection nn.Conv2d(c, o, 1) + bias -> fp32 slice of the head map; o is padded to a multiple of 8."""
        lib = self.lib
        self.biased.append(m)
        d = conv_desc(x, feat, 1, 1)
        slot = [C.byref(d), x.buf.data_ptr(), None, None, None, None, feat.buf.data_ptr(), None]
        self.keep.append(d)
        # round 4: the tap-resident kernel writes fp32 destinations (HEPI_F32 epilogue of csrc/conv_halo.hip), so the projections leave the
        # round-1 generic kernel (13 - 79 TF/s on these shapes)
        tiled = os.environ.get("CDET_PROJ_TILED", "1") != "0" and _use_tiled(lib, d)
        self._reg(m, "bias_fwd_t" if tiled else "bias_fwd", slot)
        self.fwd.append((lib.cdet_conv2d_tiled if tiled else lib.cdet_conv2d, slot))
        self._out_ptr_slots.append((slot, 6, feat.buf))  # (argument list, index, plan-owned tensor): see fresh_outputs()
        if not self.training:
            self.trace.append(dict(kind="ebias", m=m, x=x, feat=feat, block=self._cur_block, fwd_hi=len(self.fwd)))
        if not self._train_here:
            return
        rec = dict(kind="bias", m=m, x=x, feat=feat, dfeat=dfeat, block=self._cur_block, fwd_hi=len(self.fwd))
        self.trace.append(rec)

        def backward(need_dx=True):
            gx = self.grad(x)
            acc = self.written.query(gx)
            rec.update(gx=gx, gx_acc=acc, bwd_group=len(self.bwd_groups), bwd_lo=len(self._cur_bwd))
            # round 6: the projection's data gradient on the tap-resident kernel too -- a FORWARD 1x1 convolution of dfeat with the tiled DGRAD operand
            # (rows = input channels, reduction = the pad8(o) map channels; rows / columns beyond the real ones are zero in the operand), the gradient
            # already in gx rides in as the residual. The round-1 generic kernel ran these twelve launches at 44 TF/s (0.31 ms per iteration).
            dd = conv_desc(dfeat, gx, 1, 1, L.CONV_FWD, L.ACT_NONE, gx if acc else None)
            dg_tiled = os.environ.get("CDET_PROJ_TILED", "1") != "0" and _use_tiled(lib, dd)
            if not dg_tiled:
                dd = conv_desc(dfeat, gx, 1, 1, L.CONV_DGRAD, L.ACT_NONE, gx if acc else None)
            self.keep.append(dd)
            dg = [C.byref(dd), dfeat.buf.data_ptr(), None, None, None, gx.buf.data_ptr() if acc else None, gx.buf.data_ptr(), None]
            self._reg(m, "dgrad_t" if dg_tiled else "dgrad", dg)
            self._cur_bwd.append((lib.cdet_conv2d_tiled_dgrad if dg_tiled else lib.cdet_conv2d, dg))
            rec["dgrad_tiled"] = dg_tiled
            self.written.mark(gx)
            wd = conv_desc(x, dfeat, 1, 1)
            wd.Cd = m.out_channels
            self.keep.append(wd)
            self._wgrad_elems = max(self._wgrad_elems, lib.cdet_conv2d_wgrad_ws_elems(C.byref(wd)))
            cw, cb = self._ensure_grad(m.weight), self._ensure_grad(m.bias)
            wg = [C.byref(wd), x.buf.data_ptr(), dfeat.buf.data_ptr(), cw.data_ptr(), None, 1]
            nb = lib.cdet_bn_bwd_blocks(dfeat.M)
            self._part_elems = max(self._part_elems, nb * dfeat.C)
            cs = [dfeat.buf.data_ptr(), dfeat.ld, dfeat.coff, dfeat.M, dfeat.C, m.out_channels, dt(dfeat.dtype), cb.data_ptr(), 1, None]
            self._cur_bwd += [(lib.cdet_conv2d_wgrad, wg), (lib.cdet_colsum, cs)]
            rec["bwd_hi"] = len(self._cur_bwd)

            def bind(dz, part, ws):
                wg[4] = ws.data_ptr()
                cs[9] = part.data_ptr()

            self._late.append(bind)

        bwd_ops.append(backward)

    # ------------------------------------------------------------------------------------------------ composite modules
    def _c2f(self, m: C2f, x: View, bwd_ops) -> View:
        c, n = m.c, m.n
        Ho, Wo = x.H, x.W
        cat = self._new(x.N, Ho, Wo, (2 + n) * c, row_align=64)
        out = self._out(x.N, Ho, Wo, m.c2)
        self._conv_unit(m.cv1, x, cat.slice(0, 2 * c), None, bwd_ops)
        for i, b in enumerate(m.m):
            src, dst = cat.slice((1 + i) * c, c), cat.slice((2 + i) * c, c)
            t = self._new(x.N, Ho, Wo, c)
            self._conv_unit(b.cv1, src, t, None, bwd_ops)
            # y = src + cv2(cv1(src)): the gradient of dst flows into cv2's backward AND into grad(src); cv2's BatchNorm backward pass
            # does both (executed before cv1's data gradient accumulates into the same slice)
            self._conv_unit(b.cv2, t, dst, src if b.add else None, bwd_ops, shortcut=src if (b.add and self._train_here) else None)
        self._conv_unit(m.cv2, cat, out, None, bwd_ops)
        return out

    def _sppf(self, m: SPPF, x: View, bwd_ops) -> View:
        c_ = m.c1 // 2
        buf = self._new(x.N, x.H, x.W, 4 * c_)
        out = self._out(x.N, x.H, x.W, m.c2)
        self._conv_unit(m.cv1, x, buf.slice(0, c_), None, bwd_ops)
        self._f(self.lib.cdet_sppf_pool, buf.buf.data_ptr(), buf.ld, 0, buf.N, buf.H, buf.W, c_, dt(self.dtype))
        if not self.training:
            self.trace.append(dict(kind="epool", buf=buf, c=c_, block=self._cur_block, fwd_hi=len(self.fwd)))
        if self._train_here:
            prec = dict(kind="pool", buf=buf, c=c_, block=self._cur_block, fwd_hi=len(self.fwd))
            self.trace.append(prec)

            def pool_bwd(need_dx=True):
                g = self.grad(buf)
                assert self.written.query(g)
                prec.update(g=g, bwd_group=len(self.bwd_groups), bwd_lo=len(self._cur_bwd), bwd_hi=len(self._cur_bwd) + 1)
                self._b(self.lib.cdet_sppf_pool_bwd, buf.buf.data_ptr(), g.buf.data_ptr(), buf.ld, 0, buf.N, buf.H, buf.W, c_, dt(self.dtype))
            bwd_ops.append(pool_bwd)
        self._conv_unit(m.cv2, buf, out, None, bwd_ops)
        return out

    def _materialize(self, v) -> View:
        if isinstance(v, _Deferred):
            out = self._new(v.N, v.H, v.W, v.C)
            self._upsample_into(v.src, out, self._cur_ops)
            return out
        if isinstance(v, _VirtualCat):  # a consumer that cannot walk the parts itself: build the tensor after all
            cat = self._new(v.N, v.H, v.W, v.C, row_align=64)
            off = 0
            for part, up in v.parts:
                dst = cat.slice(off, part.C)
                if up:
                    self._upsample_into(part, dst, self._cur_ops)
                else:
                    self._f(self.lib.cdet_copy_channels, part.buf.data_ptr(), part.ld, part.coff, dst.buf.data_ptr(), dst.ld, dst.coff, part.M, part.C,
                            dt(self.dtype), 0)
                off += part.C
            return cat
        return v

    def _upsample_into(self, src: View, dst: View, bwd_ops):
        self._f(self.lib.cdet_upsample2, src.buf.data_ptr(), src.ld, src.coff, dst.buf.data_ptr(), dst.ld, dst.coff, src.N, src.H, src.W, src.C,
                dt(self.dtype))
        if self._train_here and id(src.buf) not in self._nograd:
            urec = dict(kind="up", src=src, dst=dst, block=self._cur_block, fwd_hi=len(self.fwd))
            self.trace.append(urec)

            def up_bwd(need_dx=True):
                gd, gs = self.grad(dst), self.grad(src)
                assert self.written.query(gd)
                acc = self.written.query(gs)
                urec.update(gd=gd, gs=gs, acc=acc, bwd_group=len(self.bwd_groups), bwd_lo=len(self._cur_bwd), bwd_hi=len(self._cur_bwd) + 1)
                self._b(self.lib.cdet_upsample2_bwd, gd.buf.data_ptr(), gd.ld, gd.coff, gs.buf.data_ptr(), gs.ld, gs.coff, src.N, src.H, src.W,
                        src.C, dt(self.dtype), int(acc))
                self.written.mark(gs)
            bwd_ops.append(up_bwd)

    def _concat(self, xs: list, bwd_ops) -> View:
        xs = [self._materialize(v) if isinstance(v, _VirtualCat) else v for v in xs]
        if self._vcat and len(xs) <= 3 and all(v.C % 32 == 0 for v in xs[:-1]) and xs[-1].C % 8 == 0:
            # eval plans (round 4): no buffer at all -- the consumer's 1x1 convolution reads the parts (and upsamples on the fly)
            return _VirtualCat([(v.src, True) if isinstance(v, _Deferred) else (v, False) for v in xs])
        x0 = xs[0]
        Ctot = sum(v.C for v in xs)
        cat = self._cat_bufs.get(self._cur_block)  # allocated by the producer of an input that lives in its slice (see _out)
        if cat is None:
            cat = self._new(x0.N, x0.H, x0.W, Ctot, row_align=64)
        assert cat.C == Ctot and (cat.N, cat.H, cat.W) == (x0.N, x0.H, x0.W)
        off = 0
        for v in xs:
            dst = cat.slice(off, v.C)
            if isinstance(v, View) and v.buf is cat.buf and v.coff == dst.coff and v.C == dst.C:
                pass  # written in place by its producer: nothing to copy, and its gradient is the slice's gradient
            elif isinstance(v, _Deferred):
                self._upsample_into(v.src, dst, bwd_ops)
            else:
                self._f(self.lib.cdet_copy_channels, v.buf.data_ptr(), v.ld, v.coff, dst.buf.data_ptr(), dst.ld, dst.coff, v.M, v.C, dt(self.dtype), 0)
                if self._train_here and id(v.buf) not in self._nograd:
                    crec = dict(kind="copy", src=v, dst=dst, block=self._cur_block, fwd_hi=len(self.fwd))
                    self.trace.append(crec)

                    def copy_bwd(need_dx=True, v=v, dst=dst, crec=crec):
                        gd, gs = self.grad(dst), self.grad(v)
                        assert self.written.query(gd)
                        acc = self.written.query(gs)
                        crec.update(gd=gd, gs=gs, acc=acc, bwd_group=len(self.bwd_groups), bwd_lo=len(self._cur_bwd), bwd_hi=len(self._cur_bwd) + 1)
                        self._b(self.lib.cdet_copy_channels, gd.buf.data_ptr(), gd.ld, gd.coff, gs.buf.data_ptr(), gs.ld, gs.coff, v.M, v.C,
                                dt(self.dtype), int(acc))
                        self.written.mark(gs)
                    bwd_ops.append(copy_bwd)
            off += v.C
        return cat

    def _layer(self, m, xs: list, bwd_ops):
        if isinstance(m, Conv):
            x = self._materialize(xs[0])
            p = m.k // 2
            y = self._out(x.N, (x.H + 2 * p - m.k) // m.s + 1, (x.W + 2 * p - m.k) // m.s + 1, m.c2)
            self._conv_unit(m, x, y, None, bwd_ops)
            return y
        if isinstance(m, C2f):
            return self._c2f(m, xs[0] if isinstance(xs[0], _VirtualCat) else self._materialize(xs[0]), bwd_ops)
        if isinstance(m, SPPF):
            return self._sppf(m, self._materialize(xs[0]), bwd_ops)
        if isinstance(m, Upsample):
            return _Deferred(self._materialize(xs[0]))
        if isinstance(m, Concat):
            return self._concat(xs, bwd_ops)
        raise NotImplementedError(type(m).__name__)

    def _sbn_group(self, mods, bwd_ops):
        """SyncBatchNorm only: open a group over the INDEPENDENT Conv units `mods` compiled next (same inputs ready, no unit feeds
        another). Forward: their [sum, sumsq] vectors share one buffer and ONE all-reduce, emitted by the returned close() together with
        the deferred finalize / activation launches. Backward: the mirror image -- the units' reduce + partial-sum launches run first,
        one all-reduce of all backward sums, then every unit's apply / data-gradient / weight-gradient launches in their own order.
        The reference's SyncBatchNorm all-reduces per layer (train.py:140-143: 2 x 97 small collectives per task pass); the six parallel
        chains of a Detect head (models/yolo.py:80-100) make 12 of them 2."""
        total = sum(2 * m.c2 for m in mods)
        gkey = tuple(id(m.bn) for m in mods)

        def pool():
            buf = self._vec(total)
            st = dict(off=0, deferred=[], buf=buf)

            def take(n):
                v = buf[st["off"]:st["off"] + n]
                st["off"] += n
                return v
            st["take"] = take
            return st

        fwd = self._sbn_fwd = pool()

        def bwd_close():  # runs LAST of the group in the reversed backward walk: all reduces are in, one collective, then the rest
            g = self._sbn_bwd
            self._sbn_bwd = None
            assert g["off"] == total
            self._cur_bwd.append((self._allreduce_call(g["buf"], ("b",) + gkey), []))
            self._cur_bwd += g["deferred"]

        def bwd_open():   # runs FIRST of the group in the reversed walk
            self._sbn_bwd = pool()

        bwd_ops.append(bwd_close)

        def close():
            assert fwd["off"] == total
            self._sbn_fwd = None
            self.fwd.append((self._allreduce_call(fwd["buf"], ("f",) + gkey), []))
            self.fwd += fwd["deferred"]
            bwd_ops.append(bwd_open)

        return close

    def _detect(self, head, task: str, xs: List[View], bwd_ops):
        nc, ncp = head.nc, _PAD8(head.nc)
        ld = 64 + ncp
        feats, dfeats = [], []
        xs = [self._materialize(x) for x in xs]
        chains = []  # (level, branch index, modules, input, a, b, map slice, gradient slice)
        for lvl, x in enumerate(xs):
            fbuf = self._new(x.N, x.H, x.W, ld, torch.float32, zero=True)
            dbuf = self._new(x.N, x.H, x.W, ld, self.dtype, zero=True) if self.training else None
            feats.append(fbuf.buf)
            dfeats.append(dbuf.buf if dbuf else None)
            for bi, (branch, c_out, coff, width) in enumerate(((head.cv2[lvl], 64, 0, 64), (head.cv3[lvl], nc, 64, ncp))):
                chains.append((lvl, bi, branch, x, fbuf.slice(coff, width), dbuf.slice(coff, width) if dbuf else None))
        if self.sync_bn and self._train_here:
            # SyncBatchNorm: stage-major order -- the six first convolutions, ONE statistics all-reduce, the six second convolutions, one
            # more, then the projections (and the mirror image in the backward): 4 collectives per head and pass instead of 24
            bufs = [(self._new(x.N, x.H, x.W, br[0].c2), self._new(x.N, x.H, x.W, br[1].c2)) for _, _, br, x, _, _ in chains]
            for stage in (0, 1):
                close = self._sbn_group([br[stage] for _, _, br, _, _, _ in chains], bwd_ops)
                for (lvl, bi, br, x, fsl, dsl), (a, b) in zip(chains, bufs):
                    self._conv_unit(br[stage], x if stage == 0 else a, a if stage == 0 else b, None, bwd_ops)
                close()
            for (lvl, bi, br, x, fsl, dsl), (a, b) in zip(chains, bufs):
                self._bias_unit(br[2], b, fsl, dsl, bwd_ops)
        else:
            for lvl, bi, branch, x, fsl, dsl in chains:
                c_start = len(self.fwd)
                a = self._new(x.N, x.H, x.W, branch[0].c2)
                b = self._new(x.N, x.H, x.W, branch[1].c2)
                self._conv_unit(branch[0], x, a, None, bwd_ops)
                self._conv_unit(branch[1], a, b, None, bwd_ops)
                self._bias_unit(branch[2], b, fsl, dsl, bwd_ops)
                self.head_chains.setdefault(task, []).append((lvl, bi, c_start, len(self.fwd)))  # six independent chains per head
        self.feats[task], self.dfeats[task] = feats, dfeats
        if not self.training:
            A = sum(f.shape[1] * f.shape[2] for f in feats)
            out_dtype = torch.float32 if self.img_dtype in (torch.float32, torch.uint8) else self.img_dtype
            y = torch.empty((self.N, 4 + nc, A), dtype=out_dtype, device=self.device)
            hw = (C.c_int32 * 6)(*[v for f in feats for v in (f.shape[1], f.shape[2])])
            st = (C.c_float * 3)(*[float(s) for s in head.stride])
            self.keep += [hw, st]
            self._f(self.lib.cdet_detect_decode, feats[0].data_ptr(), feats[1].data_ptr(), feats[2].data_ptr(), hw, st, self.N, nc, ld,
                    L.F32, y.data_ptr(), dt(out_dtype))
            dec = self.fwd[-1][1]
            self._out_ptr_slots += [(dec, 0, feats[0]), (dec, 1, feats[1]), (dec, 2, feats[2]), (dec, 9, y)]
            self.y[task] = y
            self.trace.append(dict(kind="decode", task=task, head=head, feats=list(feats), y=y, block=self._cur_block, fwd_hi=len(self.fwd)))

    # ------------------------------------------------------------------------------------------------ build
    def _build(self):
        model = self.model
        self._bn_seen: List[nn.Module] = []
        order, _ = model.execution_plan(self.tasks)
        outs: Dict[int, object] = {}
        ops_per_block: List[tuple] = []
        # ---- pre-pass: which Conv / C2f / SPPF outputs can be produced straight into a later Concat's buffer. Every output goes to
        #      the FIRST Concat of the plan that consumes it (a second consumer -- the other task's neck -- copies from there).
        #      Not with a frozen trunk: its dead blocks and the live neck would share one buffer's gradient bookkeeping.
        self._cat_bufs: Dict[int, View] = {}
        self._cur_place = None
        self._cur_block = -1
        place: Dict[tuple, tuple] = {}
        # eval plans: Concat blocks are virtual (the consumer's 1x1 convolution walks their inputs, _VirtualCat) -- then nothing is
        # placed into concat buffers either; CDET_VCAT=0: the round-3 form (in-place producers + upsample / copy launches)
        self._vcat = not self.training and os.environ.get("CDET_VCAT", "1") != "0" and os.environ.get("CDET_CONV_TILED", "1") != "0"
        if not self.frozen and not self._vcat and os.environ.get("CDET_CONCAT_INPLACE", "1") != "0":
            def src_module(kind, j):
                return model.blocks[0].model[j] if kind == "bb" else model.blocks[j]

            def channels(kind, j):
                mod = src_module(kind, j)
                if kind == "blk" and j == 0:
                    mod = model.blocks[0].model[-1]
                if isinstance(mod, (Conv, C2f, SPPF)):
                    return mod.c2
                if isinstance(mod, Upsample):
                    return channels(*model._inputs[j][0])
                if isinstance(mod, Concat):
                    return sum(channels(k2, j2) for k2, j2 in model._inputs[j])
                raise NotImplementedError(type(mod).__name__)

            # A TRAINING plan of several tasks: an output that two Concats consume (a backbone tap feeding both tasks' necks) stays in
            # a buffer of its own. In the reversed backward walk the second task's copy would write only that channel slice of the
            # first Concat's gradient before the Concat's own consumer writes the whole range (overwrite vs accumulate is decided per
            # whole range at compile time).
            n_cat_consumers: Dict[tuple, int] = {}
            for idx in order:
                if idx != 0 and isinstance(model.blocks[idx], Concat):
                    for key in model._inputs[idx]:
                        n_cat_consumers[tuple(key)] = n_cat_consumers.get(tuple(key), 0) + 1
            for idx in order:
                if idx != 0 and isinstance(model.blocks[idx], Concat):
                    ins = model._inputs[idx]
                    ctot = sum(channels(k2, j2) for k2, j2 in ins)
                    off = 0
                    for k2, j2 in ins:
                        cn = channels(k2, j2)
                        key = (k2, j2)
                        shared = self.training and n_cat_consumers[key] > 1
                        if isinstance(src_module(k2, j2), (Conv, C2f, SPPF)) and key not in place and cn % 8 == 0 and off % 8 == 0 and not shared:
                            place[key] = (idx, off, ctot)
                        off += cn
        for idx in order:
            blk = model.blocks[idx]
            self._cur_block = idx
            # gradient-dead blocks: frozen parameters (or none) and only gradient-dead producers -- the frozen shared trunk incl. its
            # parameter-free Upsample / Concat blocks
            producers = [0 if kind == "bb" else j for kind, j in model._inputs.get(idx, [])] if idx != 0 else []
            inputs_dead = all(j in self.dead for j in producers)
            has_params = any(True for _ in blk.parameters())
            if self.training and idx in self.frozen:
                if not inputs_dead:
                    raise NotImplementedError(f"block {idx} is frozen but fed by a trainable block: only a frozen trunk prefix is supported")
                self.dead.add(idx)
            elif self.training and self.frozen and not has_params and inputs_dead:
                self.dead.add(idx)
            self._train_here = self.training and idx not in self.dead
            bwd_ops: list = []
            self._cur_ops = bwd_ops
            for p in blk.parameters():
                self.block_of_param[id(p)] = idx
            if idx == 0:
                ys: List[object] = []
                cur = None
                fused2 = self._stem_conv1_fusable(blk, place)
                for li, layer in enumerate(blk.model):
                    f = layer.f
                    if self._train_here:
                        # the reversed walk reaches this closure when row li's backward is complete: flush the row's grouped weight gradients and
                        # note the position -- the trainer folds / all-reduces the trunk's gradient bucket row by row, under the rest of the
                        # backward (reference: DDP's 25 MB buckets, train.py:182-184), instead of as one 124 MB message behind it
                        def row_mark(li=li):
                            self._flush_wgrads()
                            self._sub_marks.append((li, len(self._cur_bwd)))
                        bwd_ops.append(row_mark)
                    if fused2 and li == 0:
                        ys.append(None)  # the stem's map is never materialised (csrc/stem_conv1.hip)
                        continue
                    if fused2 and li == 1:
                        p = layer.k // 2
                        h1, w1 = (self.H + 2 - 3) // 2 + 1, (self.W + 2 - 3) // 2 + 1
                        self._cur_place = place.get(("bb", li))
                        y = self._out(self.N, (h1 + 2 * p - layer.k) // layer.s + 1, (w1 + 2 * p - layer.k) // layer.s + 1, layer.c2)
                        self._cur_place = None
                        self._stem_conv1_unit(blk.model[0], layer, y)
                        cur = y
                        ys.append(cur)
                        continue
                    if li == 0:
                        p = layer.k // 2
                        y = self._new(self.N, (self.H + 2 * p - layer.k) // layer.s + 1, (self.W + 2 * p - layer.k) // layer.s + 1, layer.c2)
                        self._stem_unit(layer, y, bwd_ops)
                        cur = y
                    else:
                        if f == -1:
                            xin = [cur]
                        elif isinstance(f, int):
                            xin = [ys[f]]
                        else:
                            xin = [cur if j == -1 else ys[j] for j in f]
                        self._cur_place = place.get(("bb", li))
                        cur = self._layer(layer, xin, bwd_ops)
                        self._cur_place = None
                    ys.append(cur)
                outs[0] = ys
            else:
                xs = [outs[0][j] if kind == "bb" else outs[j] for kind, j in model._inputs[idx]]
                if idx in model.heads.values():
                    task = model.controllers[idx].task_id
                    self._detect(blk, task, xs, bwd_ops)
                else:
                    self._cur_place = place.get(("blk", idx))
                    outs[idx] = self._layer(blk, xs, bwd_ops)
                    self._cur_place = None
            ops_per_block.append((idx, bwd_ops))
            self.fwd_marks.append((idx, len(self.fwd)))
        self._train_here = self.training
        if self.training:
            # head map gradients are produced by the loss kernel (or copied in by the autograd bridge)
            for t in self.tasks:
                for d in self.dfeats[t]:
                    self.written.mark(View(d))
            for idx, bwd_ops in reversed(ops_per_block):
                self._cur_bwd = []
                self._sub_marks = []
                for op in reversed(bwd_ops):
                    op()
                self._flush_wgrads()
                self.bwd_groups.append((idx, self._cur_bwd))
                if self._sub_marks and self._cur_bwd:
                    assert self._sub_marks[-1][1] == len(self._cur_bwd)
                    self.bwd_sub[idx] = self._sub_marks
            dz = self._vec(max(self._dz_elems, 8), self.dtype)
            part = self._vec(max(self._part_elems, 8))
            ws = self._vec(max(self._wgrad_elems, 8))
            for bind in self._late:
                bind(dz, part, ws)
            self._bind_folds(part)
            self._bind_deferred_items()
        self._late = []
        if not self.training and os.environ.get("CDET_EVAL_LANES", "1") != "0":
            self._build_lanes()
        self.n_fwd_calls = len(self.fwd)
        self.n_bwd_calls = sum(len(c) for _, c in self.bwd_groups)

    # ------------------------------------------------------------------------------------------------ stream lanes (eval)
    def _build_lanes(self):
        """Eval-form launch list -> segments on HIP stream lanes. The reference runs the block DAG sequentially
        (cerberus.py:804-882); here the parts that do not depend on each other run concurrently so that one kernel's partly
        filled last round of workgroups and its prologue / epilogue sit under another kernel's MFMA loop:
          lane 0            blocks that serve two or more of the plan's tasks (the shared trunk), then the first task's chain;
          lane k (1..K-1)   task k's exclusive neck + the class chain of the head's last level + decode;
          lane K + k        task k's five other head chains (six chains per Detect head are independent: yolo.py:87-100); round 4: the
                            chains of every level but the last start right behind the neck block that produces their input.
        Cross-lane order is enforced with events: task lanes wait for the last trunk segment before them, a head's side lane
        waits for its neck, decode waits for the side lane, and lane 0 ends by waiting for every other lane (so the caller sees
        ordinary stream order). Results are bit-identical to the single-stream schedule: the same kernels on the same buffers."""
        model = self.model
        tasks = self.tasks
        head_of = {model.heads[t]: t for t in tasks}
        main_lane = {t: k for k, t in enumerate(tasks)}
        side_lane = {t: len(tasks) + k for k, t in enumerate(tasks)}  # 2 tasks: the caller's stream + lanes 1..3 = 4 hardware queues
        segs = []  # [lane, start, end, wait keys, record key, order]; start == end: a pure event-record point
        pos = 0
        last_trunk = None
        seen_trunk = {}  # lane -> last trunk key it already waited for
        n_ev = 0
        end_of = {}      # block idx -> (lane, end position) of its segment
        early = os.environ.get("CDET_EARLY_HEADS", "1") != "0"

        def waits_for_trunk(lane):
            if lane == 0 or last_trunk is None or seen_trunk.get(lane) == last_trunk:
                return []
            seen_trunk[lane] = last_trunk
            return [last_trunk]

        def add(lane, a_, b_, waits, rec, order=None):
            segs.append([lane, a_, b_, waits, rec, order if order is not None else (a_, b_, 0)])

        for idx, end in self.fwd_marks:
            start, pos = pos, end
            if start == end:
                continue
            if idx in head_of:
                t = head_of[idx]
                ml, sl = main_lane[t], side_lane[t]
                neck_key, side_key = ("neck", t), ("side", t)
                chains = self.head_chains.get(t, [])
                # Round 4: the chains of a level start as soon as THAT level's neck output exists (yolo.py:87-100 reads one input per
                # level): the 80 x 80 level -- two thirds of the head's work -- is ready one bottom-up stage before the head block, the
                # 40 x 40 level half a stage. Those chains go to the side lane right behind their producer's block, ordered by an event of
                # their own; only the last level's chains start where the head block stands in the launch list.
                prod = {}
                n_lvl = 1 + max((c[0] for c in chains), default=0)
                if early:
                    for lvl, (kind, j) in enumerate(model._inputs.get(idx, [])):
                        if kind == "blk" and j in end_of and end_of[j][0] == ml and lvl < n_lvl - 1:
                            prod[lvl] = j
                late = [c for c in chains if c[0] not in prod]
                late_side = [c for c in late if not (c[0] == late[0][0] and c[1] == 1)] if late else []
                add(ml, start, start, waits_for_trunk(ml), neck_key)  # the head's inputs are complete on the main lane here
                k_early = 0
                for lvl in sorted(prod):
                    lane_p, pe = end_of[prod[lvl]]
                    key = ("lvl", t, lvl)
                    add(lane_p, pe, pe, [], key, (pe, pe, 0))             # record point behind the producer's block
                    for n_, (l2, bi, cs, ce) in enumerate(c for c in chains if c[0] == lvl):
                        k_early += 1
                        add(sl, cs, ce, [key] if n_ == 0 else [], None, (pe, pe, k_early))
                cur = start
                for lvl, bi, cs, ce in late:
                    if late and lvl == late[0][0] and bi == 1:
                        add(ml, cs, ce, [], None)                          # the heaviest late chain stays on the task's main lane
                    else:
                        first, last = (lvl, bi) == late_side[0][:2], (lvl, bi) == late_side[-1][:2]
                        add(sl, cs, ce, [neck_key] if first else [], side_key if last else None)
                    cur = ce
                if k_early and not late_side:
                    add(sl, start, start, [], side_key)                    # (no late chain on the side lane: its early chains still gate the decode)
                cur = max([cur] + [c[3] for c in chains])
                if cur < end:  # decode needs all six chains
                    add(ml, cur, end, [side_key] if (late_side or k_early) else [], None)
                continue
            served = [t for t in tasks if t in getattr(model.controllers[idx], "serving_tasks", {})] if idx != 0 else list(tasks)
            if idx == 0 or len(served) != 1:
                n_ev += 1
                last_trunk = ("trunk", n_ev)
                add(0, start, end, [], last_trunk)
                end_of[idx] = (0, end)
            else:
                lane = main_lane[served[0]]
                add(lane, start, end, waits_for_trunk(lane), None)
                end_of[idx] = (lane, end)
        # host issue order: launch-list order, record points in front of the segment that starts where they stand; an early head chain
        # right behind its producer's record point (stable sort)
        segs.sort(key=lambda sg: sg[5])
        segs = [sg[:5] for sg in segs]
        lanes = sorted({sg[0] for sg in segs})
        if len(lanes) <= 1:
            return
        self.sched = dict(segs=segs, lanes=lanes, streams=None, events=None)

    def _run_lanes(self, stream):
        sc = self.sched
        if sc["streams"] is None:
            sc["streams"] = {ln: (None if ln == 0 else lane_stream(self.device, ln)) for ln in sc["lanes"]}
            keys = {sg[4] for sg in sc["segs"] if sg[4] is not None}
            sc["events"] = {k: torch.cuda.Event() for k in keys}
            sc["final"] = {ln: torch.cuda.Event() for ln in sc["lanes"] if ln != 0}
            sc["start"] = torch.cuda.Event()
        streams, events = sc["streams"], sc["events"]
        sc["start"].record(stream)  # side lanes may not start before the work queued ahead of this forward on the caller's stream
        started = set()
        for lane, a, b, waits, rec in sc["segs"]:
            s_ = stream if lane == 0 else streams[lane]
            if lane != 0 and lane not in started:
                started.add(lane)
                s_.wait_event(sc["start"])
            for k in waits:
                s_.wait_event(events[k])
            st = s_.cuda_stream
            for fn, args in self.fwd[a:b]:
                rc = fn(*args, st)
                if rc:
                    L.check(rc, fn.__name__)
            if rec is not None:
                events[rec].record(s_)
        for ln, ev in sc["final"].items():
            ev.record(streams[ln])
            stream.wait_event(ev)

    # ------------------------------------------------------------------------------------------------ run
    def fresh_outputs(self, fresh: bool = True):
        """Eval plans: point the launches that WRITE the outputs a caller gets (the head projections' fp32 maps, the decode kernel's
        `y`) at a newly allocated set of tensors, so that `model(x)` returns fresh tensors like the reference does
        (cerberus.py:804-882) without a device copy: 13 pointer patches per task on the host, nothing on the GPU (round 3 cloned
        the maps through a strided transposing copy: 1.29 ms per 2-task forward at batch 32). `fresh=False` goes back to the
        plan-owned set (zero-copy callers: CerberusDetInference, val.run). Everything else -- trunk, necks, head convolutions --
        keeps its compiled buffers. The tensors come from torch's caching allocator on the caller's stream; the side lanes that
        write into them are joined into that stream before run_forward returns, so a later reuse of the memory is ordered."""
        assert not self.training
        if self._home_outputs is None:
            self._home_outputs = ({t: list(v) for t, v in self.feats.items()}, dict(self.y))
        if not fresh and self._outputs_are_home:
            return
        home_f, home_y = self._home_outputs
        remap = {}
        for t in self.tasks:
            new_f = [torch.empty_like(f) for f in home_f[t]] if fresh else home_f[t]
            new_y = torch.empty_like(home_y[t]) if fresh else home_y[t]
            for old, new in zip(home_f[t] + [home_y[t]], new_f + [new_y]):
                remap[id(old)] = new
            self.feats[t], self.y[t] = list(new_f), new_y
        for slot, i, owner in self._out_ptr_slots:
            slot[i] = remap[id(owner)].data_ptr()
        self._outputs_are_home = not fresh

    _outputs_are_home = True

    def _module_block(self, m) -> int:
        w = m.conv.weight if hasattr(m, "conv") else m.weight
        return self.block_of_param.get(id(w), -1)

    def refresh_weights(self, part: Optional[str] = None):
        """(Re)pack weights of every Conv on the path when the model's weights changed (version counter). Train mode packs all
        stale modules of the plan (forward + DGRAD operands) with ONE batched launch; the item table is cached per set of
        stale modules (a plan sees two sets: everything, or everything but the blocks another task's plan already packed).
        part (training plans, trainer-driven): "early" = only the modules of self.early_blocks (the shared trunk, packed before the task
        streams fork), "late" = the rest (packed by the pass itself in front of its first other block, behind the optimizer's tail: see
        iter_forward); None = everything."""
        ver = self.model._weights_version
        if self.training:
            key = (ver, self.dtype, True)
            stale = [(0, m) for m in self.convs if getattr(m, "_pack_key", None) != key]
            stale += [(1, m) for m in self.biased if getattr(m, "_pack_key", None) != key]
            if part is not None:
                early = self.early_blocks
                stale = [(k, m) for k, m in stale if (self._module_block(m) in early) == (part == "early")]
                if not stale:
                    return
            if part is not None or (len(stale) > 4 and os.environ.get("CDET_PACK_BATCHED", "1") != "0"):
                if stale:
                    self._pack_batched(stale, key)
                return
        for m in self.convs:
            _pack_conv(m, self.dtype, self.training, ver, self.lib)
        for m in self.biased:
            _pack_biased(m, self.dtype, self.training, ver, self.lib)

    def _pack_batched(self, stale, key):
        lib, dtype, dev = self.lib, self.dtype, self.device
        sig = tuple((id(m), _needs(m)) for _, m in stale)
        tabs = self.__dict__.setdefault("_pack_tabs", {})
        tab = tabs.get(sig)
        if tab is not None and not all(getattr(m, a, None) is t for m, a, t in tab[3]):
            tab = None  # another plan (other dtype) re-allocated a packed buffer: rebuild the table
        if tab is None:
            items = []
            titems = []
            owners = []
            for kind, m in stale:
                need = _needs(m)
                if kind == 0 and (need & (_T_FWD | _T_DGRAD)):  # tiled operands of the tap-resident kernel
                    w = m.conv.weight
                    O, I, kh, kw = w.shape
                    _alloc_tiled(m, lib, dtype, dev, need)
                    wf = m._wt_f if need & _T_FWD else None
                    wd = m._wt_d if need & _T_DGRAD else None
                    if wf is not None:
                        owners.append((m, "_wt_f", wf))
                    if wd is not None:
                        owners.append((m, "_wt_d", wd))
                    titems.append((w, wf, wd, O, I, kh, kw))
                if kind == 1 and (need & (_T_FWD | _T_DGRAD)):  # a head projection whose forward / data gradient runs on the tap-resident kernel
                    w = m.weight
                    O, I, kh, kw = w.shape
                    _alloc_tiled_biased(m, lib, dtype, dev, need)
                    wf = m._wt_f if need & _T_FWD else None
                    wd = m._wt_d if need & _T_DGRAD else None
                    if wf is not None:
                        owners.append((m, "_wt_f", wf))
                    if wd is not None:
                        owners.append((m, "_wt_d", wd))
                    titems.append((w, wf, wd, O, I, kh, kw))
                if kind == 0 and not (need & (_G_FWD | _G_DGRAD)):
                    continue
                if kind == 0:
                    w = m._w8 if getattr(m, "_stem8", False) else m.conv.weight
                    O, I, kh, kw = w.shape
                    Op = O
                else:
                    w = m.weight
                    O, I, kh, kw = w.shape
                    Op = _PAD8(O)
                assert kh * kw <= 9
                # (a Conv whose forward runs on the tiled kernel still gets the generic forward operand when only its data gradient
                #  needs the generic kernel: the batched packer always writes w_fwd)
                # the batched kernel writes valid elements only: padding (K tail, rows O..Op-1) is zeroed here, once
                if getattr(m, "_wp", None) is None or m._wp.dtype != dtype or not getattr(m, "_wp_zeroed", False):
                    m._wp = torch.zeros(lib.cdet_packed_weight_elems(Op, I, kh, kw, 0), dtype=dtype, device=dev)
                    m._wpt = None
                    m._wp_zeroed = True
                    if kind == 1:
                        m._bias_pad = torch.zeros(Op, dtype=torch.float32, device=dev)
                owners.append((m, "_wp", m._wp))
                wt = None
                if kind == 1 or (need & _G_DGRAD):  # (the stem needs no data gradient -> no transposed pack)
                    if m._wpt is None:
                        m._wpt = torch.zeros(lib.cdet_packed_weight_elems(Op, I, kh, kw, 1), dtype=dtype, device=dev)
                    wt = m._wpt
                    owners.append((m, "_wpt", m._wpt))
                items.append((w, m._wp, wt, O, Op, I, kh, kw))
            arr = (L.PackItem * len(items))()
            blk = 0
            for it, (w, wf, wt, O, Op, I, kh, kw) in zip(arr, items):
                nb = ((O + 31) // 32) * ((I + 31) // 32)
                it.w_oihw, it.w_fwd, it.w_dgrad = w.data_ptr(), wf.data_ptr(), (wt.data_ptr() if wt is not None else None)
                it.O, it.O_pad, it.I, it.kh, it.kw, it.first_block, it.n_blocks = O, Op, I, kh, kw, blk, nb
                blk += nb
            dtab = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8).to(dev) if items else None
            tarr = (L.PackTiledItem * max(len(titems), 1))()
            tblk = 0
            for it, (w, wf, wd, O, I, kh, kw) in zip(tarr, titems):
                nb = ((O + 31) // 32) * ((I + 31) // 32)
                it.w_oihw, it.w_fwd, it.w_dgrad = w.data_ptr(), (wf.data_ptr() if wf is not None else None), (wd.data_ptr() if wd is not None else None)
                it.O, it.I, it.kh, it.kw, it.first_block, it.n_blocks = O, I, kh, kw, tblk, nb
                tblk += nb
            ttab = torch.frombuffer(bytearray(bytes(tarr)), dtype=torch.uint8).to(dev) if titems else None
            tab = tabs[sig] = (dtab, len(items), blk, owners, ttab, len(titems), tblk)
        dtab, n, nblk, _, ttab, tn, tnblk = tab
        with torch.no_grad():
            for kind, m in stale:
                if kind == 0 and getattr(m, "_stem8", False):
                    m._w8[:, :m.conv.weight.shape[1]].copy_(m.conv.weight.detach())
                elif kind == 1:
                    m._bias_pad[:m.bias.shape[0]].copy_(m.bias.detach().float())
        st = torch.cuda.current_stream().cuda_stream
        if n:
            L.check(lib.cdet_pack_weights_batched(dtab.data_ptr(), n, nblk, dt(dtype), st), "cdet_pack_weights_batched")
        if tn:
            L.check(lib.cdet_pack_weights_tiled(ttab.data_ptr(), tn, tnblk, dt(dtype), st), "cdet_pack_weights_tiled")
        for kind, m in stale:
            for sk, slot in getattr(m, "_plan_slots", []):
                if kind == 0 and sk == "stem_train":
                    slot[2] = m.conv.weight.data_ptr()
                elif kind == 0 and sk == "train_fwd":
                    slot[2] = m._wp.data_ptr()
                elif kind == 0 and sk == "train_fwd_t":
                    slot[2] = m._wt_f.data_ptr()
                elif kind == 1 and sk in ("bias_fwd", "bias_fwd_t"):
                    slot[2] = (m._wp if sk == "bias_fwd" else m._wt_f).data_ptr()
                    slot[4] = m._bias_pad.data_ptr()
                elif sk == "dgrad":
                    slot[2] = m._wpt.data_ptr()
                elif sk == "dgrad_t":
                    slot[2] = m._wt_d.data_ptr()
            m._pack_key = key

    def run_forward(self, img: torch.Tensor):
        for _ in self.iter_forward(img):
            pass

    def iter_forward(self, img: torch.Tensor, fired: Optional[set] = None):
        """Generator form of the forward launch list, for the trainer's interleaved multi-stream schedule: with a BlockSync attached
        it yields None after every block (the caller may let another task enqueue its next block) and yields an event while that
        event -- which the next block has to wait for -- has not been recorded in this iteration (`fired` holds the ids of the
        recorded ones). Re-reads the current stream after every resume: the caller selects it around each next()."""
        assert img.is_contiguous() and tuple(img.shape) == (self.N, 3, self.H, self.W) and img.dtype == self.img_dtype, \
            f"plan compiled for {(self.N, 3, self.H, self.W)} {self.img_dtype}, got {tuple(img.shape)} {img.dtype}"
        # trainer-driven task passes on streams: the shared trunk's operands were packed before the fork; this pass packs the rest -- its own
        # branch -- in front of its first block outside the trunk, behind the optimizer's tail (Averaging.optimizer_step updates those blocks
        # on a side stream while the next iteration's trunk already runs)
        lazy = self.training and self.block_sync is not None and bool(self.early_blocks)
        if not lazy:
            self.refresh_weights()
        self._img = img
        self.generation = getattr(self, "generation", 0) + 1  # (autograd_bridge refuses a backward across a newer forward)
        p = img.data_ptr()
        for s in self.img_slots:
            s[0] = p
        stream = torch.cuda.current_stream()
        st = stream.cuda_stream
        sy = self.block_sync
        if self.sched is not None and sy is None:
            self._run_lanes(stream)
        elif sy is None:
            for fn, args in self.fwd:
                rc = fn(*args, st)
                if rc:
                    L.check(rc, fn.__name__)
            for idx in sorted(self.deferred_stats):  # (one stream: the earlier task's pass is already in front of this one)
                for fn, args in self.deferred_stats[idx]:
                    rc = fn(*args, st)
                    if rc:
                        L.check(rc, fn.__name__)
        else:  # task passes on separate streams
            pos = 0
            decoupled = self.decoupled
            late_done = not lazy
            for idx, end in self.fwd_marks:
                if not late_done and idx not in self.early_blocks:
                    late_done = True
                    if self.tail_event is not None:
                        torch.cuda.current_stream().wait_event(self.tail_event)
                    self.refresh_weights("late")
                ev = sy.wait_fwd.get(idx)
                if ev is not None and not decoupled:  # a block shared with an earlier task waits for it (shared running statistics)
                    while fired is not None and id(ev) not in fired:
                        yield ev
                    torch.cuda.current_stream().wait_event(ev)
                stream = torch.cuda.current_stream()
                st = stream.cuda_stream
                for fn, args in self.fwd[pos:end]:
                    rc = fn(*args, st)
                    if rc:
                        L.check(rc, fn.__name__)
                pos = end
                dfr = self.deferred_stats.get(idx)
                if dfr:  # decoupled: only the running-statistics updates of the block wait for the earlier task's
                    if ev is not None:
                        while fired is not None and id(ev) not in fired:
                            yield ev
                        torch.cuda.current_stream().wait_event(ev)
                    stream = torch.cuda.current_stream()
                    st = stream.cuda_stream
                    for fn, args in dfr:
                        rc = fn(*args, st)
                        if rc:
                            L.check(rc, fn.__name__)
                ev = sy.done_fwd.get(idx)
                if ev is not None:
                    ev.record(stream)
                    if fired is not None:
                        fired.add(id(ev))
                if fired is not None:
                    yield None
        if self.training:
            for bn in self._bn_seen:
                bn._nbt_pending = getattr(bn, "_nbt_pending", 0) + 1

    def loss(self, task: str, gt: torch.Tensor, gains: dict, grad_scale: float = 1.0, want_assign: bool = False, scaler: Optional[torch.Tensor] = None):
        """Fused criterion on this plan's head maps (utils/loss.py:133-181 of the reference): writes d(loss)/d(maps) straight
        into the plan's head-gradient buffers. gt: [N, n_max, 5] fp32 (cls, x1, y1, x2, y2 px). Returns loss5 (device):
        (box, cls, dfl, total, 2*N*total); call run_backward() next."""
        lib = self.lib
        head = self.model.get_head(task)
        feats, dfe = self.feats[task], self.dfeats[task]
        d = L.LossDesc()
        d.N, d.nc, d.n_max = self.N, head.nc, gt.shape[1]
        for i, f in enumerate(feats):
            d.hw[2 * i], d.hw[2 * i + 1] = f.shape[1], f.shape[2]
            d.stride[i] = float(head.stride[i])
        d.gain_box, d.gain_cls, d.gain_dfl = float(gains["box"]), float(gains["cls"]), float(gains["dfl"])
        d.grad_scale = float(grad_scale)
        d.grad_scale_dev = scaler.data_ptr() if scaler is not None else None  # GradScaler scale on the device (trainers/averaging.py; fp16 plans)
        d.dtype, d.grad_dtype = L.F32, dt(self.dtype)
        d.f_ld, d.topk, d.alpha, d.beta = feats[0].shape[3], 10, 0.5, 6.0
        need = lib.cdet_det_loss_ws_bytes(C.byref(d))
        ws = getattr(self, "_loss_ws", None)
        if ws is None or ws.numel() < need:
            ws = self._loss_ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        out = torch.empty(5, dtype=torch.float32, device=self.device)
        asg = {}
        if want_assign:
            A = sum(f.shape[1] * f.shape[2] for f in feats)
            asg = dict(fg_mask=torch.empty((self.N, A), dtype=torch.uint8, device=self.device),
                       target_gt_idx=torch.empty((self.N, A), dtype=torch.int32, device=self.device),
                       target_labels=torch.empty((self.N, A), dtype=torch.int32, device=self.device),
                       target_bboxes=torch.empty((self.N, A, 4), device=self.device),
                       target_scores=torch.empty((self.N, A, head.nc), device=self.device))
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        assert gt.is_contiguous() and gt.dtype == torch.float32 and gt.shape[0] == self.N and gt.shape[1] >= 1
        L.check(lib.cdet_det_loss(C.byref(d), p(feats[0]), p(feats[1]), p(feats[2]), p(gt), p(dfe[0]), p(dfe[1]), p(dfe[2]), p(out),
                                  p(asg.get("fg_mask")), p(asg.get("target_gt_idx")), p(asg.get("target_labels")), p(asg.get("target_bboxes")),
                                  p(asg.get("target_scores")), p(ws), torch.cuda.current_stream().cuda_stream), "cdet_det_loss")
        return (out, asg) if want_assign else out

    def attach_grads(self):
        """p.grad <- the model-owned buffer the kernels accumulate into. If someone dropped or replaced p.grad (e.g.
        optimizer.zero_grad(set_to_none=True)) the buffer is zeroed first, so stale sums never leak into a new step."""
        for p in self._params_seen.values():
            g = self.model._grad_buffer(p)
            if p.grad is not g:
                g.zero_()
                p.grad = g

    def run_backward(self):
        for _ in self.iter_backward():
            pass

    def iter_backward(self, fired: Optional[set] = None):
        """Generator form of the backward launch list (see iter_forward)."""
        self.attach_grads()
        sy = self.block_sync
        for idx, calls in self.bwd_groups:
            if sy is not None and not self.decoupled:  # (decoupled: this task's gradients of a shared block go to a bucket of their own)
                ev = sy.wait_bwd.get(idx)
                if ev is not None:
                    while fired is not None and id(ev) not in fired:
                        yield ev
                    torch.cuda.current_stream().wait_event(ev)
            pos = 0
            for row, end in list(self.bwd_sub.get(idx, ())) + [(None, len(calls))]:
                if end > pos or row is not None:
                    stream = torch.cuda.current_stream()
                    st = stream.cuda_stream
                    for fn, args in calls[pos:end]:
                        rc = fn(*args, st)
                        if rc:
                            L.check(rc, fn.__name__)
                    pos = end
                if row is not None:  # a backbone row's gradients are complete here
                    h = self.hooks.get((idx, row))
                    if h is not None:
                        h((idx, row))
                    if sy is not None and fired is not None and end < len(calls):
                        yield None
            stream = torch.cuda.current_stream()
            h = self.hooks.get(idx)
            if h is not None:
                h(idx)
            if sy is not None:
                ev = sy.done_bwd.get(idx)
                if ev is not None:
                    ev.record(stream)
                    if fired is not None:
                        fired.add(id(ev))
                if fired is not None:
                    yield None


class BlockSync:
    """Events that order one task's pass against the other tasks' passes on the blocks they share (shared BatchNorm running
    statistics and shared gradient buffers are read-modify-write): {block: event} to wait for before / record after the block's
    forward and backward launches."""

    __slots__ = ("wait_fwd", "done_fwd", "wait_bwd", "done_bwd")

    def __init__(self):
        self.wait_fwd, self.done_fwd, self.wait_bwd, self.done_bwd = {}, {}, {}, {}


# ---------------------------------------------------------------------------------------------------------------------
# weight preparation (per module, shared by all plans)
# ---------------------------------------------------------------------------------------------------------------------
_G_FWD, _G_DGRAD, _T_FWD, _T_DGRAD = 1, 2, 4, 8
_KIND_NEED = {"eval": _G_FWD, "train_fwd": _G_FWD, "dgrad": _G_DGRAD, "eval_t": _T_FWD, "train_fwd_t": _T_FWD, "dgrad_t": _T_DGRAD,
              "bias_fwd": _G_FWD, "bias_fwd_t": _T_FWD, "stemc1_w1": _T_FWD, "eval_tc": _T_FWD}


def _use_tiled(lib, d) -> bool:
    return os.environ.get("CDET_CONV_TILED", "1") != "0" and bool(lib.cdet_conv2d_tiled_ok(C.byref(d)))


def _use_tiled_s2(lib, d) -> bool:
    return (os.environ.get("CDET_CONV_TILED", "1") != "0" and os.environ.get("CDET_CONV_S2_TILED", "1") != "0"
            and d.stride == 2 and bool(lib.cdet_conv2d_s2_tiled_ok(C.byref(d))))


def _needs(m) -> int:
    """Which packed operands the launch lists that reference this Conv need: generic / tiled x forward / data gradient."""
    need = 0
    for kind, _ in getattr(m, "_plan_slots", []):
        need |= _KIND_NEED.get(kind, 0)
    return need


def _alloc_tiled(m, lib, dtype, dev, need):
    O, I, kh, kw = (m.conv.weight if hasattr(m, "conv") else m.weight).shape
    if need & _T_FWD and (getattr(m, "_wt_f", None) is None or m._wt_f.dtype != dtype):
        m._wt_f = torch.zeros(lib.cdet_tiled_weight_elems(O, I, kh, kw), dtype=dtype, device=dev)  # zeroed once: the packer skips padding
    if need & _T_DGRAD and (getattr(m, "_wt_d", None) is None or m._wt_d.dtype != dtype):
        m._wt_d = torch.zeros(lib.cdet_tiled_weight_elems(I, O, kh, kw), dtype=dtype, device=dev)


def _alloc_tiled_biased(m, lib, dtype, dev, need):
    """Tiled operands of a head projection nn.Conv2d(I, O, 1): the forward operand has pad8(O) rows (rows O.. stay zero: allocated zeroed, the packer
    writes real elements only), the DGRAD operand I rows over a reduction of O real channels (its last 32-channel chunk zero beyond O -- the map's pad
    channels multiply zeros)."""
    O, I, kh, kw = m.weight.shape
    if need & _T_FWD and (getattr(m, "_wt_f", None) is None or m._wt_f.dtype != dtype):
        m._wt_f = torch.zeros(lib.cdet_tiled_weight_elems(_PAD8(O), I, kh, kw), dtype=dtype, device=dev)
    if need & _T_DGRAD and (getattr(m, "_wt_d", None) is None or m._wt_d.dtype != dtype):
        m._wt_d = torch.zeros(lib.cdet_tiled_weight_elems(I, _PAD8(O), kh, kw), dtype=dtype, device=dev)


def _pack_conv(m: Conv, dtype, training, ver, lib):
    key = (ver, dtype, training)
    if getattr(m, "_pack_key", None) == key:
        return
    st = torch.cuda.current_stream().cuda_stream
    w = m.conv.weight
    need = _needs(m)
    if need & (_T_FWD | _T_DGRAD):
        _alloc_tiled(m, lib, dtype, w.device, need)
        wf = m._wt_f.data_ptr() if need & _T_FWD else None
        wd = m._wt_d.data_ptr() if (need & _T_DGRAD and training) else None
        if wf or wd:
            w32 = w.detach().float().contiguous()
            O, I, kh, kw = w32.shape
            L.check(lib.cdet_pack_weight_tiled(w32.data_ptr(), wf, wd, O, I, kh, kw, dt(dtype), st), "cdet_pack_weight_tiled")
    if getattr(m, "_stem8", False):
        with torch.no_grad():
            m._w8[:, :w.shape[1]].copy_(w.detach())
        w = m._w8
    O, I, kh, kw = w.shape
    if need & _G_FWD or (training and need & _G_DGRAD):
        if getattr(m, "_wp", None) is None or m._wp.dtype != dtype:
            m._wp = torch.empty(lib.cdet_packed_weight_elems(O, I, kh, kw, 0), dtype=dtype, device=w.device)
            m._wpt = None
    if need & _G_FWD:
        L.check(lib.cdet_pack_weight(w.data_ptr(), m._wp.data_ptr(), O, O, I, kh, kw, 0, None, dt(dtype), st), "cdet_pack_weight")
    scale = bias = None
    if training and not (need & _G_DGRAD):
        pass  # the stem needs no data gradient; stride-1 convs take theirs from the tiled DGRAD operand
    elif training:
        if getattr(m, "_wpt", None) is None or m._wpt.dtype != dtype:
            m._wpt = torch.empty(lib.cdet_packed_weight_elems(O, I, kh, kw, 1), dtype=dtype, device=w.device)
        L.check(lib.cdet_pack_weight(w.data_ptr(), m._wpt.data_ptr(), O, O, I, kh, kw, 1, None, dt(dtype), st), "cdet_pack_weight")
    else:
        with torch.no_grad():
            if m.fused:
                bias = m.conv.bias.detach().float().contiguous()
            else:
                bn = m.bn
                scale = (bn.weight / torch.sqrt(bn.running_var + bn.eps)).float().contiguous()
                bias = (bn.bias - bn.running_mean * scale).float().contiguous()
        m._scale, m._bias = scale, bias
    for kind, slot in getattr(m, "_plan_slots", []):
        if kind in ("stem_eval", "stem_train"):
            wm = m.conv.weight
            assert wm.dtype == torch.float32 and wm.is_contiguous()
            slot[2] = wm.data_ptr()  # the fp32 OIHW master itself: the stem kernel converts its 96 x 32 operand on the fly
            if kind == "stem_eval" and not training:
                slot[3] = scale.data_ptr() if scale is not None else None
                slot[4] = bias.data_ptr() if bias is not None else None
        elif kind == "stemc1" and not training:  # row 0 inside the fused first-two-rows kernel: its MFMA operand, packed once per weight version
            wm = m.conv.weight
            n = lib.cdet_stem_conv1_pack_elems(wm.shape[0])
            if getattr(m, "_ws1", None) is None or m._ws1.dtype != dtype or m._ws1.numel() != n:
                m._ws1 = torch.empty(n, dtype=dtype, device=wm.device)
            assert wm.dtype == torch.float32 and wm.is_contiguous()
            L.check(lib.cdet_stem_conv1_pack(wm.data_ptr(), m._ws1.data_ptr(), wm.shape[0], dt(dtype), st), "cdet_stem_conv1_pack")
            slot[2] = m._ws1.data_ptr()
            slot[3] = scale.data_ptr() if scale is not None else None
            slot[4] = bias.data_ptr() if bias is not None else None
        elif kind == "stemc1_w1" and not training:
            slot[5] = m._wt_f.data_ptr()
            slot[6] = scale.data_ptr() if scale is not None else None
            slot[7] = bias.data_ptr() if bias is not None else None
        elif kind in ("eval", "eval_t") and not training:
            slot[2] = (m._wp if kind == "eval" else m._wt_f).data_ptr()
            slot[3] = scale.data_ptr() if scale is not None else None
            slot[4] = bias.data_ptr() if bias is not None else None
        elif kind == "eval_tc" and not training:  # 1x1 over a virtual Concat (cdet_conv2d_tiled_cat: weights / scale / bias one slot further)
            slot[3] = m._wt_f.data_ptr()
            slot[4] = scale.data_ptr() if scale is not None else None
            slot[5] = bias.data_ptr() if bias is not None else None
        elif kind == "train_fwd" and training:
            slot[2] = m._wp.data_ptr()
        elif kind == "train_fwd_t" and training:
            slot[2] = m._wt_f.data_ptr()
        elif kind == "dgrad" and training:
            slot[2] = m._wpt.data_ptr()
        elif kind == "dgrad_t" and training:
            slot[2] = m._wt_d.data_ptr()
    m._pack_key = key


def _pack_biased(m: nn.Conv2d, dtype, training, ver, lib):
    key = (ver, dtype, training)
    if getattr(m, "_pack_key", None) == key:
        return
    st = torch.cuda.current_stream().cuda_stream
    w = m.weight
    O, I, kh, kw = w.shape
    Op = _PAD8(O)
    if getattr(m, "_wp", None) is None or m._wp.dtype != dtype:
        m._wp = torch.empty(lib.cdet_packed_weight_elems(Op, I, kh, kw, 0), dtype=dtype, device=w.device)
        m._wpt = None
        m._bias_pad = torch.zeros(Op, dtype=torch.float32, device=w.device)
    L.check(lib.cdet_pack_weight(w.data_ptr(), m._wp.data_ptr(), O, Op, I, kh, kw, 0, None, dt(dtype), st), "cdet_pack_weight")
    with torch.no_grad():
        m._bias_pad[:O].copy_(m.bias.detach().float())
    need = _needs(m)
    if need & (_T_FWD | (_T_DGRAD if training else 0)):  # forward / data gradient on the tap-resident kernel (padding stays zero: allocated zeroed)
        _alloc_tiled_biased(m, lib, dtype, w.device, need)
        L.check(lib.cdet_pack_weight_tiled(w.detach().float().contiguous().data_ptr(), m._wt_f.data_ptr() if need & _T_FWD else None,
                                           m._wt_d.data_ptr() if (need & _T_DGRAD and training) else None, O, I, kh, kw, dt(dtype), st),
                "cdet_pack_weight_tiled")
    if training:
        if m._wpt is None:
            m._wpt = torch.empty(lib.cdet_packed_weight_elems(Op, I, kh, kw, 1), dtype=dtype, device=w.device)
        L.check(lib.cdet_pack_weight(w.data_ptr(), m._wpt.data_ptr(), O, Op, I, kh, kw, 1, None, dt(dtype), st), "cdet_pack_weight")
    for kind, slot in getattr(m, "_plan_slots", []):
        if kind in ("bias_fwd", "bias_fwd_t"):
            slot[2] = (m._wp if kind == "bias_fwd" else m._wt_f).data_ptr()
            slot[4] = m._bias_pad.data_ptr()
        elif kind == "dgrad" and training:
            slot[2] = m._wpt.data_ptr()
        elif kind == "dgrad_t" and training:
            slot[2] = m._wt_d.data_ptr()
    m._pack_key = key
