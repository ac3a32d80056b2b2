"""Training-step and Gatys-step executors.

StyleTrainer restates the per-step data flow of train_style_network
(reference full_graph_stylizer_network.py:198-216): content targets from the VGG
replica fed with the batch, stylizer forward, VGG + Gram + losses on the
stylized batch, backward to the 48 stylizer variables, TF1 Adam.  GatysOptimizer
restates normal_style_transfer (full_graph_stylizer_network.py:257-279,
:308-329): the image itself is the variable.

The kernel sequence of a step is static, so it is captured once into HIP graphs
and replayed.  With data parallelism the stylizer backward is cut into block
ranges; after each range the gradient bucket it completed is all-reduced (RCCL)
while the next range runs.
"""
import numpy as np
import torch

from . import ops, tuning
from .stylizer import StylizerNet
from .tuning import SERIAL as _SERIAL
from .vggnet import VggFeatures


def _segments(cuts):
    """Block ranges (hi..lo) of the stylizer backward from the blocks each later range starts at."""
    tops = [15] + sorted((int(c) - 1 for c in cuts), reverse=True)
    los = [t + 1 for t in tops[1:]] + [0]
    return list(zip(tops, los))


# Block ranges (hi..lo) of the stylizer backward; one all-reduce bucket each, reduced while the next range
# runs.  Every extra range costs about 47 us per step on one MI355X (a graph boundary, and the weight-gradient
# branch drained at it), so there are two.  The cut sits where the LAST bucket -- the one no backward work is
# left to hide -- is small: blocks 15..3 own 6.29 MB of the 6.71 MB of gradients and are reduced under the
# backward of blocks 2..0 (the three full-resolution layers, the longest stretch of the pass per parameter);
# the 0.40 MB behind blocks 2..0 is exposed, and a collective of that size costs its latency, not bandwidth.
# Adam then runs per bucket, so the update of the large bucket overlaps the reduction of the small one.
# This default was chosen on ONE rank (graph-boundary cost measured, all-reduce time estimated); it has not
# been timed with real peers.  tuning.BWD_CUTS lists the first block of every range but the last one's: "3" (the
# default), "7", "11,7", "" (one bucket); scripts/sweep_bwd_cuts.sh times them.
BWD_SEGMENTS = _segments(tuning.BWD_CUTS)


def _store_targets(owner, grams):
    """Style targets live in buffers allocated ONCE per executor: a captured step has their
    addresses baked in, so a later style image must land in the same memory to be seen by
    replayed graphs."""
    if owner.style_targets is None:
        owner.style_targets = [g.clone() for g in grams]
    else:
        for t, g in zip(owner.style_targets, grams):
            assert t.shape == g.shape
            t.copy_(g)


class GradBuckets:
    """Bucketed sum-all-reduce of a flat gradient buffer.

    Buckets are contiguous slices, reduced in the order the backward pass
    finishes them.  Works on any torch.distributed backend (RCCL on GPUs; gloo
    in the CPU tests)."""

    def __init__(self, flat_grad, ranges, group=None):
        self.flat, self.ranges, self.group = flat_grad, list(ranges), group
        covered = sorted(self.ranges)
        assert covered[0][0] == 0 and covered[-1][1] == flat_grad.numel()
        for (a0, a1), (b0, b1) in zip(covered, covered[1:]):
            assert a1 == b0, 'gradient buckets must tile the flat buffer'
        self._pending = {}
        self.issue_seconds, self.issued = 0.0, 0
        self.replay_seconds, self.replays, self.steps = 0.0, 0, 0   # host time inside graph.replay() (filled by the trainer)

    def reduce_bucket(self, i):
        import time
        import torch.distributed as dist
        s, e = self.ranges[i]
        if self.flat.is_cuda and dist.get_backend(self.group) == 'gloo':
            # gloo stages device tensors through the host from a thread of its own; issued behind a
            # HIP-graph launch that is still in flight, that copy was observed never to complete.
            # RCCL reductions are stream-ordered device work and need no such wait.
            torch.cuda.current_stream().synchronize()
        t0 = time.perf_counter()
        work = dist.all_reduce(self.flat[s:e], op=dist.ReduceOp.SUM, group=self.group, async_op=True)
        self.issue_seconds += time.perf_counter() - t0
        self.issued += 1
        self._pending[i] = work

    def wait_bucket(self, i):
        """Orders the current stream behind bucket i's reduction (RCCL: a stream wait, the host does not block)."""
        w = self._pending.pop(i, None)
        if w is not None:
            w.wait()

    def wait(self):
        for i in sorted(self._pending):
            self._pending.pop(i).wait()

    def report(self):
        """Bucket sizes and the host-side cost of issuing one collective (what sits on the step's critical
        path between two graph replays)."""
        mb = [round((e - s) * 4 / 1e6, 3) for s, e in self.ranges]
        out = {'bucket_mb': mb, 'exposed_mb': mb[-1], 'overlapped_mb': round(sum(mb[:-1]), 3),
               'collectives_issued': self.issued,
               'host_issue_us_per_collective': round(self.issue_seconds / max(1, self.issued) * 1e6, 1)}
        if self.replays:
            # what the HOST spends per step between the device's segments: if this approaches the step time, the
            # host (not the GPU or the links) paces a data-parallel step
            out['graph_segments_per_step'] = self.replays // max(1, self.steps)
            out['host_replay_us_per_segment'] = round(self.replay_seconds / self.replays * 1e6, 1)
            out['host_us_per_step'] = round((self.replay_seconds + self.issue_seconds) / max(1, self.steps) * 1e6, 1)
        return out


class StyleTrainer:
    def __init__(self, batch, height, width, device, vgg_weights, vgg_mean, style_weight, content_weight, tv_weight,
                 dtype=torch.float32, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, params=None, seed=1,
                 world_size=1, group=None, use_graph=True, max_grad_norm=None):
        """max_grad_norm: clip the gradients of all 48 variables (averaged over the ranks) to this global norm before the
        update, as tf.clip_by_global_norm does; grad_norm then holds the norm before clipping.  None: no clipping, as in
        the reference.  (The clipped update has its rates in double: a norm that is never reached gives the unclipped run to
        1.3e-5 of a step, not to the bit.)"""
        self.n, self.h, self.w, self.device, self.dtype = batch, height, width, device, dtype
        self.sw, self.cw, self.tvw = style_weight, content_weight, tv_weight
        self.lr, self.b1, self.b2, self.eps = lr, beta1, beta2, eps
        self.world, self.group, self.use_graph = world_size, group, use_graph
        self.vgg = VggFeatures(vgg_weights, vgg_mean, device, dtype)
        # ONE VGG pass per step over [content pictures | stylized pictures]: the frozen weights are fetched once,
        # half the launches, and the deep layers (16 x 16 maps at 256 x 256) get twice the blocks.  The content
        # half only passes forward: its conv5_2 output is the content target of the stylized half.
        self.fused_vgg = tuning.FUSED_VGG
        if self.fused_vgg:
            self.vgg_in = torch.empty((2 * batch, height, width, 3), dtype=torch.float32, device=device)
            self.batch_in = self.vgg_in[:batch]
            self.net = StylizerNet(batch, height, width, device, dtype, params=params, seed=seed, training=True,
                                   out_f32=self.vgg_in[batch:])
            self.rep_content = None
            self.rep_loss = self.vgg.replica(2 * batch, height, width, keep_for_backward=True, prefix=batch)
        else:
            self.net = StylizerNet(batch, height, width, device, dtype, params=params, seed=seed, training=True)
            self.rep_content = self.vgg.replica(batch, height, width, keep_for_backward=False)
            self.rep_loss = self.vgg.replica(batch, height, width, keep_for_backward=True)
            self.batch_in = torch.empty((batch, height, width, 3), dtype=torch.float32, device=device)
        self.losses = torch.zeros(4, dtype=torch.float32, device=device)  # total, style, content, tv
        self.loss_slots = ops.loss_slots(self.rep_loss.LOSS_SLOTS, device)   # per-block partial sums of the terms
        self.m = torch.zeros_like(self.net.flat)
        self.v = torch.zeros_like(self.net.flat)
        self.step_dev = torch.zeros(1, dtype=torch.int32, device=device)
        self.style_targets = None
        self.max_grad_norm = max_grad_norm
        self.grad_list = self.grad_norm = None
        if max_grad_norm is not None:
            if not 0 < max_grad_norm < float('inf'):
                raise ValueError('max_grad_norm must be finite and > 0, got %r' % (max_grad_norm,))
            self.grad_list = ops.GradList([self.net.flat_grad])
            self.grad_norm = torch.zeros(1, dtype=torch.float32, device=device)
        self.buckets = None
        if world_size > 1:
            self.buckets = GradBuckets(self.net.flat_grad, [self.net.param_range(hi, lo) for hi, lo in BWD_SEGMENTS],
                                       group)
        self._graphs = None
        # Nothing of a step is accumulated with atomics, so nothing has to be cleared: every gradient, Gram matrix
        # and loss term is written by the kernel (or the fixed-order fold) that owns it.  The step begins by
        # advancing the Adam step counter.
        self._zero = ops.ZeroList([], step_dev=self.step_dev)
        # the content targets only meet the rest of the step at the content loss
        self._content_stream = (torch.cuda.Stream(device=device)
                                if device.type == 'cuda' and 'c' not in _SERIAL and not self.fused_vgg else None)

    # ------------------------------------------------------------- targets
    def set_style_image(self, style_f32):
        """Gram targets of a style image of any size [1,H,W,3] (full_graph_stylizer_network.py:185)."""
        _, h, w, _ = style_f32.shape
        rep = self.vgg.replica(1, h, w, keep_for_backward=False)
        grams, _ = rep.forward(style_f32.to(self.device, torch.float32).contiguous())
        _store_targets(self, grams)
        torch.cuda.synchronize()
        return self.style_targets

    # --------------------------------------------------------------- pieces
    def _front(self):
        self._zero.run()
        cs = self._content_stream
        if self.fused_vgg:
            self.net.forward(self.batch_in)          # the stylized pictures land behind the content pictures
            d_out = self.rep_loss.loss_and_grad(self.vgg_in, self.style_targets, None, self.sw, self.cw, self.tvw,
                                                self.loss_slots)
            return self._sum_losses(d_out)
        if cs is None:
            self.rep_content.forward(self.batch_in, want_grams=False)
            out = self.net.forward(self.batch_in)
        else:
            # The content-target pass goes first, on its own stream, and the stylizer forward follows on the main
            # one (issuing the stylizer first, or interleaving the two passes layer by layer, measured 8 % slower:
            # the content pass then shares a hardware queue with the Gram jobs and runs behind them).
            cs.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(cs):
                self.rep_content.forward(self.batch_in, want_grams=False)
            out = self.net.forward(self.batch_in)
        d_out = self.rep_loss.loss_and_grad(out, self.style_targets, self.rep_content.content,
                                            self.sw, self.cw, self.tvw, self.loss_slots, content_stream=cs)
        return self._sum_losses(d_out)

    def _sum_losses(self, d_out):
        # every loss kernel has been issued and joined: one launch turns their partial sums into the three terms.
        # Only the host reads them: the launch goes to the stream of the weight-gradient jobs (joined by the
        # backward pass that follows), off the data-gradient chain.
        side = self.net._side
        if side is not None:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                ops.loss_slots_sum(self.loss_slots, self.rep_loss.LOSS_TERMS, self.losses)
        else:
            ops.loss_slots_sum(self.loss_slots, self.rep_loss.LOSS_TERMS, self.losses)
        return d_out

    def _adam(self, lo=0, hi=None, advance=True):
        """TF1 Adam on flat[lo:hi]; the step counter was advanced by the launch that cleared the accumulators.
        advance: the first call of a step; with clipping it needs every gradient of the step."""
        sl = slice(lo, hi)
        clip = {}
        if self.grad_list is not None:
            if advance:
                self.grad_list.sum_squares()
            clip = dict(clip=self.grad_list, max_norm=self.max_grad_norm, norm=self.grad_norm)
        ops.adam_tf1(self.net.flat[sl], self.net.flat_grad[sl], self.m[sl], self.v[sl], self.lr, self.b1, self.b2,
                     self.eps, grad_scale=1.0 / self.world, step_dev=self.step_dev, advance=False, **clip)

    def _update(self):
        self._adam()
        self.net.repack()

    def _segments(self):
        """The step as a list of callables.  Data parallel: bucket i is ready after backward range i; the
        update is one Adam launch per bucket (each waits for its own reduction only) and the re-pack."""
        segs = []
        for si, (hi, lo) in enumerate(BWD_SEGMENTS):
            if si == 0:
                segs.append(lambda hi=hi, lo=lo: self.net.backward(self._front(), hi, lo))
            else:
                segs.append(lambda hi=hi, lo=lo: self.net.backward(None, hi, lo))
        if self.buckets is None:
            segs.append(self._update)
            return segs
        last = len(self.buckets.ranges) - 1
        for bi, (s, e) in enumerate(self.buckets.ranges):
            def upd(bi=bi, s=s, e=e):
                self._adam(s, e, advance=(bi == 0))
                if bi == last:
                    self.net.repack()
            segs.append(upd)
        return segs

    def _between(self, i):
        """Collective traffic around segment i of a data-parallel step (i counts _segments() entries)."""
        nb = len(BWD_SEGMENTS)
        if i < nb:
            self.buckets.reduce_bucket(i)          # gradients of range i are complete: start reducing them

    def _before(self, i):
        nb = len(BWD_SEGMENTS)
        if i == nb and self.grad_list is not None:
            self.buckets.wait()                    # the norm needs every bucket
        elif i >= nb:
            self.buckets.wait_bucket(i - nb)       # Adam of bucket i - nb needs that bucket only

    def _run_eager(self):
        segs = self._segments()
        for i, seg in enumerate(segs):
            if self.buckets is not None:
                self._before(i)
            seg()
            if self.buckets is not None:
                self._between(i)

    def _capture(self):
        # warm-up on a side stream (graph capture needs every lazy initialisation done)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self._run_eager()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        if self.buckets is not None:
            # no collective may be in flight on any rank when capture begins
            import torch.distributed as dist
            self.buckets.wait()
            torch.cuda.synchronize()
            dist.barrier(group=self.group)
            torch.cuda.synchronize()
        segs = self._segments()
        if self.buckets is None:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                for seg in segs:
                    seg()
            self._graphs = [g]
        else:
            self._graphs = []
            pool = None
            for seg in segs:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, pool=pool):
                    seg()
                pool = g.pool()
                self._graphs.append(g)

    def comm_report(self):
        return None if self.buckets is None else self.buckets.report()

    # ----------------------------------------------------------------- step
    def step(self, batch_f32=None):
        """One optimisation step on `batch_f32` (fp32 [n,h,w,3] in [0,1]); None re-uses the staged batch."""
        assert self.style_targets is not None, 'call set_style_image first'
        if batch_f32 is not None:
            self.batch_in.copy_(batch_f32, non_blocking=True)
        if not self.use_graph:
            self._run_eager()
            return
        if self._graphs is None:
            state = (self.net.flat.clone(), self.m.clone(), self.v.clone(), self.step_dev.clone())
            self._capture()
            # the warm-up pass updated the weights once: restore so that capture is not a step
            self.net.flat.copy_(state[0]); self.m.copy_(state[1]); self.v.copy_(state[2]); self.step_dev.copy_(state[3])
            self.net.repack()
        if self.buckets is None:
            self._graphs[0].replay()
        else:
            import time
            for i, g in enumerate(self._graphs):
                self._before(i)
                t0 = time.perf_counter()
                g.replay()
                self.buckets.replay_seconds += time.perf_counter() - t0
                self.buckets.replays += 1
                self._between(i)
            self.buckets.steps += 1

    def read_losses(self):
        """[total, style, content, tv] of the last step (synchronises)."""
        l = self.losses.cpu().numpy().astype(np.float64)
        l[0] = l[1] + l[2] + l[3]
        return l

    def stylize(self, x_f32):
        """Forward of the current weights on a batch of the training shape."""
        return self.net.forward(x_f32.to(self.device, torch.float32).contiguous()).clone()


class GatysOptimizer:
    """Adam(0.02, beta1 .99, eps 1e-1) on the image itself (full_graph_stylizer_network.py:278-279)."""

    def __init__(self, content_f32, device, vgg_weights, vgg_mean, style_weight, content_weight, tv_weight,
                 dtype=torch.float32, lr=0.02, beta1=0.99, beta2=0.999, eps=1e-1, use_graph=True):
        _, h, w, _ = content_f32.shape
        self.device, self.dtype = device, dtype
        self.sw, self.cw, self.tvw = style_weight, content_weight, tv_weight
        self.lr, self.b1, self.b2, self.eps, self.use_graph = lr, beta1, beta2, eps, use_graph
        self.vgg = VggFeatures(vgg_weights, vgg_mean, device, dtype)
        self.rep = self.vgg.replica(1, h, w, keep_for_backward=True)
        self.image = content_f32.to(device, torch.float32).contiguous().clone()   # tf.Variable(content_image), :257
        content_rep = self.vgg.replica(1, h, w, keep_for_backward=False)
        _, c = content_rep.forward(self.image)
        self.content_target = c.clone()
        self.style_targets = None
        self.grad32 = torch.empty_like(self.image)
        self.m = torch.zeros_like(self.image)
        self.v = torch.zeros_like(self.image)
        self.step_dev = torch.zeros(1, dtype=torch.int32, device=device)
        self.losses = torch.zeros(4, dtype=torch.float32, device=device)
        self.loss_slots = ops.loss_slots(self.rep.LOSS_SLOTS, device)
        self._zero = ops.ZeroList([], step_dev=self.step_dev)   # nothing to clear (no atomics): advances the step counter
        self._graph = None

    def set_style_image(self, style_f32):
        _, h, w, _ = style_f32.shape
        rep = self.vgg.replica(1, h, w, keep_for_backward=False)
        grams, _ = rep.forward(style_f32.to(self.device, torch.float32).contiguous())
        _store_targets(self, grams)
        torch.cuda.synchronize()

    def _run(self):
        self._zero.run()
        d = self.rep.loss_and_grad(self.image, self.style_targets, self.content_target, self.sw, self.cw, self.tvw,
                                   self.loss_slots)
        ops.loss_slots_sum(self.loss_slots, self.rep.LOSS_TERMS, self.losses)
        if self.dtype == torch.float32:
            g = d
        else:
            g = ops.cast(d, torch.float32, out=self.grad32)
        ops.adam_tf1(self.image, g, self.m, self.v, self.lr, self.b1, self.b2, self.eps, step_dev=self.step_dev,
                     advance=False)
        # the reference's clip (:328-329) only builds an un-run assign op: the image is NOT clipped

    def step(self):
        assert self.style_targets is not None
        if not self.use_graph:
            self._run()
            return
        if self._graph is None:
            state = (self.image.clone(), self.m.clone(), self.v.clone(), self.step_dev.clone())
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                self._run()
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            self._graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self._graph):
                self._run()
            self.image.copy_(state[0]); self.m.copy_(state[1]); self.v.copy_(state[2]); self.step_dev.copy_(state[3])
        self._graph.replay()

    def read_losses(self):
        l = self.losses.cpu().numpy().astype(np.float64)
        l[0] = l[1] + l[2] + l[3]
        return l
