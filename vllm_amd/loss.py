"""Host-side mirror of the reference's contrastive loss, same names and argument meaning.

    Temperature               model/modeling_abc.py:36-43
    compute_contrastive_loss  model/abc_util.py:43-56
    compute_gathered_loss     model/abc_util.py:5-31
    compute_distillation_loss (no counterpart in the reference: a teacher's top list instead of the one positive)

The logits / logsumexp / label-smoothed cross entropy / argmax and their backward run in
libabcsearch.so (abc_infonce_fwd / abc_infonce_bwd, exact fp32 on the matrix cores); the candidate
all-gather is torch.distributed (RCCL over xGMI on ROCm).  No CPU path.
"""
from __future__ import annotations

import torch
import torch.distributed as dist
from torch.autograd.function import once_differentiable

from . import _lib
from .kernels import _launch, _on, _stream


class Temperature(torch.nn.Module):
    """Scalar learned temperature, init 0.07; forward(x) = x / temp (model/modeling_abc.py:36-43)."""

    def __init__(self, init: float = 0.07):
        super().__init__()
        self.temp = torch.nn.Parameter(torch.tensor(init, requires_grad=True, dtype=torch.float32))

    def forward(self, x):
        return x / (self.temp.float())


# Workspaces (logits for the backward, split-K slabs, statistics, counters: ~9 MB at B=128 x C=1024) are leased from a
# small pool per (device, stream, size) instead of allocated per call: a lease returns to the pool when the autograd
# node that holds it dies (after backward, or when the loss is dropped), so two losses alive at once get two buffers and
# a training loop reuses one.  Work on one stream runs in order, which is what makes reuse within a key safe.
_ws_pool: dict = {}
_WS_POOL_MAX = 4


class _Lease:
    __slots__ = ("key", "buf")

    def __init__(self, nbytes: int, device: torch.device, stream: int):
        self.key = (device.index, stream, nbytes)
        free = _ws_pool.get(self.key)
        self.buf = free.pop() if free else torch.empty(nbytes, dtype=torch.uint8, device=device)

    def __del__(self):
        try:
            free = _ws_pool.setdefault(self.key, [])
            if len(free) < _WS_POOL_MAX:
                free.append(self.buf)
        except Exception:                                    # interpreter shutdown
            pass


def release_workspaces() -> None:
    """Drop the pooled InfoNCE workspaces (buffers held by live autograd graphs stay with them)."""
    _ws_pool.clear()


def _f32c(x: torch.Tensor) -> torch.Tensor:
    return x if (x.dtype is torch.float32 and x.is_contiguous()) else x.float().contiguous()


class _InfoNCE(torch.autograd.Function):
    """loss, accuracy = InfoNCE(q, p, temp).  `p` [C, d] is the full candidate matrix and carries NO gradient
    itself; `p_local` is the tensor whose rows are p[:n] and that receives their gradient (p itself when every row is
    local, the rank's own block under the gather: remote blocks are constants, model/abc_util.py:19-21)."""

    @staticmethod
    def forward(ctx, q, p, p_local, temp, eps: float):
        if not (q.is_cuda and p.is_cuda):
            raise _lib.AbcError("InfoNCE kernels run on the GPU only (no CPU fallback)")
        lib = _lib.load()
        q, p = _f32c(q), _f32c(p)
        B, d = q.shape
        C = p.shape[0]
        need = lib.abc_infonce_workspace_bytes(B, C, d)
        if need == 0:
            raise _lib.AbcError(f"InfoNCE: unsupported shape B={B} C={C} d={d} (need B <= C, d % 8 == 0)")
        dev = q.device
        # the device scalar the kernels read: the parameter's own storage when it is an fp32 tensor on this device
        t = temp if (temp.dtype is torch.float32 and temp.device == dev and temp.numel() == 1) else \
            temp.detach().to(device=dev, dtype=torch.float32).reshape(1)
        # loss and accuracy are tensors of their own (a caller may change them in place, as it may the reference's);
        # logsumexp and argmax stay internal: [lse[B] f32, argmax[B] i32 bits]
        loss = torch.empty((), dtype=torch.float32, device=dev)
        acc = torch.empty((), dtype=torch.float32, device=dev)
        aux = torch.empty(2 * B, dtype=torch.float32, device=dev)
        with _on(q):
            st = _stream(q)
            lease = _Lease(need, dev, st)
            ws = lease.buf
            base = aux.data_ptr()
            rc = lib.abc_infonce_fwd(q.data_ptr(), p.data_ptr(), t.data_ptr(), eps, B, C, d, loss.data_ptr(), base,
                                     base + 4 * B, acc.data_ptr(), ws.data_ptr(), ws.numel(), st)
        _lib.check(rc, "abc_infonce_fwd")
        ctx.save_for_backward(q, p, t)
        ctx.keep = (aux, lease)                                              # lse lives in `aux`, the logits in the lease
        ctx.meta = (eps, B, C, d, int(p_local.shape[0]), temp.dtype)
        ctx.mark_non_differentiable(acc)
        return loss, acc

    @staticmethod
    def backward(ctx, grad_loss, _grad_acc):
        q, p, t = ctx.saved_tensors
        aux, lease = ctx.keep
        eps, B, C, d, local_rows, tdtype = ctx.meta
        lib = _lib.load()
        need_q, need_p, need_t = ctx.needs_input_grad[0], ctx.needs_input_grad[2], ctx.needs_input_grad[3]
        go = _f32c(grad_loss)
        dq = torch.empty_like(q) if need_q else None
        dp = torch.empty((local_rows, d), dtype=torch.float32, device=q.device) if need_p else None
        dt = torch.empty((), dtype=torch.float32, device=q.device) if need_t else None
        ws = lease.buf
        with _on(q):
            rc = lib.abc_infonce_bwd(q.data_ptr(), p.data_ptr(), aux.data_ptr(), t.data_ptr(), eps, go.data_ptr(), B, C, d,
                                     local_rows if need_p else 0, None if dq is None else dq.data_ptr(),
                                     None if dp is None else dp.data_ptr(), None if dt is None else dt.data_ptr(),
                                     ws.data_ptr(), ws.numel(), _stream(q))
        _lib.check(rc, "abc_infonce_bwd")
        if dt is not None and tdtype is not torch.float32:
            dt = dt.to(tdtype)
        return dq, None, dp, dt, None


def _temp_param(temperature, device: torch.device) -> torch.Tensor:
    t = getattr(temperature, "temp", temperature)
    if not torch.is_tensor(t):
        t = torch.full((), float(t), dtype=torch.float32, device=device)    # (a fill: a copy from the host could not be captured)
    return t


def _loss_and_acc(q_embeds, p_embeds, temperature, label_smoothing, local_rows, p_local=None):
    """p_embeds: the full candidate matrix; its first `local_rows` rows are `p_local` (default: p_embeds[:local_rows]),
    the only rows that receive a gradient."""
    temp = _temp_param(temperature, q_embeds.device)
    if temp.device != q_embeds.device:
        temp = temp.to(q_embeds.device)
    if p_local is None:
        p_local = p_embeds if local_rows == p_embeds.shape[0] else p_embeds[:local_rows]
    held = None
    if torch.is_grad_enabled() and q_embeds.is_cuda and torch.cuda.is_current_stream_capturing():
        held = _captured_leaves((q_embeds, p_embeds, temp), refuse=False)
    loss, accuracy = _InfoNCE.apply(q_embeds, p_embeds.detach(), p_local, temp, float(label_smoothing))
    del held
    return loss, accuracy


def compute_contrastive_loss(q_embeds, p_embeds, temperature, label_smoothing=0.0):
    """score = temperature(q @ p.T); cross entropy against arange(bs) with label smoothing; argmax
    accuracy.  Same call and return as model/abc_util.py:43-56; differentiable w.r.t. q_embeds,
    p_embeds and temperature.temp."""
    return _loss_and_acc(q_embeds, p_embeds, temperature, label_smoothing, p_embeds.size(0))


def _captured_leaves(leaves, refuse: bool) -> list:
    """Under graph capture: mark the gradient nodes of these leaves as the capturing stream's, and (refuse) raise where a leaf's node was
    there before.  A leaf has one gradient node while any autograd graph of it lives, bound to the stream that graph was built on; a
    captured backward that reaches a node of an eager graph makes the eager stream wait inside the capture, which ends the process when the
    capture ends.  Whether a node was there before: one that only this function holds is gone when it lets go, with its mark.
    Only the tensors handed over are looked at.  Of leaves further up (an encoder's parameters) a node that the capture itself has made and one
    from before look alike; there it is for the caller, as for every captured backward, to let go of earlier graphs.
    Returns the marked nodes: hold them until the call's own graph does."""
    held = []
    for x in leaves:
        if not (torch.is_tensor(x) and x.requires_grad and x.is_leaf):
            continue
        stream = torch.cuda.current_stream(x.device).cuda_stream
        node = torch.autograd.graph.get_gradient_edge(x).node
        mine = node.metadata.get("abc_capture") == stream
        node.metadata["abc_probe"] = True
        del node
        node = torch.autograd.graph.get_gradient_edge(x).node
        if node.metadata.pop("abc_probe", False) and not mine:
            if refuse:
                raise _lib.AbcError(
                    "capture: an autograd graph of a leaf (queries, candidates or temperature) is alive from before; its gradient belongs to "
                    "another stream and capturing this backward would end the process.  Drop earlier losses and outputs of these leaves "
                    "before the capture (inside one capture: call this loss before other uses of them)")
            continue
        node.metadata["abc_capture"] = stream
        held.append(node)
    return held


class _Distill(torch.autograd.Function):
    """loss, agreement = distillation from a teacher's list.  `memory` and the list are constants."""

    @staticmethod
    def forward(ctx, q, p, temp, memory, index, score, teacher_temp: float):
        lib = _lib.load()
        B, d = q.shape
        C, k = p.shape[0], index.shape[1]
        M, mem = (0, None) if memory is None else (memory.shape[0], memory.data_ptr())
        dtype = _lib.DT_BF16 if q.dtype is torch.bfloat16 else _lib.DT_F32
        need = lib.abc_distill_workspace_bytes(dtype, B, C, M, d, k)
        if need == 0:
            _lib.check(-1, "abc_distill_workspace_bytes")
        dev = q.device
        t = temp if temp.dtype is torch.float32 else temp.detach().to(torch.float32)
        loss, agree = torch.empty((), dtype=torch.float32, device=dev), torch.empty((), dtype=torch.float32, device=dev)
        # scratch of its own (the caching allocator's, in stream order): two losses alive, or two captured graphs, share nothing
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _launch(lib.abc_distill_fwd, "abc_distill_fwd", dev, dtype, q.data_ptr(), p.data_ptr(), mem, t.data_ptr(), index.data_ptr(),
                score.data_ptr(), teacher_temp, B, C, M, d, k, loss.data_ptr(), agree.data_ptr(), ws.data_ptr(), need)
        if any(ctx.needs_input_grad):
            ctx.save_for_backward(q, p, t, memory, ws)                      # (freed with the graph, not with the last loss that is kept)
            ctx.meta = (dtype, B, C, M, d, k, need, temp.dtype, temp.shape)
        ctx.mark_non_differentiable(agree)
        return loss, agree

    @staticmethod
    def backward(ctx, grad_loss, _grad_agree):
        # once_differentiable costs some 10 us of bookkeeping; only a backward that is itself recorded needs it
        return _distill_bwd_once(ctx, grad_loss, _grad_agree) if torch.is_grad_enabled() else _distill_bwd(ctx, grad_loss, _grad_agree)


def _distill_bwd(ctx, grad_loss, _grad_agree):
    q, p, t, memory, fwd_ws = ctx.saved_tensors
    dtype, B, C, M, d, k, fwd_need, tdtype, tshape = ctx.meta
    lib = _lib.load()
    need_q, need_p, need_t = ctx.needs_input_grad[:3]
    go = _f32c(grad_loss)
    dev = q.device
    dq = torch.empty_like(q) if need_q else None
    dp = torch.empty_like(p) if need_p else None
    dt = torch.empty(tshape, dtype=torch.float32, device=dev) if need_t else None
    need = lib.abc_distill_bwd_workspace_bytes(dtype, B, C, M, d, k)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _launch(lib.abc_distill_bwd, "abc_distill_bwd", dev, dtype, q.data_ptr(), p.data_ptr(), None if memory is None else memory.data_ptr(),
            t.data_ptr(), go.data_ptr(), B, C, M, d, k, None if dq is None else dq.data_ptr(),
            None if dp is None else dp.data_ptr(), None if dt is None else dt.data_ptr(), fwd_ws.data_ptr(), fwd_need, ws.data_ptr(), need)
    if dt is not None and tdtype is not torch.float32:
        dt = dt.to(tdtype)
    return dq, dp, dt, None, None, None, None


_distill_bwd_once = once_differentiable(_distill_bwd)


def compute_distillation_loss(q_embeds, p_embeds, temperature, teacher_index, teacher_scores, teacher_temperature=1.0, memory=None):
    """Draw the softmax of each query over its candidates towards a teacher's top list: the mean over the queries of
    KL(teacher's list || softmax(temperature(q @ candidates.T))).

    The candidates are the rows of p_embeds [C, D] and after them the rows of `memory` [M, D], constants that receive no
    gradient (read back from a search.EmbeddingStore, or the other ranks' rows c_global[n:] of gathered_candidates).
    teacher_index [B, k] numbers them (0 .. C + M - 1), teacher_scores [B, k] are the teacher's scores of them, as topk returns them:
    an index below 0 or a score of -inf is no entry.  The teacher's shares are softmax(teacher_scores / teacher_temperature) over a row's
    entries, which carry no gradient.  A row's value is sum_i share_i (log share_i - log softmax_column(i)) over the entries: the divergence
    where no column comes twice, as in topk's lists.  A column may come twice: the gradients are those of its added shares, and the value
    lies below the divergence of the added shares by the entropy within the column, a constant (so that it may be negative).  A row
    without an entry counts nowhere and gets a gradient of zero; an index past the candidates makes the loss NaN.

    q_embeds [B, D], p_embeds and memory all bf16 run on bf16 products with fp32 sums and return bf16 gradients; any other mix is
    computed in fp32, on the 16-bit parts of its values: an infinity in an embedding makes its logits NaN there (in bf16 +-inf where the
    products are).  A width that is no multiple of 8 costs padded copies of queries, candidates and memory in every call.  Returns (loss, agreement): agreement is the share of the rows with an entry whose best candidate is the
    list's best entry.  Differentiable (once) w.r.t. q_embeds, p_embeds and temperature.temp.  

    Under graph capture take gradients with torch.autograd.grad and have the temperature on the embeddings' device.  No autograd graph from
    before the capture may hold a leaf that the backward reaches (torch would end the process): of q_embeds, p_embeds and the temperature
    that are leaves themselves this is checked and refused; of an encoder's parameters behind them, or of embeddings computed before the
    capture, it is not.  No counterpart in the reference."""
    temp = _temp_param(temperature, q_embeds.device)
    dev, width = q_embeds.device, q_embeds.shape[-1]
    embeds = (q_embeds, p_embeds) if memory is None else (q_embeds, p_embeds, memory)
    same = True                                                             # all bf16 or all fp32, as they come
    for t in embeds:
        if t.dim() != 2 or t.shape[1] != width or t.device != dev or not t.is_floating_point():
            raise _lib.AbcError(f"distillation: expected floating-point rows of one width on one device, got "
                                f"{[(t.dtype, tuple(t.shape), str(t.device)) for t in embeds]}")
        same = same and t.dtype is q_embeds.dtype
    if not (q_embeds.is_cuda and teacher_index.device == dev and teacher_scores.device == dev):
        raise _lib.AbcError("distillation runs on the GPU only (no CPU fallback), with the teacher's list on the embeddings' device")
    if teacher_index.dim() != 2 or teacher_index.shape != teacher_scores.shape or teacher_index.shape[0] != q_embeds.shape[0] or \
            teacher_index.dtype not in (torch.int64, torch.int32) or not teacher_scores.is_floating_point():
        raise _lib.AbcError(f"distillation: expected teacher_index (int64 / int32) and teacher_scores (floating point) "
                            f"[{q_embeds.shape[0]}, k], got {teacher_index.dtype} {tuple(teacher_index.shape)} and "
                            f"{teacher_scores.dtype} {tuple(teacher_scores.shape)}")
    if temp.numel() != 1:
        raise _lib.AbcError("distillation: the temperature is one number")
    teacher_temperature = float(teacher_temperature)
    if not teacher_temperature > 0.0:
        raise _lib.AbcError("distillation: teacher_temperature must be positive")
    held = None
    if torch.cuda.is_current_stream_capturing():
        if temp.device != dev:
            raise _lib.AbcError(f"capture: the temperature is on {temp.device}, and a copy of it to {dev} cannot be captured; move it there first")
        if torch.is_grad_enabled():
            held = _captured_leaves((q_embeds, p_embeds, temp), refuse=True)
    if temp.device != dev:
        temp = temp.to(dev)
    if not (same and (q_embeds.dtype is torch.bfloat16 or q_embeds.dtype is torch.float32)):
        q_embeds, p_embeds = q_embeds.float(), p_embeds.float()
        memory = None if memory is None else memory.float()
    if width % 8:                                                           # zero columns change no product
        q_embeds, p_embeds = (torch.nn.functional.pad(t, (0, -width % 8)) for t in (q_embeds, p_embeds))
        memory = None if memory is None else torch.nn.functional.pad(memory, (0, -width % 8))
    if memory is not None:
        memory = None if memory.shape[0] == 0 else _aligned(memory.detach())
    if teacher_index.dtype is not torch.int64:
        teacher_index = teacher_index.to(torch.int64)
    out = _Distill.apply(_aligned(q_embeds), _aligned(p_embeds), temp, memory, teacher_index.contiguous(), _f32c(teacher_scores.detach()),
                         teacher_temperature)
    del held
    return out


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """x contiguous, on a 16-byte boundary (a slice of a larger tensor may start anywhere)."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _all_gather_rows(x: torch.Tensor) -> torch.Tensor:
    """[n, ...] -> [world * n, ...], ONE collective.  RCCL (backend "nccl") takes the device tensor as it is; under
    a gloo group (CPU-side tests, one-GPU rehearsals) device tensors cross in host memory, because gloo's
    collectives on device tensors do not complete on this stack (vllm_amd/parallel.py)."""
    world = dist.get_world_size()
    x = x.detach().contiguous()
    staged = x.is_cuda and dist.get_backend() == "gloo"
    src = x.cpu() if staged else x
    out = torch.empty((world * src.shape[0],) + tuple(src.shape[1:]), dtype=src.dtype, device=src.device)
    dist.all_gather_into_tensor(out, src)
    return out.to(x.device) if staged else out


def gathered_candidates(c_emb: torch.Tensor):
    """all_gather of the candidate block, local block swapped into slot 0 (model/abc_util.py:15-27).
    Returns (c_global [W*n, D] -- rows [0, n) are the local block -- and n).  c_global carries no autograd history:
    the loss function takes c_emb itself as the tensor rows [0, n) send their gradient to."""
    n = c_emb.size(0)
    if not dist.is_initialized() or dist.get_world_size() == 1:
        return c_emb, n
    world, rank = dist.get_world_size(), dist.get_rank()
    gathered = _all_gather_rows(c_emb)                                       # one collective, no gradient
    order = _slot_order(world, rank)
    if rank == 0:
        return gathered, n                                                   # already [c_0, c_1, ...]: slot 0 is the own block
    gathered = gathered.view((world,) + tuple(c_emb.shape))
    gathered[[0, rank]] = gathered[[rank, 0]]                                # swap slots 0 and rank in place (2 blocks move)
    assert order[0] == rank
    return gathered.view((world * n,) + tuple(c_emb.shape[1:])), n


def _slot_order(world: int, rank: int):
    """Which rank's block sits in each slot of c_global on `rank`: own block first, rank 0's block in
    slot `rank` (model/abc_util.py:24-27)."""
    order = list(range(world))
    order[0], order[rank] = order[rank], order[0]
    return order


class _AllGatherWithGrad(torch.autograd.Function):
    """all_gather whose backward is a reduce-scatter(SUM): every rank's loss sends a gradient to every
    candidate block.  Opt-in; the reference's gather is gradient-free
    (model/abc_util.py:19-21), UniIR's is this one (torch.distributed.nn.all_gather, clip_sf.py:103)."""

    @staticmethod
    def forward(ctx, c_emb):
        world, rank = dist.get_world_size(), dist.get_rank()
        gathered = _all_gather_rows(c_emb).view((world,) + tuple(c_emb.shape))
        ctx.order = _slot_order(world, rank)
        ctx.shape = tuple(c_emb.shape)
        return torch.cat([gathered[r] for r in ctx.order], dim=0)

    @staticmethod
    def backward(ctx, g):
        world, rank = dist.get_world_size(), dist.get_rank()
        gv = g.contiguous().view((world,) + ctx.shape)
        canon = torch.empty_like(gv)                       # slot j holds the gradient for rank order[j]'s block
        for j, r in enumerate(ctx.order):
            canon[r] = gv[j]
        if dist.get_backend() == "nccl":                   # RCCL: one reduce-scatter over xGMI
            out = torch.empty(ctx.shape, dtype=g.dtype, device=g.device)
            dist.reduce_scatter_tensor(out, canon.view((world * ctx.shape[0],) + ctx.shape[1:]), op=dist.ReduceOp.SUM)
            return out
        # gloo (CPU tests, one-GPU rehearsals) has no reduce-scatter; device tensors cross in host memory
        h = canon.cpu() if canon.is_cuda else canon
        dist.all_reduce(h, op=dist.ReduceOp.SUM)
        return h[rank].to(g.device).clone()


def compute_gathered_loss(q_emb, c_emb, temperature, label_smoothing=0.0, differentiable_gather=False):
    """Compute the loss by gathering candidates across GPUs; the first [batch_size] entries of c_emb
    are the positives.  Same call and return as model/abc_util.py:5-31: (loss, accuracy, num_cand);
    queries are not gathered and only the local candidate block receives a gradient.

    differentiable_gather=True (not in the reference, off by default) lets the gradient of every
    rank's loss reach every candidate block: backward adds one reduce-scatter of the [W*n, D] gradient."""
    q_emb = q_emb.float()
    c_emb = c_emb.float()
    if differentiable_gather and dist.is_initialized() and dist.get_world_size() > 1:
        c_all = _AllGatherWithGrad.apply(c_emb)
        loss, acc = _loss_and_acc(q_emb, c_all, temperature, label_smoothing, c_all.size(0))
        return loss, acc, _num_cand(c_all.size(0), loss.device)
    c_global, n_local = gathered_candidates(c_emb)
    # the gathered blocks are constants: only rows [0, n_local) of c_global (= c_emb) get a gradient, and the backward
    # kernel writes exactly those rows
    loss, acc = _loss_and_acc(q_emb, c_global, temperature, label_smoothing, n_local, p_local=c_emb)
    return loss, acc, _num_cand(c_global.size(0), loss.device)


def _num_cand(n: int, device) -> torch.Tensor:
    """torch.tensor([n], device=...) of the reference (abc_util.py:30) without the host-to-device copy: a fill."""
    return torch.full((1,), n, dtype=torch.int64, device=device)
