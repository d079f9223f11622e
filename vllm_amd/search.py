"""Host-side mirror of the reference's search entry points, same names and argument meaning.

    get_topk_candidates   evaluate/eval_mscoco.py:18-50 (copies in eval_flickr30k.py, eval_vg_instruct.py,
                          mmeb_classification.py, mmeb_vqa.py)
    negatives_for_sample  pretrain/create_negative_index.py:45-52
    batch / compute_topk  visualization/neg_mine.py:21-77

The arithmetic (score contraction, top-k, mask, compare-count) runs in libabcsearch.so through
`vllm_amd.kernels`; torch only moves tensors.  There is no CPU path: without a GPU these raise.
"""
from __future__ import annotations

import os
import weakref
from typing import Dict, Iterable, List, Optional, Sequence, Tuple

import torch

from . import kernels
from ._lib import AbcError

_COMPUTE = {"f32": torch.float32, "bf16": torch.bfloat16, "i8": torch.int8}


def _device(device=None) -> torch.device:
    if device is not None:
        return torch.device(device)
    if not torch.cuda.is_available():
        raise AbcError("no ROCm device visible: vllm_amd.search has no CPU fallback")
    return torch.device("cuda", torch.cuda.current_device())


class Embeddings:
    """A matrix of embeddings resident in HBM in the dtype the kernels contract in."""

    def __init__(self, x: torch.Tensor, compute: str = "f32", device=None):
        if compute not in _COMPUTE:
            raise AbcError(f"compute must be one of {sorted(_COMPUTE)}")
        dev = _device(device if device is not None else (x.device if x.is_cuda else None))
        self.compute = compute
        self.scale = None
        x = x.to(dev)
        if compute == "i8":
            if x.dtype == torch.int8:
                raise AbcError("pass fp32 embeddings; quantisation happens here")
            self.data, self.scale = kernels.quantize_i8(x.float())
        elif compute == "bf16":
            self.data = x if x.dtype == torch.bfloat16 else kernels.cast_bf16(x.float())
        else:
            self.data = x.float().contiguous()
        # the kernels take rows of whole 128-byte pieces (64 bf16 / 32 fp32 / 128 int8 elements): any other width (the
        # reference's get_topk_candidates takes any D) is padded with zero columns once, here, which changes no score
        per = 128 // self.data.element_size()
        extra = (-self.data.shape[1]) % per if self.data.dim() == 2 else 0
        if extra:
            self.data = torch.nn.functional.pad(self.data, (0, extra))

    @property
    def shape(self):
        """[rows, columns as resident: D rounded up to whole 128-byte pieces]"""
        return self.data.shape

    def rows(self, lo: int, hi: int) -> "Embeddings":
        out = object.__new__(Embeddings)
        out.compute, out.data = self.compute, self.data[lo:hi]
        out.scale = None if self.scale is None else self.scale[lo:hi]
        return out

    def take(self, index: torch.Tensor) -> "Embeddings":
        out = object.__new__(Embeddings)
        out.compute, out.data = self.compute, self.data[index].contiguous()
        out.scale = None if self.scale is None else self.scale[index].contiguous()
        return out


class EmbeddingStore:
    """Embeddings held in 4 or 8 bits that change while they are in use: rows are quantised as they are written into slots, and
    read back by index -- a corpus that grows, the candidates of earlier training steps kept as negatives.

    form "fp4": 4-bit codes (e2m1) with a bf16 scale for every `group` (32, 64 or 128) values, 0.52 bytes a value at 128; `scores` runs a
    few queries over it.  form "i8": the int8 rows of Embeddings(x, "i8"), one fp32 scale each; `embeddings` hands them to topk.

    Calls on one store run in the order of the stream they are made on; a store used on two streams is the caller's to order, like
    any tensor.  Slots that nothing was written to hold zeros.  No counterpart in the reference (its corpora are saved fp32 tensors)."""

    def __init__(self, capacity: int, dim: int, form: str = "fp4", group: int = 128, device=None):
        if form not in ("fp4", "i8"):
            raise AbcError(f"form must be fp4 or i8, not {form}")
        if form == "fp4" and group not in (32, 64, 128):
            raise AbcError(f"group must be 32, 64 or 128, not {group}")
        if not 0 < int(capacity) < 1 << 31 or not 1 <= int(dim) <= 8192:
            raise AbcError(f"a store of {capacity} rows of {dim} values: 1 to 2^31 - 1 rows of 1 to 8192 values")
        dev = _device(device)
        width = (int(dim) + 127) // 128 * 128
        self.capacity, self.dim, self.form, self._next = int(capacity), int(dim), form, 0
        if form == "fp4":
            self.data = torch.zeros((self.capacity, width // 2), dtype=torch.uint8, device=dev)
            self.scale = torch.zeros((self.capacity, width // group), dtype=torch.bfloat16, device=dev)
        else:
            self.data = torch.zeros((self.capacity, width), dtype=torch.int8, device=dev)
            self.scale = torch.ones((self.capacity,), dtype=torch.float32, device=dev)

    def write(self, x: torch.Tensor, slots: torch.Tensor) -> None:
        """Row i of x [n, dim] (f32 / bf16) replaces what slot slots[i] holds; a slot outside the store drops its row, and of rows
        that name the same slot the last one stays."""
        if slots is None:
            raise AbcError("write needs slots; append takes the next ones")
        self._width(x)
        kernels.store_write(x, slots, self.data, self.scale)

    def append(self, x: torch.Tensor) -> int:
        """Write x into the next slots, past the last one on from slot 0, over the oldest rows; returns the first slot taken.
        The position is the host's: a captured graph would write the same slots at every replay, so capture is refused (use write)."""
        self._width(x)
        n = x.shape[0]
        if n > self.capacity:
            raise AbcError(f"{n} rows do not fit a store of {self.capacity}")
        if torch.cuda.is_current_stream_capturing():
            raise AbcError("append cannot be captured into a graph: its position is kept on the host; use write with slots")
        first = self._next
        kernels.store_write(x, None, self.data, self.scale, first)
        self._next = (first + n) % self.capacity
        return first

    def read(self, index: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float32,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The values of rows `index` (any shape; None: all), [*index.shape, dim] f32 / bf16.  Negative: zeros (the -1 of a top-k
        list); past the store: NaN.  `out`: a tensor to write into."""
        return kernels.store_read(index, self.data, self.scale, self.dim, dtype, out)

    def rows(self, lo: int, hi: int) -> "EmbeddingStore":
        """Slots [lo, hi) as a store of their own, sharing this one's memory."""
        if not 0 <= lo < hi <= self.capacity:
            raise AbcError(f"rows [{lo}, {hi}) of a store of {self.capacity}")
        out = object.__new__(EmbeddingStore)
        out.capacity, out.dim, out.form, out._next = hi - lo, self.dim, self.form, 0
        out.data, out.scale = self.data[lo:hi], self.scale[lo:hi]
        return out

    def scores(self, q: torch.Tensor) -> torch.Tensor:
        """f32 [nq, capacity]: inner products of a few queries q [nq, dim] (f32 / bf16) with every row (fp4 form)."""
        self._width(q)
        return kernels.store_scores(q, self.data, self.scale)

    def embeddings(self) -> Embeddings:
        """The int8 rows as a corpus for topk / mine_negatives, sharing this store's memory (i8 form)."""
        if self.form != "i8":
            raise AbcError("topk contracts int8 rows: the fp4 form is searched by scores")
        emb = object.__new__(Embeddings)
        emb.compute, emb.data, emb.scale = "i8", self.data, self.scale
        return emb

    def _width(self, x: torch.Tensor) -> None:
        if x.dim() != 2 or x.shape[1] != self.dim:
            raise AbcError(f"expected rows of {self.dim} values, got {tuple(x.shape)}")


def topk(q: Embeddings, c: Embeddings, k: int, upper_bound=None, idx_offset: int = 0, rank_ref=None,
         rank_self_offset=None):
    """Exact top-k of q @ c.T (values, indices[, rank counts]) on the GPU."""
    if q.compute != c.compute:
        raise AbcError("query and corpus must use the same compute dtype")
    return kernels.topk(q.data, c.data, k, upper_bound=upper_bound, idx_offset=idx_offset, rank_ref=rank_ref,
                        rank_self_offset=rank_self_offset, q_scale=q.scale, c_scale=c.scale)


def positive_scores(q: Embeddings, c: Embeddings, offset: int = 0) -> torch.Tensor:
    """s_pos[i] = q[i] . c[offset + i]  (create_negative_index.py:48, neg_mine.py:32-35)."""
    n = q.shape[0]
    cc = c.rows(offset, offset + n)
    return kernels.rowdot(q.data, cc.data, q_scale=q.scale, c_scale=cc.scale)


# ----------------------------------------------------------------------------------------------
# a1: evaluate/eval_mscoco.py:18-50
# ----------------------------------------------------------------------------------------------
def get_topk_candidates(queries: Sequence[Tuple[object, torch.Tensor]],
                        candidates: Sequence[Tuple[object, torch.Tensor]], k: int = 3,
                        compute: str = "f32") -> Dict[object, list]:
    """Return {query_id: [top-k candidate ids, best first]} by dot-product similarity.

    Same contract as the reference: `queries`/`candidates` are lists of (id, Tensor[1, D]); the dict is
    keyed by query id, so duplicated ids collapse to the last occurrence.  The score matrix is never
    materialised and nothing but the [Nq, k] index table returns to the host.
    """
    return get_topk_candidates_multi(queries, candidates, (k,), compute=compute)[k]


def _rows(embs, what: str) -> torch.Tensor:
    """The [N, D] matrix of a list of embeddings: [1, D] (or [n, D]) pieces are concatenated (eval_mscoco.py:38-39), [D]
    vectors stacked (the candidate form of mmeb_vqa.py:24).  One list holds one form."""
    dims = {int(e.dim()) for e in embs}
    if dims == {1}:
        return torch.stack(tuple(embs), dim=0)
    if dims == {2}:
        return torch.cat(tuple(embs), dim=0)
    raise AbcError(f"{what} embeddings must all be [D] vectors or all [n, D] matrices, got dims {sorted(dims)}")


def get_topk_candidates_multi(queries, candidates, ks: Iterable[int], compute: str = "f32") -> Dict[int, Dict[object, list]]:
    """One search at max(ks), prefixes reused for the smaller k (the reference recomputes the whole
    matmul for every k in [1, 5, 10], eval_mscoco.py:76-77,87-88)."""
    ks = sorted(set(int(k) for k in ks))
    query_ids, query_embs = zip(*queries)
    candidate_ids, candidate_embs = zip(*candidates)
    dev = _device()
    q = Embeddings(_rows(query_embs, "query"), compute, dev)
    c = Embeddings(_rows(candidate_embs, "candidate"), compute, dev)
    kmax = ks[-1]
    _, idx, _ = topk(q, c, kmax)
    idx = idx.cpu().tolist()
    out = {}
    for k in ks:
        results = {}
        for i, q_id in enumerate(query_ids):
            results[q_id] = [candidate_ids[j] for j in idx[i][:k] if j >= 0]
        out[k] = results
    return out


# ----------------------------------------------------------------------------------------------
# a3: pretrain/create_negative_index.py:45-52
# ----------------------------------------------------------------------------------------------
def mine_negatives(q: Embeddings, c: Embeddings, k: int = 100, ratio: float = 0.95, offset: int = 0,
                   fill_masked_tail: bool = True) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Batched hard-negative mining: for query i (positive = corpus row offset+i) drop every candidate
    scoring above ratio * s_pos[i] and return the best k of the rest.

    Returns (indices i64 [n,k], values f32 [n,k], s_pos f32 [n]) on the GPU.  If fewer than k
    candidates survive, the reference's argsort puts masked (-inf) columns in the tail in unspecified
    order; with fill_masked_tail the tail is filled with masked columns (best first), else with -1.
    """
    s_pos = positive_scores(q, c, offset)
    ub = s_pos * ratio                                   # fp32 multiply, as scores[idx]*.95
    vals, idx, _ = topk(q, c, k, upper_bound=ub)
    if fill_masked_tail:
        fill_masked_tail_rows(idx, ub, lambda rows: topk(q.take(rows), c, k)[:2])
    return idx, vals, s_pos


def fill_masked_tail_rows(idx: torch.Tensor, ub: torch.Tensor, unbounded_topk) -> None:
    """Rows of `idx` with fewer than k survivors (-1 holes) get the masked columns appended, best first, as the
    reference's argsort()[:top] does (create_negative_index.py:50-51 always yields `top` entries; the consumer
    indexes up to 5*negatives-1, conceptual_captions.py:152-156).  `unbounded_topk(rows) -> (vals, idx)` is a
    second search of those rows without the bound; the single-GPU and the sharded driver both come through here,
    so a mining run writes the same lists at every world size."""
    k = idx.shape[1]
    holes = (idx < 0).any(dim=1).nonzero().flatten()
    if not holes.numel():
        return
    v2, i2 = unbounded_topk(holes)
    for r, row in enumerate(holes.tolist()):
        masked = i2[r][(v2[r] > ub[row]) & (i2[r] >= 0)]
        n_ok = int((idx[row] >= 0).sum())
        take = min(k - n_ok, masked.numel())
        idx[row, n_ok:n_ok + take] = masked[:take]


_resident_last: list = []            # [(key, weak reference to the tensor, Embeddings)]: the corpus of the last per-sample call


def _resident(c: torch.Tensor, compute: str) -> Embeddings:
    """The reference's loop hands the SAME corpus tensor to every per-sample call (create_negative_index.py:37-38): its
    resident form (upload, bf16 cast or int8 quantisation: a pass over the whole corpus) is built once and kept while the
    calls keep naming that tensor, unmodified (same object, storage, shape, dtype and version counter).  One entry; it
    holds device memory until another corpus comes or release_resident() is called."""
    key = (c.data_ptr(), tuple(c.shape), c.dtype, c.device, c._version, compute)
    if _resident_last and _resident_last[0][0] == key and _resident_last[0][1]() is c:
        return _resident_last[0][2]
    emb = Embeddings(c, compute)
    _resident_last[:] = [(key, weakref.ref(c), emb)]
    return emb


def release_resident() -> None:
    """Drop the corpus kept by the per-sample form of negatives_for_sample."""
    _resident_last.clear()


def negatives_for_sample(idx: int, negative_dict: dict, q: torch.Tensor, c, top: int = 100, compute: str = "f32"):
    """Same call as the reference: negative_dict[idx] = the `top` best candidates for query row idx
    among those not scoring above 0.95 * scores[idx].  `c` may be a tensor or a resident Embeddings; a tensor's resident
    form is kept from one call to the next (_resident), so the reference's loop does not convert the corpus per query."""
    cc = c if isinstance(c, Embeddings) else _resident(c, compute)
    qq = Embeddings(q[idx:idx + 1], compute, cc.data.device)
    ids, _, _ = mine_negatives(qq, cc, top, offset=idx)
    negative_dict[idx] = [j for j in ids[0].cpu().tolist() if j >= 0]


# ----------------------------------------------------------------------------------------------
# a5 / a6: visualization/neg_mine.py
# ----------------------------------------------------------------------------------------------
def batch(query, cand, idx: int, batch_size: int, top_k: int, compute: str = "f32"):
    """Same call and return as neg_mine.batch: CPU tensors (score [b,k] f32, topk_idx [b,k] i64,
    mask_sum_norm [b] f32 = fraction of candidates scoring above the positive, scores_for_answer [b])."""
    q = query if isinstance(query, Embeddings) else Embeddings(query, compute)
    c = cand if isinstance(cand, Embeddings) else Embeddings(cand, compute, q.data.device)
    n = q.shape[0]
    batch_idx = idx + batch_size if idx + batch_size < n else n
    qs = q.rows(idx, batch_idx)
    s_pos = positive_scores(qs, c, idx)
    score, topk_idx, rank = topk(qs, c, top_k, rank_ref=s_pos, rank_self_offset=idx)
    # mask_sum / cand.shape[0] (neg_mine.py:39) on the HOST: torch's fp32 division on this GPU is not correctly rounded (one
    # ulp off the IEEE quotient in 7 of 4 444 rows of a soak case); the counts themselves are integers from the kernel
    mask_sum_norm = rank.cpu() / c.shape[0]
    return score.cpu(), topk_idx.cpu(), mask_sum_norm, s_pos.cpu()


def compute_topk(path: str, top_k: int, compute: str = "f32", batch_size: int = 3_000) -> None:
    """neg_mine.compute_topk: reads query.pt / cand.pt under `path`, writes top_k.pt (float32
    [2,Nq,k]: [0]=scores, [1]=indices as float, the reference's layout), relative_scoring.pt,
    absolute_scoring.pt and, in addition, top_k_idx.pt (int64 indices, exact beyond 2^24 rows)."""
    query = torch.load(os.path.join(path, "query.pt"), weights_only=True)
    cand = torch.load(os.path.join(path, "cand.pt"), weights_only=True)
    q = Embeddings(query, compute)
    c = Embeddings(cand, compute, q.data.device)
    scores, idxs, rel, absolute = [], [], [], []
    i = 0
    while i < q.shape[0]:
        s, t, p, a = batch(q, c, i, batch_size, top_k)
        scores.append(s)
        idxs.append(t)
        rel.append(p)
        absolute.append(a)
        i += batch_size
    scores, idxs = torch.cat(scores, 0), torch.cat(idxs, 0)
    torch.save(torch.stack((scores, idxs.to(torch.float32))), os.path.join(path, "top_k.pt"))
    torch.save(idxs, os.path.join(path, "top_k_idx.pt"))
    torch.save(torch.cat(rel, 0), os.path.join(path, "relative_scoring.pt"))
    torch.save(torch.cat(absolute, 0), os.path.join(path, "absolute_scoring.pt"))
