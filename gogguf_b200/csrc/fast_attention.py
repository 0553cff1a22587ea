"""Host side of the tensor-core attention kernels (csrc/attention_fast.cu): choice between the
decode kernel (every sequence brings one token) and the prefill kernel, scratch for the splits."""
from __future__ import annotations

import functools
import struct
from typing import Callable, List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import kernels as K
from .build import KernelError, kernel, module, stream_ptr
from .tcgen05_gemm import status_word


def decode_splits(n_tokens: int, nkv: int, max_ctx: int) -> int:
    return int(module("attention_fast").lib.gg_attn_decode_splits(int(n_tokens), int(nkv), int(max_ctx)))


def _gate(gate):
    return (gate.data_ptr(), gate.stride(0)) if gate is not None else (0, 0)


def attn_decode(q, k_pool, v_pool, out, positions, seq_of_token, table, page_size, n_tokens, nq, nkv, d,
                scale, window, splits, part_o=None, part_ml=None) -> None:
    kernel("attention_fast", "gg_attn_decode")(
        q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr(),
        part_o.data_ptr() if part_o is not None else 0, part_ml.data_ptr() if part_ml is not None else 0,
        positions.data_ptr(), seq_of_token.data_ptr(), table.data_ptr(), table.shape[-1], page_size,
        k_pool.shape[0], n_tokens, nq, nkv, d, float(scale), int(window), int(splits),
        status_word(q.device).data_ptr(), stream_ptr())


# The launchers' arguments (csrc/attention_fast.cu: DecodeCall, csrc/attention_shared.cu: SharedCall).
_DECODE_CALL, _SHARED_CALL = struct.Struct("=25q2d").pack, struct.Struct("=24q2d").pack


@functools.lru_cache(maxsize=4096)
def decode_tma_splits(n_tokens: int, nkv: int, max_ctx: int, cluster: bool = False) -> int:
    return int(module("attention_fast").lib.gg_attn_decode_tma_splits(int(n_tokens), int(nkv), int(max_ctx),
                                                                      int(bool(cluster))))


def attn_decode_tma(q, k_pool, v_pool, out, positions, seq_of_token, table, page_size, n_tokens, nq, nkv, d,
                    scale, window, splits, part_o=None, part_ml=None, cluster: bool = False, sink=None,
                    out_scale: float = 1.0, dv: Optional[int] = None, chunk: int = 0, gate=None) -> None:
    """Decode attention with the cache streamed through a TMA ring (pools: [page][nkv][64][d]).
    cluster=True merges the splits inside thread-block clusters (no scratch, no second kernel).
    sink: float32 per query head, joins the softmax's denominator; out_scale: a factor on the result (neither is
    taken by the form that merges its splits with a second kernel).  dv: the values' head size (default d); chunk: a
    position sees its own chunk of that many positions only; gate (rows of nq * dv logits): multiplied in by its sigmoid."""
    kernel("attention_fast", "gg_attn_decode_tma_packed")(_DECODE_CALL(
        q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr(),
        part_o.data_ptr() if part_o is not None else 0, part_ml.data_ptr() if part_ml is not None else 0,
        positions.data_ptr(), seq_of_token.data_ptr(), table.data_ptr(), table.shape[-1], page_size,
        k_pool.shape[0], n_tokens, nq, nkv, d, d if dv is None else int(dv), int(window), int(chunk), int(splits),
        int(bool(cluster)), sink.data_ptr() if sink is not None else 0, *_gate(gate),
        status_word(q.device).data_ptr(), scale, out_scale), stream_ptr())


# The most runs over the prefixes, rows of a tile, and the most CTAs that may share a row's own pages (csrc/attention_shared.cu).
SHARED_RUNS, SHARED_ROWS, SHARED_SHARES = 296, 128, 8


def shared_scratch(n_tokens: int, nq: int, nkv: int, dv: int, shares: Optional[int] = None) -> int:
    """Floats of scratch that `attn_decode_shared` needs (for whatever `shares` it chooses itself, or for a given number): the parts'
    rows, two numbers beside each, and where a row's parts are."""
    if n_tokens <= 0 or nkv <= 0 or nq <= 0 or nq % nkv or dv <= 0:
        raise KernelError(f"shared attention: {nq} heads on {nkv} kv heads of {dv}, {n_tokens} tokens")
    if shares is None:
        shares = shared_shares(n_tokens, nkv, 2 * SHARED_SHARES)
    return (nq * n_tokens * (2 + shares) + SHARED_ROWS * SHARED_RUNS) * (dv + 2) + 4 * n_tokens * nkv


def shared_shares(n_tokens: int, nkv: int, own_pages: int) -> int:
    """CTAs that share a row's own pages, of which the longest row has `own_pages`: up to one and a half for each place on the device, and
    two pages each at least (25 rows of 4 kv heads of 80, some of which have 37 pages of their own, 1 / 2 / 4 shares: 25.6 / 18.1 /
    16.4 us; 64 rows of 8 kv heads, with up to 8 pages, 28 / 30 / 34)."""
    return max(1, min(444 // (n_tokens * nkv), own_pages // 2, SHARED_SHARES))


def prefix_pays(groups: Sequence[Tuple[int, int]], n_tokens: int, nkv: int) -> bool:
    """Is reading the prefixes of groups of (members, pages) once, in a step of n_tokens rows, quicker than every row for itself?  From
    12 pages of prefixes on that a CTA of the unshared kernel would read (measured, us, unshared / shared with two pages of a row's own,
    32 heads of 128 on 8 kv heads: 2 rows, 8 pages a CTA 10.0 / 12.7, 16 15.3 / 14.8, 32 26 / 20; 8 rows, 8 10.6 / 12.1, 16 16.0 / 14.7;
    32 rows, 32 26 / 19; 64 rows, 14 20.9 / 18.1, 27 31 / 19; 16 heads of 64 on 8: 8 rows, 8 8.7 / 10.2, 16 14.1 / 11.5; 24 heads of 80 on
    4: 16 rows, 8 11.2 / 12.7, 16 16.7 / 13.9).

    It counts pages, neither head sizes nor the query heads of a kv head.  Of 168 measured calls it takes the slower form, by more
    than 5 %, in six: with sixteen query heads a kv head sharing gains sooner (32 heads of 128 on 2, read apart: 64 rows, 16 pages shared
    20.4 / 16.0, 8 17.4 / 15.4; 32 rows, 32 17.2 / 15.7); and around the bound (read together: 32 heads on 8, 32 rows, 16 pages 15.9 / 17.1;
    16 heads of 64 on 8, 64 rows, 8 13.8 / 14.9; 2 rows, 128 11.6 / 12.3)."""
    pairs, splits = n_tokens * nkv, 1
    while splits * 2 <= min(8, 296 // pairs):
        splits *= 2
    return sum(members * pages for members, pages in groups) * nkv >= 12 * min(296, pairs * splits)


def shared_runs(groups: Sequence[Tuple[int, int]], nq: int, nkv: int) -> int:
    """CTAs over the prefixes of groups of (members, pages): one an SM at most, which leaves room for the CTAs of the rows' own pages beside
    it, until those would have more than six pages each (measured, us, one against two an SM: 64 rows of 32 heads on 32 pages 28 / 36;
    12 rows of 32 heads on 2 kv heads, 256 pages 23 / 20; 64 rows on 512 pages 74 / 62), and with four pages each at least: a CTA's beginning
    and end cost as much as three (64 rows on 16 pages, 2 / 3 / 4 / 8 pages a CTA: 27.0 / 26.0 / 25.7 / 26.2; 32 rows on 32 pages 22.1 /
    23.3 / 20.8 / 22.9; 48 and 16 rows of 40 heads on 20 pages 29.2 / 26.7 / 25.6 / 31.5)."""
    most = SHARED_ROWS // (nq // nkv)
    units = sum(pages * -(-members // most) for members, pages in groups) * nkv
    if units > 6 * (SHARED_RUNS // 2):
        return SHARED_RUNS
    return min(SHARED_RUNS // 2, -(-units // 4)) or SHARED_RUNS // 2


def step_launch(groups: Sequence[Tuple[int, int]], own_pages: int, n_tokens: int, nq: int, nkv: int) -> Tuple[int, int]:
    """(runs, shares) of a model's step: `shared_runs` up to a power of two (or all SMs, or two a SM), and `shared_shares` of the own pages
    down to one, so that a captured step is the same launch for prompts of about a length and while answers grow."""
    runs, half = shared_runs(groups, nq, nkv), SHARED_RUNS // 2
    runs = SHARED_RUNS if runs > half else min(half, 1 << (runs - 1).bit_length())
    return runs, shared_shares(n_tokens, nkv, 1 << max(0, own_pages.bit_length() - 1))


def shared_groups(table: np.ndarray, limits: Sequence[int]) -> List[Tuple[List[int], int]]:
    """The rows of a page table that read the same leading pages: [(rows, pages)], each with two rows and one page at least.
    `limits[r]`: how many leading pages of row r may be shared (those that lie wholly before its newest position).  A row is
    in one group at most: where some rows of a group share more pages than all of it, the cut that saves more reads is taken."""
    table = np.asarray(table)

    def best(rows: List[int], depth: int, cuts: int = 0) -> Tuple[int, List[Tuple[List[int], int]]]:
        if len(rows) < 2:
            return 0, []
        most = min(limits[r] for r in rows)
        part = table[rows, depth:most]
        differs = np.nonzero((part != part[0]).any(axis=0))[0]
        common = depth + int(differs[0]) if differs.size else most
        whole = (len(rows) - 1) * common, ([(rows, common)] if common else [])
        below = {}
        for r in rows if cuts < 100 else ():            # (sequences that branch off one another a hundred times are read as one group)
            if limits[r] > common:
                below.setdefault(int(table[r, common]), []).append(r)
        saved, groups = 0, []
        for members in below.values():
            s, g = best(members, common + 1, cuts + 1)
            saved, groups = saved + s, groups + g
        return (saved, groups) if saved > whole[0] else whole

    roots = {}
    for r, n in enumerate(limits):
        if n > 0:
            roots.setdefault(int(table[r, 0]), []).append(r)
    return [g for rows in roots.values() for g in best(rows, 1)[1]]


class PrefixPlan:
    """Which token rows of a decode step read which prefix together, as `attn_decode_shared` takes it: `groups` is a list of
    (token rows, leading pages that are the same in all their sequences).  Every shared page must lie wholly before its rows'
    own positions.  A plan serves all layers of a step that read through the same page table.  `own_pages`: the pages that each
    row reads beside the shared ones, where that is known (it only chooses the launch and its order)."""

    def __init__(self, groups: Sequence[Tuple[Sequence[int], int]], n_tokens: int, device, own_pages: Optional[Sequence[int]] = None):
        host = torch.empty(self.words_for(n_tokens), dtype=torch.int32)
        self.pack(groups, n_tokens, host.numpy(), own_pages)
        self.n_tokens = n_tokens
        self.words = host.to(device)
        self.own_pages = None if own_pages is None else max(own_pages)
        self.groups: Optional[List[Tuple[int, int]]] = [(len(rows), int(pages)) for rows, pages in groups]
        self.longest = max((pages for _, pages in self.groups), default=0)

    def pays(self, nkv: int) -> bool:
        """`prefix_pays` of this plan's groups (True where they are not known, or where the plan's maker has found so), worked out once."""
        if not self.found and self._pays[0] != nkv:
            self._pays = (nkv, self.groups is None or prefix_pays(self.groups, self.n_tokens, nkv))
        return self._pays[1]

    def launch(self, nq: int, nkv: int, width: int) -> Tuple[int, int]:
        """(runs, shares) of a launch over a page table of `width` pages, where the caller does not choose them."""
        if self.found:
            return step_launch(self.groups or (), width if self.own_pages is None else self.own_pages, self.n_tokens, nq, nkv)
        return (shared_runs(self.groups or (), nq, nkv),
                shared_shares(self.n_tokens, nkv, width if self.own_pages is None else self.own_pages))

    _pays = (0, True)             # kv heads, and the answer for them
    found = False                 # a model's step: what shares was chosen because it pays

    @staticmethod
    def words_for(n_tokens: int) -> int:
        return 5 + 8 * n_tokens

    @classmethod
    def over(cls, words: torch.Tensor, n_tokens: int, own_pages: Optional[int] = None,
             groups: Optional[Sequence[Tuple[int, int]]] = None, found: bool = False) -> "PrefixPlan":
        """A plan whose words are (or will be) on the device already, packed by `pack`; `groups`: (members, pages) of those it will
        hold, and `own_pages`, the most that a row reads beside them, choose the launch (any others are right, too).  `found`: the
        groups of a model's step, chosen because reading them together pays: that is not asked again (the rows that fill up a captured
        step would be counted), and the launch is `step_launch`'s."""
        plan = cls.__new__(cls)
        if words.dtype != torch.int32 or words.numel() != cls.words_for(n_tokens) or not words.is_contiguous():
            raise KernelError(f"shared attention: a plan of {n_tokens} tokens has {cls.words_for(n_tokens)} int32 words")
        plan.n_tokens, plan.words, plan.own_pages, plan.groups = (
            n_tokens, words, own_pages, None if groups is None else list(groups))
        plan.found = bool(found)
        plan.longest = max((pages for _, pages in plan.groups or ()), default=0)
        return plan

    @classmethod
    def pack(cls, groups: Sequence[Tuple[Sequence[int], int]], n_tokens: int, out: np.ndarray, own_pages: Optional[Sequence[int]] = None) -> None:
        """Write the plan's words (csrc/attention_shared.cu: SharedArgs) to `out`, with the rows of most `own_pages` first in the order in
        which those are read; refuses rows that are not the step's, that
        appear twice, and groups without a row or page."""
        if n_tokens <= 0:
            raise KernelError("shared attention: a plan needs at least one token row")
        first = out[4:5 + n_tokens]
        pages, lead, rows, pages_of, group_of, member_of, order = (out[5 + k * n_tokens:5 + (k + 1) * n_tokens] for k in range(1, 8))
        out[:cls.words_for(n_tokens)] = 0
        group_of[:] = -1
        if own_pages is not None and len(own_pages) > n_tokens:
            raise KernelError(f"shared attention: own pages of {len(own_pages)} rows, the step has {n_tokens}")
        most = np.zeros(n_tokens, dtype=np.int64)
        most[:len(own_pages or ())] = own_pages or ()
        order[:] = np.argsort(-most, kind="stable")
        at = 0
        for g, (members, shared) in enumerate(groups):
            members = list(members)
            if not members or shared <= 0:
                raise KernelError("shared attention: a group has at least one row and one page")
            if min(members) < 0 or max(members) >= n_tokens or len(set(members)) != len(members) or (group_of[members] >= 0).any():
                raise KernelError(f"shared attention: rows {members} are not rows of {n_tokens} tokens, or appear twice")
            pages[g], lead[g] = shared, members[0]
            rows[at:at + len(members)] = members
            group_of[members] = g
            pages_of[members] = shared
            member_of[members] = np.arange(len(members))
            at += len(members)
            first[g + 1] = at
        out[0] = len(groups)

    @classmethod
    def of_pages(cls, pages: Sequence[Sequence[int]], lengths: Sequence[int], page_size: int, device) -> "PrefixPlan":
        """The plan of a step with one token per sequence: `pages[r]` lists the pages of row r's sequence, `lengths[r]` is its
        length with the new token."""
        if len(pages) != len(lengths):
            raise KernelError(f"shared attention: {len(pages)} page lists and {len(lengths)} lengths")
        if not pages:
            raise KernelError("shared attention: a plan needs at least one token row")
        for r, (p, n) in enumerate(zip(pages, lengths)):
            if n < 0 or len(p) * page_size < n:
                raise KernelError(f"shared attention: row {r} has {n} positions in {len(p)} pages of {page_size}")
        table = np.full((len(pages), max(1, max(len(p) for p in pages))), -1, dtype=np.int64)
        for r, p in enumerate(pages):
            table[r, :len(p)] = p
        groups = shared_groups(table, [max(0, (n - 1) // page_size) for n in lengths])
        own = [-(-n // page_size) for n in lengths]
        for rows, shared in groups:
            for r in rows:
                own[r] -= shared
        return cls(groups, len(pages), device, own_pages=own)


def attn_decode_shared(q, k_pool, v_pool, out, positions, seq_of_token, table, page_size, plan: PrefixPlan, scratch, nq, nkv, d, scale,
                       sink=None, out_scale: float = 1.0, dv: Optional[int] = None, gate=None, together: Optional[bool] = None, runs: Optional[int] = None,
                       shares: Optional[int] = None) -> None:
    """Decode attention (`attn_decode_tma`, without windows and chunks) of the plan's token rows: the keys and values of a prefix
    that several rows share are read once for all of them, in three kernels, where that pays (`prefix_pays`; `together` True or
    False decides instead).  What is shared, the plan and the table are read before the kernel that was launched before this call has
    ended (what other kernels and PyTorch wrote before that is there), so that one must not write to them; only a row's own positions
    may be the kernel before's.  The pages hold finite numbers behind a row's newest position, too (a cache begins as zeros): their
    weight is 0.  scratch: float32, `shared_scratch` of it; two launches that may run at the same time need scratch of
    their own.  runs: CTAs over the prefixes (default: `shared_runs`); shares: CTAs that share a row's own pages (default:
    `shared_shares`; `PrefixPlan.launch`)."""
    dv = d if dv is None else int(dv)
    T = plan.n_tokens
    if not takes(nq, nkv, d, dv):
        raise KernelError(f"shared attention: {nq} heads on {nkv} kv heads of {d} and {dv} are outside what the kernels take")
    bf16, i32, f32, words = torch.bfloat16, torch.int32, torch.float32, plan.words
    here = torch._C._cuda_getDevice() if q.is_cuda else -1
    wrong = None if here >= 0 else q
    for t in (q, k_pool, v_pool, out):
        if t.dtype is not bf16 or t.get_device() != here or not t.is_contiguous():
            wrong = t
    for t in (positions, seq_of_token, table, words):
        if t.dtype is not i32 or t.get_device() != here or not t.is_contiguous():
            wrong = t
    for t in (scratch,) if sink is None else (scratch, sink):
        if t.dtype is not f32 or t.get_device() != here or not t.is_contiguous():
            wrong = t
    if wrong is not None:
        raise KernelError("shared attention: q, the pools and out are bfloat16, positions, seq_of_token, the table and the plan int32, "
                          "scratch and a sink float32, all contiguous and on the current CUDA device: got "
                          f"{wrong.dtype} of {tuple(wrong.shape)} with strides {wrong.stride()} on {wrong.device}")
    k_shape, t_shape = k_pool.shape, table.shape
    pools, width = k_shape[0], t_shape[-1]
    if (q.numel() < T * nq * d or out.numel() < T * nq * dv or positions.numel() < T or seq_of_token.numel() < T or len(t_shape) != 2
            or k_shape != (pools, nkv, page_size, d) or v_pool.shape != (pools, nkv, page_size, dv)):
        raise KernelError("shared attention: shapes disagree")
    if plan.longest > width:
        raise KernelError(f"shared attention: the plan's prefixes are longer than the table's {width} pages")
    p_sink = p_gate = ldg = 0
    if sink is not None:
        if sink.numel() != nq:
            raise KernelError(f"shared attention: a sink has {nq} elements")
        p_sink = sink.data_ptr()
    if gate is not None:
        if (gate.dtype != bf16 or gate.dim() != 2 or gate.shape[0] < T or gate.shape[1] < nq * dv or gate.stride(1) != 1
                or gate.get_device() != here):
            raise KernelError(f"shared attention: a gate is bfloat16 with {T} rows of {nq * dv}, on the current CUDA device")
        p_gate, ldg = gate.data_ptr(), gate.stride(0)
    if together is None:
        together = plan.pays(nkv)
    if not together:
        if page_size != 64:
            raise KernelError(f"shared attention: pages of 64 positions, not {page_size}")
        splits = decode_tma_splits(T, nkv, width * page_size, True)
        if not (d == dv and d in (64, 128)):
            splits = min(splits, 8)
        attn_decode_tma(q, k_pool, v_pool, out, positions, seq_of_token, table, page_size, T, nq, nkv, d, scale, 0, splits, cluster=True,
                        sink=sink, out_scale=out_scale, dv=dv, gate=gate)
        return
    if runs is None or shares is None:
        launch = plan.launch(nq, nkv, width)
        runs, shares = launch[0] if runs is None else runs, launch[1] if shares is None else shares
    if not 1 <= runs <= SHARED_RUNS:
        raise KernelError(f"shared attention: 1 to {SHARED_RUNS} runs, not {runs}")
    if not 1 <= shares <= SHARED_SHARES:
        raise KernelError(f"shared attention: 1 to {SHARED_SHARES} shares, not {shares}")
    room = shared_scratch(T, nq, nkv, dv, shares)
    if scratch.numel() < room:
        raise KernelError(f"shared attention: scratch must have {room} elements")
    kernel("attention_shared", "gg_attn_decode_shared")(_SHARED_CALL(
        q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr(), positions.data_ptr(), seq_of_token.data_ptr(), table.data_ptr(),
        width, page_size, pools, words.data_ptr(), T, nq, nkv, d, dv, runs, shares, p_sink, p_gate, ldg, scratch.data_ptr(), scratch.numel(),
        status_word(q.device).data_ptr(), scale, out_scale), stream_ptr())


def attn_prefill(q, k_pool, v_pool, out, cu_seqlens, ctx_lens, seq_of_token, table, page_size, n_seqs,
                 max_tiles, nq, nkv, d, scale, window, sink=None, out_scale: float = 1.0, dv: Optional[int] = None,
                 chunk: int = 0, gate=None) -> None:
    kernel("attention_fast", "gg_attn_prefill")(
        q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr(), cu_seqlens.data_ptr(),
        ctx_lens.data_ptr(), seq_of_token.data_ptr(), table.data_ptr(), table.shape[-1], page_size,
        k_pool.shape[0], n_seqs, max_tiles, nq, nkv, d, d if dv is None else int(dv), float(scale), int(window), int(chunk),
        sink.data_ptr() if sink is not None else 0, float(out_scale), *_gate(gate),
        status_word(q.device).data_ptr(), stream_ptr())


def attn_prefill_tc(q, k_pool, v_pool, out, cu_seqlens, ctx_lens, seq_of_token, table, page_size, n_tokens,
                    n_seqs, max_tiles, nq, nkv, d, scale, window, sink=None, out_scale: float = 1.0,
                    dv: Optional[int] = None, chunk: int = 0, gate=None, splits: int = 1) -> None:
    """Prefill attention on tcgen05: 128-query tiles, S and O in tensor memory; the pages of a tile shared by `splits` CTAs."""
    kernel("attention_fast", "gg_attn_prefill_tc")(
        q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out.data_ptr(), cu_seqlens.data_ptr(),
        ctx_lens.data_ptr(), seq_of_token.data_ptr(), table.data_ptr(), table.shape[-1], page_size,
        k_pool.shape[0], n_tokens, n_seqs, max_tiles, nq, nkv, d, d if dv is None else int(dv), float(scale), int(window),
        int(chunk), int(splits), sink.data_ptr() if sink is not None else 0, float(out_scale), *_gate(gate),
        status_word(q.device).data_ptr(), stream_ptr())


# (query tile, head) pairs whose shares are all on the device at once, by the CTAs of a cluster: pairs fill all 296 places, larger
# clusters do not (64 clusters of four run side by side and 72 do not; 32 of eight do).
_RESIDENT = {2: 148, 4: 66, 8: 32}


def prefill_tiles(n_tokens: int, n_seqs: int, max_new: int) -> int:
    """At least as many 128-query tiles as the sequences of a step have."""
    return min(n_tokens // 128 + n_seqs, n_seqs * -(-max_new // 128))


def prefill_splits(n_tokens: int, n_seqs: int, nq: int, reach: int, max_new: Optional[int] = None, wide: int = 128) -> int:
    """CTAs that share the pages of a query tile which reads up to `reach` positions: the 1, 2, 4 or 8 that a few constants
    call quickest, of those that fit the device and leave a share two pages, from 512 positions on.  A page takes a CTA 0.55 us; a cluster that adds up its
    shares takes 2 us, 0.065 us for every row that a CTA adds up (0.1 with rows of up to 64 values), and 2 us more
    where the shares are what puts two CTAs on an SM.  Measured (us, in 1 / 2 / 4 / 8 shares): 333 tokens of 16 heads of
    64 on 520 positions 10.4 / 14.8 / 13.4, of 32 heads of 128 on 1,024 16.8 / 17.5, on 6,400 79 / 51; 128 tokens of 16 heads of 64 on
    1,024 14.4 / 17.6 / 13.7 / 12.1.  A sequence's shares depend on the whole step, and with them the order in which its
    values are added."""
    rows = n_tokens if max_new is None else max_new
    pairs, pages = prefill_tiles(n_tokens, n_seqs, rows) * nq, -(-reach // 64)
    best, gained = 1, 0.0
    for splits, most in _RESIDENT.items():
        if pairs > most or reach < 512 or 2 * splits > pages:
            break
        gain = 0.55 * (pages - -(-pages // splits)) - (2.0 if pairs * splits <= 148 else 4.0)
        gain -= (0.065 if wide > 64 else 0.1) * -(-min(rows, 128) // splits)
        if gain > gained:
            best, gained = splits, gain
    return best


@functools.lru_cache(maxsize=4096)
def takes(nq: int, nkv: int, d: int, dv: int) -> bool:
    """Do the tensor-core kernels take these sizes?  Head sizes in multiples of 8 up to 128, at most 16 query heads per kv
    head."""
    return nq % nkv == 0 and nq // nkv <= 16 and all(0 < n <= 128 and n % 8 == 0 for n in (d, dv))


def try_make(nq: int, nkv: int, d: int, scale: float, window: int, dv: Optional[int] = None,
             chunk: int = 0) -> Optional[Callable]:
    """f(q, k_pool, v_pool, out, ctx, table, page_size, sink=None, out_scale=1.0, gate=None, prefix=None) for bfloat16, or
    None when the sizes are outside what the tensor-core kernels take; then the plain kernel serves.  prefix: the `PrefixPlan` of
    a decode step whose sequences share pages (not read by windowed or chunked attention)."""
    dv = d if dv is None else dv
    if not takes(nq, nkv, d, dv):
        return None
    exact = d == dv and d in (64, 128)

    def run(q, k_pool, v_pool, out, ctx, table, page_size, sink=None, out_scale=1.0, gate=None, prefix=None):
        T = ctx.n_tokens
        kw = dict(sink=sink, out_scale=out_scale, dv=dv, chunk=chunk, gate=gate)
        if page_size != 64 or q.dtype != torch.bfloat16:
            K.attention_plain(q, k_pool, v_pool, out, ctx.positions, ctx.seq_of_token, table, page_size,
                              T, nq, nkv, d, scale, window, **kw)
            return
        if ctx.decode and prefix is not None and not window and not chunk:
            scratch = ctx.ws.get("attn_prefix_parts", (shared_scratch(T, nq, nkv, dv),), torch.float32)
            attn_decode_shared(q, k_pool, v_pool, out, ctx.positions, ctx.seq_of_token, table, page_size, prefix, scratch, nq, nkv, d,
                               scale, sink=sink, out_scale=out_scale, dv=dv, gate=gate)
            return
        if ctx.decode:
            # (what lies before a window or a chunk is not read: no more splits than the pages that are)
            reach = min([ctx.max_ctx] + [n + 64 for n in (window, chunk) if n])
            splits = decode_tma_splits(T, nkv, reach, cluster=True)
            if not exact:
                splits = min(splits, 8)
            attn_decode_tma(q, k_pool, v_pool, out, ctx.positions, ctx.seq_of_token, table, page_size, T, nq, nkv, d,
                            scale, window, splits, cluster=True, **kw)
            return
        max_tiles = prefill_tiles(T, ctx.n_seqs, ctx.max_new)
        reach = min([ctx.max_ctx] + [n + 192 for n in (window, chunk) if n])
        if ctx.max_new >= 32 or (reach >= 512 and max_tiles * nq <= _RESIDENT[2]):
            # 128-query tiles on tcgen05 (S and O in tensor memory); a few tokens per sequence too where a walk over their history
            # is what takes the time (3 tokens on 520, 32 heads of 128: 10.9 us against 20.6; 16 heads of 64: 9.5 against 12.6; 10
            # tokens on 6,400, 32 heads of 128: 20 in shares against 194)
            splits = prefill_splits(T, ctx.n_seqs, nq, reach, ctx.max_new, dv)
            attn_prefill_tc(q, k_pool, v_pool, out, ctx.cu_seqlens, ctx.ctx_lens, ctx.seq_of_token, table, page_size,
                            T, ctx.n_seqs, max_tiles, nq, nkv, d, scale, window, splits=splits, **kw)
        else:
            # a few tokens per sequence: 64-query tiles on mma.sync waste less
            max_tiles = T // 64 + ctx.n_seqs
            attn_prefill(q, k_pool, v_pool, out, ctx.cu_seqlens, ctx.ctx_lens, ctx.seq_of_token, table, page_size,
                         ctx.n_seqs, max_tiles, nq, nkv, d, scale, window, **kw)

    return run
