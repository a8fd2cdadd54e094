"""Serving with a paged key / value cache (no counterpart in the reference): a pool of pages of a fixed number of tokens, shared by sequences that list
theirs in a page table.

    k_cache, v_cache   (pages, page size, nheads_k, headdim) fp16 or bf16, any strides with a contiguous last dimension; page size: a power of two
                       from 16 to 1024.  PagedKVCache lays a page out head by head, so that a head's keys of a page are one piece of memory.
    page_table         (batch, pages per sequence) int32: token j of sequence b is in page page_table[b, j // page_size]
    seqlens_k          (batch,) int32: tokens of each sequence that the cache holds, the new ones among them
    cu_seqlens_q       (batch + 1,) int32: where each sequence's new tokens begin in the packed (total, heads, headdim) tensors

A step of a model advances seqlens_k by the new tokens once; every layer then stores them (paged_append_func) and attends
(flash_attn_paged_func).  Nothing here waits for the GPU or reads its memory on the host: the functions' calls can be captured into a graph, whose replays
find new lengths, tables and tokens in the same tensors (PagedKVCache's book is the host's: its steps are made, and its evictions called, outside).
max_seqlen_k then has to hold for all of them; it bounds the work that is cut, not the memory that is read.

A cache in 8 bits: k_cache and v_cache are torch.float8_e4m3fn, and beside them k_scales and v_scales (pages, nheads_k, page size) uint8 hold an exponent + 127 for every
slot and key head, of which the row stands for its values times 2^exponent.  paged_append_func rounds each row once, to the nearest values under the smallest exponent
that brings its largest finite magnitude to 448 or below (-15 to 8 for fp16, -100 to 120 for bf16; under the largest one values end at 240; inf and NaN become NaN):
a value is off by 2^-4 of itself at most, and by 2^-10 of the scale where it is small.  What a row stands for is exact in the dtype it came from, which is the one to read it
in and to attend with.  Key weights and eviction are those of caches in 16 bits.

What lies in page_table and seqlens_k is never trusted with an address: entries outside the pool are read as its first or last page and never written to,
lengths count as far as the table goes.  Pages that several sequences list (a common prompt), or one lists twice, may be read by all of them and must not be
appended to, weighted or evicted from: the order in which several workgroups write one slot is not defined.  Keys and values behind a sequence's length are not
read.  A value that is inf or NaN reaches every new token of its sequence that is handled together with one that sees it, as in the package's other
attention functions: a weight of 0 does not cancel it."""
from array import array

import torch
from torch.autograd import forward_ad

from . import flash_attn_gfx950 as _backend


def _inference(*tensors, constants=()):
    """constants: tensors that no gradient is formed of, but whose tangents would be lost just as well"""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("the paged cache has no backward: call it under torch.no_grad()")
    # (a tangent is there under no_grad, too)
    if torch._C._is_fwd_grad_enabled() and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (*tensors, *constants)):
        raise RuntimeError("the paged cache has no derivative in forward mode")


def paged_append_func(q, k, v, k_cache, v_cache, page_table, cu_seqlens, seqlens_k, q_weight=None, k_weight=None, cos_half=None, sin_half=None,
                      positions=None, eps=1e-6, key_weights=None, key_positions=None, k_scales=None, v_scales=None):
    """Stores the new tokens' k and v (total, nheads_k, headdim) into the pages of their sequences, behind what is there: row i of sequence b goes to
    slot seqlens_k[b] - (its new tokens) + i.  In the same pass k, and q (total, nheads, headdim) if it is given, are normalised (q_weight, k_weight: see
    apply_qk_norm_rotary) and turned by their positions (cos_half, sin_half) - positions[row], or the slot, clamped to the tables: they are on the device, and what
    the tables have to reach is the caller's to know (PagedStep does).  Returns the new q, or None.
    key_weights, key_positions (pages, nheads_k, page size): set to 0 and the position for the new tokens (for paged_key_weights_func and
    paged_evict_func).  k_scales, v_scales: of a cache in 8 bits, into which k and v are quantised.  Rows behind the last sequence, and tokens for which the page
    table has no room, are not stored; their rows of the returned q hold nothing."""
    done = _backend.passes().paged_append(q, k, v, k_cache, v_cache, page_table, cu_seqlens, seqlens_k, q_weight, k_weight, cos_half, sin_half, positions, eps,
                                          key_weights, key_positions, k_scales, v_scales)
    if done is not None:
        return None if q is None else done
    _inference(q, k, v, q_weight, k_weight, constants=(k_cache, v_cache, cos_half, sin_half, key_weights))
    return _backend.paged_append(q, k, v, k_cache, v_cache, page_table, cu_seqlens, seqlens_k, None, q_weight, k_weight, cos_half, sin_half, positions, eps,
                                 key_weights, key_positions, k_scales, v_scales)


def flash_attn_paged_func(q, k_cache, v_cache, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale=None, causal=True,
                          return_softmax_lse=False, k_scales=None, v_scales=None):
    """Attention of the new tokens q (total, nheads, headdim) over their sequences' pages; nheads is a multiple of nheads_k, and query head h attends with
    key head h // (nheads // nheads_k).  causal: a sequence's last new token sees all its keys, the one before it one less, and so on (the new tokens'
    own keys are in the cache); a token that sees no key gives zeros.  max_seqlen_q, max_seqlen_k: at least the longest of each.  k_scales, v_scales: of a cache in 8 bits.
    Returns out (total, nheads, headdim), or (out, softmax_lse), softmax_lse (batch, nheads, max_seqlen_q rounded up to 16) fp32, -inf for a token
    that sees no key.  Rows of out behind the last sequence hold nothing."""
    done = _backend.passes().paged_fwd(q, k_cache, v_cache, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal,
                                       return_softmax_lse, k_scales, v_scales)
    if done is not None:
        return done
    _inference(q, k_cache, v_cache)
    scale = q.shape[-1] ** (-0.5) if softmax_scale is None else softmax_scale
    r = _backend.paged_fwd(q, k_cache, v_cache, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, scale, causal, return_softmax_lse,
                           k_scales=k_scales, v_scales=v_scales)
    return (r[0], r[1]) if return_softmax_lse else r[0]


def flash_attn_paged_prefix_func(q, k_cache, v_cache, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, cu_groups, prefix_lens, max_prefix_len,
                                 softmax_scale=None, causal=True, return_softmax_lse=False, k_scales=None, v_scales=None):
    """flash_attn_paged_func for sequences that begin with the same keys (a system prompt, several answers to one question), which are read once for all of them.
    cu_groups (groups + 1,) int32: group g is the sequences cu_groups[g] .. cu_groups[g + 1] - 1, from 0 to the batch's end.  prefix_lens (batch,) int32: how many
    leading keys the sequences of a group have in the same pages - one number within a group, 0 for nothing, and no more keys than the sequence's first new token sees.
    Whole pages count; what is left of a prefix is read as each sequence's own.  max_prefix_len: at least the longest; prefixes count up to it.  As always each sequence
    lists all its pages, and its result is that of flash_attn_paged_func, rounded elsewhere.  (Groups that do not hold all sequences, or whose sequences differ in what they are
    said to share, get results of no use; nothing outside the tensors is read or written.)  Sharing pays for long prefixes, many sequences and a few new tokens; where it does
    not, by the sizes that the host knows, every sequence reads its own."""
    done = _backend.passes().paged_fwd(q, k_cache, v_cache, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal,
                                       return_softmax_lse, k_scales, v_scales, cu_groups, prefix_lens, max_prefix_len)
    if done is not None:
        return done
    _inference(q, k_cache, v_cache)
    scale = q.shape[-1] ** (-0.5) if softmax_scale is None else softmax_scale
    if cu_groups is None or prefix_lens is None:
        raise RuntimeError("cu_groups and prefix_lens say which sequences share what: flash_attn_paged_func takes those that share nothing")
    r = _backend.paged_fwd(q, k_cache, v_cache, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, scale, causal, return_softmax_lse,
                           k_scales=k_scales, v_scales=v_scales, cu_groups=cu_groups, prefix_lens=prefix_lens, max_prefix_len=max_prefix_len)
    return (r[0], r[1]) if return_softmax_lse else r[0]


def paged_read_func(k_cache, v_cache, page_table, cu_seqlens, seqlens_k, total, k_scales=None, v_scales=None, dtype=None):
    """The keys and values that the cache holds, packed: the counterpart of paged_append_func.  Row i of sequence b's cu_seqlens[b + 1] - cu_seqlens[b] rows is slot
    seqlens_k[b] - (its rows) + i, so cu_seqlens made of seqlens_k gives whole sequences, and that of the last step what the step stored.  total: rows of the results
    (total, nheads_k, headdim), cu_seqlens' last entry or more.  dtype: the cache's; for a cache in 8 bits (k_scales, v_scales) fp16 or bf16, whichever it was made from:
    nothing is rounded.  Rows that stand for no slot are zeros.  Returns (k, v)."""
    if dtype is None and k_scales is None:
        dtype = k_cache.dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("keys and values are read as fp16 or bf16 (dtype), the one that they came from")
    done = _backend.passes().paged_read(k_cache, v_cache, page_table, cu_seqlens, seqlens_k, total, 0 if dtype == torch.float16 else 1, k_scales, v_scales)
    if done is not None:
        return done
    _inference(k_cache, v_cache)
    return _backend.paged_read(k_cache, v_cache, page_table, cu_seqlens, seqlens_k, total, dtype, k_scales, v_scales)


def paged_key_weights_func(q, softmax_lse, k_cache, key_weights, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale=None,
                           causal=True):
    """Adds to key_weights (pages, nheads_k, page size) fp32 what every key has received of the new tokens' attention: the sum of its probabilities
    over the tokens and over the query heads of its group.  q and softmax_lse: those of flash_attn_paged_func over the same cache.  In place; returns
    key_weights."""
    if _backend.passes().paged_key_weights(q, softmax_lse, k_cache, key_weights, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale,
                                           causal):
        return key_weights
    _inference(q, k_cache, constants=(softmax_lse, key_weights))
    scale = q.shape[-1] ** (-0.5) if softmax_scale is None else softmax_scale
    return _backend.paged_key_weights(q, softmax_lse, k_cache, key_weights, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, scale, causal)


def paged_evict_func(k_cache, v_cache, key_weights, key_positions, page_table, seqlens_k, next_positions, budget, recent, max_seqlen_k):
    """Cuts every sequence's cache to `budget` keys a head, in place, and returns the new lengths min(seqlens_k, budget).  Of a longer sequence stay
    the keys whose position is at least next_positions[b] - recent, and then those with the largest key_weights (NaN counts as -inf; ties: the lower
    slot; of more than `budget` recent keys those in the lowest slots stay, whatever their positions).  Each key head chooses for itself; a kept key
    from behind the budget takes the place, and the weight and position, of one that goes.  Slots from `budget` on are left as they were.  next_positions: (batch,) int32, the position that each sequence's next token would have."""
    done = _backend.passes().paged_evict(k_cache, v_cache, key_weights, key_positions, page_table, seqlens_k, next_positions, budget, recent, max_seqlen_k)
    if done is not None:
        return done
    _inference(k_cache, v_cache, constants=(key_weights,))
    return _backend.paged_evict(k_cache, v_cache, key_weights, key_positions, page_table, seqlens_k, next_positions, budget, recent, max_seqlen_k)


class PagedKVCache:
    """A pool of pages for the keys and values of a model's layers, and the book of which pages each sequence has.  All layers of a sequence use the
    same page numbers, each in a pool of its own.

        cache = PagedKVCache(layers, pages, page_size, nheads_k, headdim, dtype, device)
        a, b = cache.add(), cache.add()
        step = cache.step([a, b], [prompt_a, prompt_b])            # numbers of new tokens; then, layer by layer:
        q = step.append(layer, q, k, v, ...)                       # packed (total, heads, headdim) tensors of the new tokens
        out = step.attend(layer, q)
        cache.evict([a, b], budget, recent)                        # if made with key_weights=True
        c = cache.fork(b, 512)                                     # begins with b's first 512 tokens
        k, v, cu_seqlens = cache.read(layer, [b, c])               # what the cache holds of them, packed
        cache.remove(a)

    dtype: the model's.  store_dtype=torch.float8_e4m3fn: pages in 8 bits, half the memory and, at headdim 128, 0.57 of the time of a decode step that is bound by reading them
    (0.6 at 64, 0.9 at 32, more at 16; not with key_weights).  A fork shares the whole pages of what it begins with; the steps of sequences that share them, named one after the other, read them once for all
    where that pays (flash_attn_paged_prefix_func).

    A page holds a head's tokens one after the other.  Everything is enqueued on the current stream in the order of the calls; a removed sequence's pages may be
    given to another at once, so steps of one cache belong on one stream."""

    def __init__(self, layers, pages, page_size, nheads_k, headdim, dtype=torch.float16, device=None, key_weights=False, store_dtype=None):
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise RuntimeError("page_size must be a power of two from 16 to 1024, got %d" % page_size)
        if layers < 1 or pages < 1 or nheads_k < 1 or headdim not in (16, 32, 64, 128) or dtype not in (torch.float16, torch.bfloat16):
            raise RuntimeError("layers, pages and nheads_k must be positive, headdim 16, 32, 64 or 128, dtype fp16 or bf16")
        if store_dtype not in (None, dtype, torch.float8_e4m3fn):
            raise RuntimeError("store_dtype must be the dtype or float8_e4m3fn")
        eight = store_dtype == torch.float8_e4m3fn
        if eight and key_weights:
            raise RuntimeError("key_weights, and the eviction that goes by them, are those of a cache in 16 bits")
        self.page_size, self.dtype = page_size, dtype
        shape = (layers, pages, nheads_k, page_size, headdim)
        device = torch.device("cuda" if device is None else device)
        # (zeros: entries of a page table that are no pages are read as the first or last one)
        self._k, self._v = (torch.zeros(shape, dtype=torch.uint8 if eight else dtype, device=device).transpose(2, 3) for _ in range(2))
        self._scales = None
        if eight:
            self._k, self._v = (t.view(torch.float8_e4m3fn) for t in (self._k, self._v))
            self._scales = [torch.zeros(shape[:4], dtype=torch.uint8, device=device) for _ in range(2)]
        self.key_weights = torch.zeros(shape[:4], dtype=torch.float32, device=device) if key_weights else None
        self.key_positions = torch.zeros(shape[:4], dtype=torch.int32, device=device) if key_weights else None
        self.device = self._k.device
        self._free = list(range(pages - 1, -1, -1))
        self._pages, self._len, self._seen = {}, {}, {}
        self._shared = {}  # sequence: its leading pages that others may list, too
        self._users = {}   # page: how many sequences list it, if more than one has
        self._next_id = 0

    def layer(self, i):
        """(k_cache, v_cache) of layer i: (pages, page size, nheads_k, headdim)"""
        return self._k[i], self._v[i]

    def scales(self, i):
        """k_scales and v_scales of layer i, as the functions' keywords; {} for a cache in 16 bits"""
        return {} if self._scales is None else dict(k_scales=self._scales[0][i], v_scales=self._scales[1][i])

    def add(self):
        """A new, empty sequence."""
        seq, self._next_id = self._next_id, self._next_id + 1
        self._pages[seq], self._len[seq], self._seen[seq] = array("i"), 0, 0
        return seq

    def fork(self, seq, tokens=None):
        """A new sequence that begins with the first `tokens` tokens of seq (all of them).  It lists the same pages for them; a last page that they do not fill is
        copied, in every layer.  Between steps: what the last one made room for has been stored by all layers."""
        self._not_under_capture("a fork")
        self._book([seq])
        if self.key_weights is not None:
            raise RuntimeError("a cache with key_weights counts what a sequence's keys receive: its pages are not shared")
        tokens = self._len[seq] if tokens is None else int(tokens)
        if tokens < 0 or tokens > self._len[seq]:
            raise RuntimeError("the sequence has %d tokens, not %d" % (self._len[seq], tokens))
        whole, rest = divmod(tokens, self.page_size)
        if rest and not self._free:
            raise RuntimeError("the cache has no free page for the tokens behind the shared ones")
        new = self.add()
        pages = self._pages[new]
        pages.extend(self._pages[seq][:whole])
        for page in pages:
            self._users[page] = self._users.get(page, 1) + 1
        for s in (seq, new) if whole else ():
            self._shared[s] = max(self._shared.get(s, 0), whole)
        if rest:
            page, old = self._free.pop(), self._pages[seq][whole]
            for t in (self._k.view(torch.uint8), self._v.view(torch.uint8), *self._scales) if self._scales else (self._k, self._v):
                t[:, page].copy_(t[:, old])
            pages.append(page)
        self._len[new] = self._seen[new] = tokens
        return new

    def read(self, layer, seqs):
        """(k, v, cu_seqlens): what the cache holds of the sequences in a layer, packed (total, nheads_k, headdim) one sequence after the other"""
        self._not_under_capture("reading whole sequences")
        seqs = list(seqs)
        self._book(seqs)
        ends = [0]
        for s in seqs:
            ends.append(ends[-1] + self._len[s])
        table, lens, _, cu = self._tables(seqs, ends)
        with torch.no_grad():
            return (*paged_read_func(*self.layer(layer), table, cu, lens, ends[-1], dtype=self.dtype, **self.scales(layer)), cu)

    def remove(self, seq):
        pages, shared = self._pages.pop(seq), self._shared.pop(seq, 0)
        for page in reversed(pages):
            if shared and page in self._users:
                self._users[page] -= 1
                if self._users[page] == 1:
                    del self._users[page]
            else:
                self._free.append(page)
        del self._len[seq], self._seen[seq]

    def _groups(self, seqs):
        """Runs of sequences that begin with the same pages: (where each begins and the end, the tokens shared by each sequence's run); None if there is none"""
        cu, lens = [0], []
        for i, s in enumerate(seqs):
            common = 0
            if i and self._shared.get(s) and self._shared.get(seqs[i - 1]):
                a, b = self._pages[s], self._pages[seqs[i - 1]]
                lo, hi = 0, min(self._shared[s], self._shared[seqs[i - 1]])
                if a[:hi] == b[:hi]:
                    lo = hi
                while lo < hi:  # (the longest equal beginning)
                    mid = (lo + hi + 1) // 2
                    lo, hi = (mid, hi) if a[:mid] == b[:mid] else (lo, mid - 1)
                common = lo
            run = i - cu[-1]
            common = common if run == 1 else min(common, lens[-1]) if lens else 0
            if common and run * common >= (run - 1) * lens[-1]:  # (as many pages saved as by the shorter run, at least)
                lens[cu[-1]:] = [common] * (run + 1)
            else:
                if i:
                    cu.append(i)
                lens.append(0)
        return (cu + [len(seqs)], [n * self.page_size for n in lens]) if any(lens) else None

    def length(self, seq):
        """Tokens of the sequence that the cache holds"""
        return self._len[seq]

    def free_pages(self):
        return len(self._free)

    def _book(self, seqs):
        if not seqs or len(set(seqs)) != len(seqs) or any(s not in self._pages for s in seqs):
            raise RuntimeError("a step takes different sequences of this cache, one at least")

    def _device_ints(self, *lists):
        """int32 tensors on the device, by way of one copy"""
        flat = array("i")
        for l in lists:
            flat.extend(l)
        flat = torch.frombuffer(flat, dtype=torch.int32)
        flat = flat.pin_memory().to(self.device, non_blocking=True) if self.device.type == "cuda" else flat.clone()
        out, at = [], 0
        for l in lists:
            out.append(flat[at:at + len(l)])
            at += len(l)
        return out

    def _not_under_capture(self, what):
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("%s is made of the host's numbers, which a graph's replays would not find again: not while a stream is captured" % what)

    def step(self, seqs, new_tokens):
        """Makes room for new_tokens[i] further tokens of seqs[i] and returns the PagedStep that stores them and attends."""
        self._not_under_capture("a step")
        seqs, new = list(seqs), [int(n) for n in new_tokens]
        self._book(seqs)
        if len(new) != len(seqs) or min(new) < 0 or sum(new) == 0:
            raise RuntimeError("a number of new tokens for each sequence, one token at least")
        need = {s: -(-(self._len[s] + n) // self.page_size) - len(self._pages[s]) for s, n in zip(seqs, new)}
        if sum(max(0, n) for n in need.values()) > len(self._free):
            raise RuntimeError("the cache has %d free pages, the step needs %d" % (len(self._free), sum(max(0, n) for n in need.values())))
        positions = []
        for s, n in zip(seqs, new):
            self._pages[s].extend(self._free.pop() for _ in range(max(0, need[s])))
            positions.extend(range(self._seen[s], self._seen[s] + n))
            self._len[s] += n
            self._seen[s] += n
        return PagedStep(self, seqs, new, positions)

    def evict(self, seqs, budget, recent):
        """Cuts the sequences to `budget` tokens a key head in every layer, the `recent` newest among them (paged_evict_func); pages that become empty are free
        again."""
        self._not_under_capture("an eviction of whole sequences")
        seqs = list(seqs)
        self._book(seqs)
        if self.key_weights is None:
            raise RuntimeError("eviction goes by key_weights: make the cache with key_weights=True")
        if budget < 1 or recent < 0 or recent > budget:  # (of more recent keys than the budget the lowest slots' would stay, not the newest)
            raise RuntimeError("budget must be positive, recent not negative and at most the budget")
        longest = max(self._len[s] for s in seqs)
        if longest <= budget:
            return
        table, lens, seen = self._tables(seqs)
        with torch.no_grad():
            for i in range(self._k.shape[0]):
                paged_evict_func(*self.layer(i), self.key_weights[i], self.key_positions[i], table, lens, seen, budget, recent, longest)
        for s in seqs:
            self._len[s] = min(self._len[s], budget)
            keep = -(-self._len[s] // self.page_size)
            self._free.extend(reversed(self._pages[s][keep:]))
            del self._pages[s][keep:]

    def _tables(self, seqs, *more):
        cols = max(1, max(len(self._pages[s]) for s in seqs))
        rows = array("i")
        for s in seqs:
            rows.extend(self._pages[s])
            rows.extend(array("i", [-1]) * (cols - len(self._pages[s])))
        table, lens, seen, *rest = self._device_ints(rows, [self._len[s] for s in seqs], [self._seen[s] for s in seqs], *more)
        return (table.view(len(seqs), cols), lens, seen, *rest)


class PagedStep:
    """New tokens of some sequences of a PagedKVCache: the tensors that the functions above take.  The layers' calls are made while the step is the
    cache's last one for its sequences."""

    def __init__(self, cache, seqs, new, positions):
        self.cache = cache
        ends, at = [0], 0
        for n in new:
            at += n
            ends.append(at)
        groups = cache._groups(seqs) if cache._users else None
        self.page_table, self.seqlens_k, _, self.cu_seqlens, self.positions, *rest = cache._tables(seqs, ends, positions, *(groups or ()))
        self.total, self.max_seqlen_q = at, max(new)
        self.max_seqlen_k = max(cache._len[s] for s in seqs)
        self.max_position = max(cache._seen[s] for s, n in zip(seqs, new) if n > 0)  # table rows that the new tokens' positions reach
        self.prefix = ()  # of runs of sequences that begin with the same pages: cu_groups, prefix_lens, max_prefix_len
        if groups is not None:
            self.prefix = (*rest, max(groups[1]))

    def _own(self, t):
        if t.shape[0] != self.total:
            raise RuntimeError("the step has %d tokens, not %d" % (self.total, t.shape[0]))
        if t.dtype != self.cache.dtype:  # (what rows in 8 bits stand for is exact in the dtype that they came from)
            raise RuntimeError("the cache was made for %s, not %s" % (self.cache.dtype, t.dtype))

    def append(self, layer, q, k, v, **norm_and_rotary):
        """paged_append_func into the layer's pages (q_weight, k_weight, cos_half, sin_half, eps); tokens are turned by their numbers in their sequences,
        which go on where an eviction has cut the cache: tables of max_position rows at least."""
        c = self.cache
        weights = (None, None) if c.key_weights is None else (c.key_weights[layer], c.key_positions[layer])
        self._own(k)
        cos = norm_and_rotary.get("cos_half")
        if cos is not None and cos.shape[0] < self.max_position:  # (the kernels clamp positions to the tables: the keys would stay turned wrongly)
            raise RuntimeError("the tables have %d rows, the step's tokens positions up to %d" % (cos.shape[0], self.max_position - 1))
        return paged_append_func(q, k, v, *c.layer(layer), self.page_table, self.cu_seqlens, self.seqlens_k,
                                 positions=self.positions, key_weights=weights[0], key_positions=weights[1],
                                 **c.scales(layer), **norm_and_rotary)

    def attend(self, layer, q, softmax_scale=None):
        """flash_attn_paged_func over the layer's pages, causal (flash_attn_paged_prefix_func where sequences share pages); a cache with key_weights counts what
        its keys receive"""
        self._own(q)
        c = self.cache
        k, v = c.layer(layer)
        where = (self.page_table, self.cu_seqlens, self.seqlens_k, self.max_seqlen_q, self.max_seqlen_k, softmax_scale)
        if self.prefix:
            return flash_attn_paged_prefix_func(q, k, v, *where[:-1], *self.prefix, softmax_scale, **c.scales(layer))
        if c.key_weights is None:
            return flash_attn_paged_func(q, k, v, *where, **c.scales(layer))
        out, lse = flash_attn_paged_func(q, k, v, *where, return_softmax_lse=True)
        paged_key_weights_func(q, lse, k, c.key_weights[layer], *where)
        return out
