"""Requests served step by step over a Forward's paged cache, with all that a step needs on the device: the new tokens' places and
pages (hq_batch_plan_ex), their embeddings (hq_embed_ex), the layers with the requests' adapters, the classifier for each
request's last token, and the tokens drawn from the logits (hq_sample_ex).  Nothing comes back to the host inside a step: a step
can be captured into a graph and replayed on new contents of its tensors (`longest` is the captured step's).  A Serving has its Forward to itself: the pages that it gives out are the Forward's.
"""
from . import check, library
from .cache import Batch, Pool
from .forward import on_its_device


class Serving:
    """`forward.sequences` places for requests, each with its pages and its settings (tensors on the device that a caller fills
    between steps): which (its adapter, -1: none), temperature, top_k, top_p, min_p as hq_sample_ex takes them; lengths: the positions
    that each place holds; missing: the pages that the last step lacked (its requests' answers are then without what these would
    have held); chance: the drawn tokens' chances."""

    def __init__(self, forward, adapters=None):
        torch, n, device = forward.torch, forward.sequences, forward.y.device
        if n > forward.tokens:
            raise ValueError(f"refused: {n} places over steps of {forward.tokens} tokens")
        if adapters is not None:  # (a step would refuse them with its places and pages taken)
            forward.adapters_fit(adapters, forward.tokens)
        self.forward, self.torch, self.lib, self.adapters, self.device = forward, torch, library(), adapters, device

        def ints(count, value=0):
            return torch.full((count,), value, dtype=torch.int32, device=device)

        def floats(count, value):
            return torch.full((count,), value, dtype=torch.float32, device=device)

        self.starts, self.lengths, self.which, self.top_k = ints(n + 1), ints(n), ints(n, -1), ints(n)
        self.temperature, self.top_p, self.min_p = floats(n, 1.0), floats(n, 1.0), floats(n, 0.0)
        self.table = torch.full((n, forward.width), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(forward.pages - 1, -1, -1, dtype=torch.int32, device=device)  # (page 0 is on top)
        self.left, self.missing = ints(1, forward.pages), ints(1)
        self.pool = Pool(self.free.data_ptr(), self.left.data_ptr(), self.left.data_ptr(), self.missing.data_ptr(), forward.pages,
                         forward.page)
        self.position = ints(forward.tokens)
        self.x = torch.empty_like(forward.y)
        self.scores = torch.empty(n, forward.ck.shape.vocab, dtype=torch.float32, device=device)
        self.tokens, self.chance = ints(n, -1), floats(n, 0.0)
        self.work = torch.empty(self.lib.hq_sample_work_bytes(n, forward.ck.shape.vocab), dtype=torch.uint8, device=device)

    @on_its_device
    def step(self, ids, fresh, u, longest=0):
        """ids (int32): the step's new tokens, place after place; fresh (int32): how many each place has of them; u (float32): a
        number of [0, 1) a place; longest: the most that one has (0: not known).  Returns each place's next token (int32, a buffer
        of this object's): -1 where it has no new ones."""
        torch, f, n = self.torch, self.forward, self.forward.sequences
        count = ids.shape[0]
        for name, t, kind, shape in (("ids", ids, torch.int32, (count,)), ("fresh", fresh, torch.int32, (n,)),
                                     ("u", u, torch.float32, (n,))):
            if t.dtype != kind or tuple(t.shape) != shape or not t.is_contiguous() or t.device != self.x.device:
                raise ValueError(f"refused: {name} is {tuple(t.shape)} of {t.dtype} on {t.device}, not {shape} of {kind} on "
                                 f"{self.x.device} in one piece")
        if not 0 < count <= f.tokens:
            raise ValueError(f"refused: {count} tokens for steps of {f.tokens}")
        stream = torch.cuda.current_stream().cuda_stream
        batch = Batch(self.starts.data_ptr(), self.lengths.data_ptr(), self.table.data_ptr(), n, count, longest, f.width)
        at, x = self.position[:count], self.x[:count]
        check(self.lib.hq_batch_plan_ex(batch, self.pool, self.lengths.data_ptr(), fresh.data_ptr(), 0, at.data_ptr(), 0, stream))
        f.embed(ids, x)
        y = f.step(x, self.starts, self.lengths, self.table, longest, at, self.adapters,
                   None if self.adapters is None else self.which)
        last = (self.starts[1:] - 1).clamp(0, count - 1)
        rows = y.index_select(0, last)
        f.logits(rows, self.scores)
        check(self.lib.hq_sample_ex(self.tokens.data_ptr(), self.chance.data_ptr(), self.scores.data_ptr(), u.data_ptr(),
                                    self.temperature.data_ptr(), self.top_k.data_ptr(), self.top_p.data_ptr(),
                                    self.min_p.data_ptr(), n, self.scores.shape[1], 4 * self.scores.shape[1],
                                    self.work.data_ptr(), self.work.numel(), stream))
        self.tokens.masked_fill_(self.starts[1:] == self.starts[:-1], -1)
        return self.tokens

    @on_its_device
    def finish(self, done):
        """done (bool, on the device, a place each): these requests end; their pages go back to the pool, their places are empty"""
        torch, f = self.torch, self.forward
        if done.dtype != torch.bool or tuple(done.shape) != (f.sequences,) or done.device != self.x.device:
            raise ValueError(f"refused: done is {tuple(done.shape)} of {done.dtype} on {done.device}")
        to = done.int() * f.width
        check(self.lib.hq_pages_give_ex(self.pool, self.table.data_ptr(), f.sequences, f.width, 0, to.data_ptr(),
                                        torch.cuda.current_stream().cuda_stream))
        self.lengths.masked_fill_(done, 0)
