"""The operators together, as a server uses them that answers one prompt several times: the prompt's cells in fp16, every answer's own in 8
bits; a step writes the new rows (store_q8), attends (shared_attention_q8), draws tokens (sample) and reports them (token_logprobs).

Each step's attention is checked against the formula in 64 bits over the prompt's cells and the rows so far as the format in 64 bits
rounds them (tolerance: test_gpu_shared_attn.py); a captured step replays over all of them and gives the eager run's bits."""
import numpy as np
import pytest

import q8_cache as Q
from test_gpu_paged_attn import formula, make

pytestmark = pytest.mark.gpu

H, KV, HD, B, V, PROMPT, STEPS = 8, 2, 64, 5, 500, 75, 36


class Server:
    """What lives on the device: the caches, the answers' pages and lengths, the step's inputs and outputs."""

    def __init__(self, torch, dev, seed):
        rng = np.random.default_rng(seed)
        self.x = make(torch, dev, rng, H, KV, HD, [PROMPT])
        d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
        self.pages = rng.permutation(2 * B + 3)[:2 * B].reshape(B, 2)  # of each answer
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)
        self.length, self.lens, self.first, self.blocks = i32([PROMPT]), i32([0] * B), i32([2 * b for b in range(B)]), i32(self.pages.ravel())
        self.cache = torch.full((2 * B + 3, KV, 68 * HD), 255, dtype=torch.uint8, device=dev)  # scales of NaN
        self.head = d(rng.standard_normal((H * HD, V)).astype(np.float32))
        self.q, self.rows = torch.zeros(B, H, HD, dtype=torch.float16, device=dev), torch.zeros(B, 2, KV, HD, device=dev)
        self.cells, self.u = i32([0] * B), torch.zeros(B, device=dev)
        self.feed = [(d((2 * rng.standard_normal((B, H, HD))).astype(np.float16)), d(rng.standard_normal((B, 2, KV, HD)).astype(np.float32)),
                      d(rng.random(B).astype(np.float32))) for _ in range(STEPS)]

    def next(self, torch, step):
        """The step's inputs; answer b starts b steps late (its row goes nowhere until then)."""
        q, rows, u = self.feed[step]
        self.q.copy_(q)
        self.rows.copy_(rows)
        self.u.copy_(u)
        at = [step - b for b in range(B)]
        self.cells.copy_(torch.tensor([-1 if i < 0 else int(self.pages[b, i // 32]) * 32 + i % 32 for b, i in enumerate(at)], dtype=torch.int32))
        self.lens.copy_(torch.tensor([max(0, i + 1) for i in at], dtype=torch.int32))

    def step(self, lstk):
        lstk.store_q8(self.cache, self.rows[:, 0], self.rows[:, 1], self.cells)
        prefix = lstk.SharedPrefix(self.x["kc"], self.x["vc"], self.length, self.x["blocks"], PROMPT)
        out = lstk.shared_attention_q8(self.q, prefix, self.cache, self.lens, self.first, self.blocks, 64)
        logits = (out.float().reshape(B, H * HD, 1) * self.head).sum(1)
        token, prob = lstk.sample(logits, self.u)
        return (out, logits, token, prob) + lstk.token_logprobs(logits, token, n_top=3)


def test_answers(lstk, dev):
    import torch
    s = Server(torch, dev, 1)
    eager = []
    so_far = [[] for _ in range(B)]
    for step in range(STEPS):
        s.next(torch, step)
        out, logits, token, prob, lp, entropy, ids, at = r = s.step(lstk)
        eager.append([t.clone() for t in r])
        o, rows, q = out.float().cpu().numpy().astype(np.float64), s.feed[step][1].cpu().numpy(), s.q.cpu().numpy()
        for b in range(B):
            if step >= b:
                so_far[b].append([Q.values(*Q.quantise(rows[b, i])) for i in range(2)])
            own = np.array(so_far[b]).reshape(-1, 2, KV, HD)
            cells = s.x["rows"][0]
            K, W = (np.concatenate([s.x[n][:, cells].astype(np.float64), own[:, i].transpose(1, 0, 2)], 1) for i, n in ((0, "K"), (1, "V")))
            want, tol = formula(q[b], K, W, np.arange(K.shape[1]), HD ** -0.5)
            assert (np.abs(o[b] - want) <= tol).all(), (step, b)
        # the drawn token's probability, twice: sample's is w over a sum of weights good to 2e-14, token_logprobs' off by (75 + 2 D) 2^-24
        assert (lp.double() - prob.double().log()).abs().max() <= 4e-5
        assert (at[:, 0] >= lp).all() and torch.equal(ids[:, 0].long(), logits.argmax(1))
    # the same answers by a captured step
    s = Server(torch, dev, 1)
    s.next(torch, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.step(lstk)  # (torch's own first call of each kind is not captured)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = s.step(lstk)
    for step in range(STEPS):
        s.next(torch, step)
        g.replay()
        for a, b in zip(r, eager[step]):
            assert torch.equal(a, b), step
        if step % 5 == 0:
            torch.cuda.synchronize()
            lstk.token_logprobs(eager[step][1], eager[step][2], n_top=3)  # eager work between
