"""From hidden states to search results: trains a small vocabulary head and searches with what it answers.

Texts are runs of word ids; a fixed table of word vectors and a moving average stand in for an encoder's body, and a
linear layer and the vocabulary matrix above it are trained with the library's operators:

  embed_tokens   the words' vectors
  vocab_loss     the word at a position that was hidden from the input
  distill_loss   a teacher's top logits at every position (here: a sharper head with the true word vectors)
  term_weights   texts as sparse vectors: queries against their documents, with a penalty on active terms

Then the documents' term weights become an index, and the queries' are searched on it; and again with layer and vocabulary
in 8 bits, as they would be served (quantize_rows, int8_linear, term_weights).

    python gpu-sparse_amd/examples/train_and_search.py --steps 60
"""
import argparse
import os
import sys

import numpy as np
import torch

_PKG = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

import gpusparse as gs  # noqa: E402

DEV = "cuda:0"


class Texts:
    """Documents of a few topics, queries cut out of them, and hidden states for both."""

    def __init__(self, n_docs, vocab, dim, length, seed=0):
        self.gen = torch.Generator(device=DEV)
        self.gen.manual_seed(seed)
        self.vocab, self.dim = vocab, dim
        self.words = torch.randn((vocab, dim), generator=self.gen, device=DEV)
        topics = torch.rand((32, vocab), generator=self.gen, device=DEV) ** 12
        of = torch.randint(0, 32, (n_docs,), generator=self.gen, device=DEV)
        self.docs = torch.multinomial(topics[of] + 1e-4, length, generator=self.gen)
        lens = torch.randint(length // 2, length + 1, (n_docs, 1), generator=self.gen, device=DEV)
        self.doc_mask = torch.arange(length, device=DEV)[None] < lens
        pick = torch.rand((n_docs, length // 2), generator=self.gen, device=DEV).argsort(dim=1)[:, : max(3, length // 8)]
        self.queries = self.docs.gather(1, pick)

    def hidden(self, ids, hide=None):
        """[texts, length, dim], each of unit variance: word vectors with half of their neighbours', hidden words as zeros."""
        x = gs.embed_tokens(ids, self.words)
        if hide is not None:
            x = x.masked_fill(hide[:, :, None], 0.0)
        return torch.nn.functional.layer_norm(x + 0.5 * (x.roll(1, dims=1) + x.roll(-1, dims=1)), (self.dim,))


class Head(torch.nn.Module):
    def __init__(self, vocab, dim, dtype):
        super().__init__()
        gen = torch.Generator(device=DEV)
        gen.manual_seed(1)
        self.turn = torch.nn.Parameter(torch.eye(dim, device=DEV) + 0.05 * torch.randn((dim, dim), generator=gen, device=DEV))
        self.weight = torch.nn.Parameter(torch.randn((vocab, dim), generator=gen, device=DEV) / dim ** 0.5)
        self.bias = torch.nn.Parameter(torch.full((vocab,), -2.0, device=DEV))
        self.dtype = dtype

    def forward(self, x):
        return (x @ self.turn).to(self.dtype), self.weight.to(self.dtype), self.bias.to(self.dtype)


class Head8:
    """A trained head in 8 bits."""

    def __init__(self, head):
        self.turn = gs.quantize_rows(head.turn.detach().t())
        self.weight = gs.quantize_rows(head.weight.detach())
        self.bias = head.bias.detach()
        self.dtype = head.dtype

    def __call__(self, x):
        return gs.int8_linear(x, self.turn, dtype=self.dtype), self.weight, self.bias


def train(head, texts, steps, batch, top=16, log=print):
    opt = torch.optim.Adam(head.parameters(), lr=2e-3)
    teacher = texts.words / texts.dim ** 0.5
    first = last = None
    for step in range(steps):
        rows = torch.randint(0, texts.docs.shape[0], (batch,), generator=texts.gen, device=DEV)
        ids, mask = texts.docs[rows], texts.doc_mask[rows]
        hide = (torch.rand(ids.shape, generator=texts.gen, device=DEV) < 0.15) & mask
        h, w, b = head(texts.hidden(ids, hide))
        targets = torch.where(hide, ids, -100)
        masked = gs.vocab_loss(h, w, targets, b)

        full = texts.hidden(ids)
        z, tid = gs.topk_rows((full.reshape(-1, texts.dim) @ teacher.t()).contiguous(), top)
        tid = torch.where(mask.reshape(-1, 1), tid, -1).view(*ids.shape, top)
        h, _, _ = head(full)
        taught = gs.distill_loss(h, w, tid, z.view(*ids.shape, top), b, temperature=2.0)

        d = gs.term_weights(h, w, b, mask=mask)
        hq, _, _ = head(texts.hidden(texts.queries[rows]))
        q = gs.term_weights(hq, w, b)
        match = torch.nn.functional.cross_entropy(q @ d.t(), torch.arange(batch, device=DEV))
        active = (d.abs().mean(0) ** 2).sum() + (q.abs().mean(0) ** 2).sum()

        loss = masked + 0.1 * taught + match + 1e-3 * active
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        parts = [x.item() for x in (loss, masked, taught, match)]
        first, last = first or parts, parts
        if step % 20 == 0 or step == steps - 1:
            log("step %3d  loss %.3f  masked words %.3f  teacher %.3f  match %.3f" % (step, *parts))
    return first, last


@torch.no_grad()
def search(head, texts, k=10, terms=64, batch=256):
    """Share of queries whose document is among the first k: documents indexed, queries searched."""
    h, w, b = head(texts.hidden(texts.docs[:1]))
    ptr, ind, val = [np.zeros(1, np.int64)], [], []
    for s in range(0, texts.docs.shape[0], batch):
        h, _, _ = head(texts.hidden(texts.docs[s:s + batch]))
        d = gs.term_weights(h, w, b, mask=texts.doc_mask[s:s + batch])
        at = d.nonzero()
        ptr.append(ptr[-1][-1] + (d > 0).sum(1).cumsum(0).cpu().numpy())
        ind.append(at[:, 1].int().cpu().numpy())
        val.append(d[at[:, 0], at[:, 1]].cpu().numpy())
    csr = gs.CSR(np.concatenate([p[-len(p):] for p in ptr]), np.concatenate(ind), np.concatenate(val),
                 (texts.docs.shape[0], texts.vocab))
    index = gs.build_from_csr(csr, DEV)
    found = 0
    for s in range(0, texts.queries.shape[0], batch):
        h, _, _ = head(texts.hidden(texts.queries[s:s + batch]))
        weights, ids = gs.topk_rows(gs.term_weights(h, w, b), terms)
        ids = torch.where(weights > 0, ids, -1).int()
        _, docs = gs.search(index, (ids, weights), k)
        own = torch.arange(s, s + docs.shape[0], device=DEV)
        found += int((docs == own[:, None]).any(dim=1).sum())
    return found / texts.queries.shape[0], csr.nnz / csr.shape[0]


def run(steps=60, n_docs=2000, vocab=4000, dim=128, length=48, batch=64, dtype=torch.bfloat16, log=print):
    texts = Texts(n_docs, vocab, dim, length)
    head = Head(vocab, dim, dtype)
    before, _ = search(head, texts)
    first, last = train(head, texts, steps, batch, log=log)
    after, per_doc = search(head, texts)
    after8, per_doc8 = search(Head8(head), texts)
    log("documents found among the first 10: %.3f before, %.3f after, %.3f in 8 bits; %.0f terms per document (%.0f)"
        % (before, after, after8, per_doc, per_doc8))
    return {"before": before, "after": after, "after8": after8, "first": first, "last": last, "terms_per_doc": per_doc}


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--docs", type=int, default=2000)
    ap.add_argument("--vocab", type=int, default=4000)
    a = ap.parse_args()
    run(a.steps, a.docs, a.vocab)


if __name__ == "__main__":
    main()
