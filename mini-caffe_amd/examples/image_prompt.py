"""Questions about images, answered token by token.

A network of this framework turns each image into a map of features; its cells become
tokens in front of a question's.  One attention layer with a paged cache then serves both
requests together: the prompts in one packed pass, after that a token per request and
step.  Weights are random, so the answers mean nothing; that the steps over the cache give
the tokens that a pass over the whole sequence gives is checked at the end.

    python mini-caffe_amd/examples/image_prompt.py
"""
import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import minicaffe as mc  # noqa: E402
from minicaffe import attention as A  # noqa: E402
from minicaffe import craft, zoo  # noqa: E402
from minicaffe import kernels as K  # noqa: E402
from minicaffe.base import LIB, check_mc  # noqa: E402

HEADS, HEADS_KV, DIM, WORDS = 8, 2, 64, 200
SECTIONS = [8, 12, 12]          # pairs turned by time, height and width
BLOCK, BLOCKS, WIDTH = 16, 40, 12


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def features(size, seed):
    """The last map of a small residual network, as [cells, channels], and its height and width."""
    spec, inputs = zoo.resnet50_spec(batch=1, size=size, stages=(1, 1, 1, 1), width=16, num_classes=10, bn_seed=5)
    net = mc.Net.from_buffers(craft.to_prototxt(spec, "eye"))
    craft.load_weights(net, spec)
    last = [layer["bottom"][0] for layer in spec if layer["type"] == "Pooling"][-1]
    net.mark_output(last)
    image = np.random.default_rng(seed).standard_normal((1, 3, size, size)).astype(np.float32)
    net.forward(**{name: image for name in inputs})
    grid = net.get_blob(last).data[0]
    channels, height, width = grid.shape
    cells = torch.from_numpy(grid.reshape(channels, -1).T.copy()).cuda()
    return cells / cells.std(), height, width


class Product(object):
    """top = bottom W^T on the matrix cores."""

    def __init__(self, generator, inputs, outputs):
        self.plan = K.ConvPlan(K.conv_geom(inputs, 1, 1, outputs, 1))
        self.weights = torch.randn((outputs, inputs), generator=generator, device="cuda") / math.sqrt(inputs)
        self.plan.set_weights(self.weights.data_ptr())
        self.outputs = outputs

    def __call__(self, x):
        y = torch.empty((len(x), self.outputs), device="cuda")
        self.plan.forward(len(x), x.data_ptr(), y.data_ptr())
        return y


class Model(object):
    """An embedding, one attention layer with its residual, and a classifier over the words."""

    def __init__(self, channels, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.words = torch.randn((WORDS, channels), generator=g, device="cuda")
        self.qkv = Product(g, channels, (HEADS + 2 * HEADS_KV) * DIM)
        self.out = Product(g, HEADS * DIM, channels)
        self.head = Product(g, channels, WORDS)
        self.frequencies = (1e4 ** (-torch.arange(DIM // 2, dtype=torch.float64) / (DIM // 2))).float().cuda()
        self.turn = A.rotary_geom(A.F32, HEADS, HEADS_KV, DIM, DIM, SECTIONS)
        self.geom = A.AttentionGeom(A.F32, HEADS, HEADS_KV, DIM, 1, 1 / math.sqrt(DIM))

    def queries(self, x, positions, cache=None, slots=None):
        """Turned queries and keys, and values; with a cache the keys and values go there."""
        y = self.qkv(x).view(len(x), HEADS + 2 * HEADS_KV, DIM)
        q, k, v = y[:, :HEADS], y[:, HEADS:HEADS + HEADS_KV], y[:, HEADS + HEADS_KV:]
        stored = dict(v=A.heads_of(v), cache=cache, slots=slots.data_ptr()) if cache else {}
        A.rotary(self.turn, self.frequencies.data_ptr(), positions.data_ptr(), positions.stride(0), len(x), A.heads_of(q),
                 A.heads_of(q), k=A.heads_of(k), k_out=A.heads_of(k), **stored)
        return q, k, v

    def answers(self, x, attended):
        """The likeliest word behind each token."""
        logits = self.head(x + self.out(attended.reshape(len(x), -1)))
        best = torch.empty(len(x), device="cuda")
        check_mc(LIB.mcArgMax(logits.data_ptr(), best.data_ptr(), len(x), WORDS, 1, 1, 0, None))
        return best.long()

    def prompt(self, x, positions, starts, cache=None, slots=None):
        q, k, v = self.queries(x, positions, cache, slots)
        out = torch.empty((len(x), HEADS, DIM), device="cuda")
        A.attention_packed(self.geom, A.heads_of(q), A.heads_of(k), A.heads_of(v), starts.data_ptr(), starts.data_ptr(),
                           len(starts) - 1, len(x), len(x), A.heads_of(out))
        return self.answers(x, out)

    def step(self, x, positions, starts, contexts, table, cache, slots, longest):
        q, _, _ = self.queries(x, positions, cache, slots)
        out = torch.empty((len(x), HEADS, DIM), device="cuda")
        A.attention_paged(self.geom, A.heads_of(q), cache, table.data_ptr(), WIDTH, starts.data_ptr(), contexts.data_ptr(), len(x),
                          len(x), 1, longest, A.heads_of(out))
        return self.answers(x, out)


class Server(object):
    """The cache, its blocks and the lengths of the requests, all on the GPU."""

    def __init__(self, requests):
        self.n = requests
        self.keys, self.values = (torch.zeros((BLOCKS, BLOCK, HEADS_KV, DIM), device="cuda") for _ in range(2))
        self.cache = A.PagedCache.of(self.keys, self.values)
        self.free, self.counts = ints(list(range(BLOCKS))), [ints([BLOCKS]), ints([0])]
        self.table, self.lens = ints([[-1] * WIDTH] * requests), [ints([0] * requests), ints([0] * requests)]
        self.starts, self.denied = ints([0] * (requests + 1)), ints([0])

    def reserve(self, new, tokens):
        """Room for `new` tokens of each request; returns their slots."""
        slots, positions = ints([0] * tokens), ints([0] * tokens)
        new = ints(new)
        A.cache_reserve(self.n, BLOCK, WIDTH, tokens, BLOCKS, self.lens[0].data_ptr(), new.data_ptr(), self.free.data_ptr(),
                        self.counts[0].data_ptr(), self.table.data_ptr(), self.lens[1].data_ptr(), self.starts.data_ptr(),
                        slots.data_ptr(), positions.data_ptr(), self.counts[1].data_ptr(), self.denied.data_ptr())
        self.lens.reverse()
        self.counts.reverse()
        return slots

    def release(self, finished):
        finished = ints(finished)
        A.cache_release(self.n, BLOCK, WIDTH, BLOCKS, finished.data_ptr(), self.table.data_ptr(), self.lens[0].data_ptr(),
                        self.free.data_ptr(), self.counts[0].data_ptr(), self.counts[0].data_ptr())


def prompt_positions(height, width, words):
    """An image's cells share a time and count rows and columns; the words behind count on from the larger side."""
    cell = np.arange(height * width)
    text = max(height, width) + np.arange(words)
    return np.concatenate([[0 * cell, cell // width, cell % width], [text, text, text]], axis=1)


def main(steps=8):
    mc.set_runtime_mode(1, 0)
    prompts, r = [], np.random.default_rng(1)
    model = None
    for seed, (size, words) in enumerate(((224, 9), (160, 21))):
        cells, height, width = features(size, seed)
        model = model or Model(cells.shape[1])
        question = model.words[torch.from_numpy(r.integers(0, WORDS, words)).cuda()]
        prompts.append((torch.cat([cells, question]), prompt_positions(height, width, words)))
    server = Server(len(prompts))

    lengths = [len(x) for x, _ in prompts]
    x = torch.cat([x for x, _ in prompts])
    positions = ints(np.concatenate([p for _, p in prompts], axis=1))
    slots = server.reserve(lengths, sum(lengths))
    words = model.prompt(x, positions, server.starts, server.cache, slots)[server.starts[1:].long() - 1]
    following = ints([p.max() + 1 for _, p in prompts])
    answers = [words]
    for i in range(1, steps):
        slots = server.reserve([1] * len(prompts), len(prompts))
        at = (following + (i - 1)).expand(3, -1).contiguous()
        words = model.step(model.words[words], at, server.starts, server.lens[0], server.table, server.cache, slots, max(lengths) + i)
        answers.append(words)
    answers = torch.stack(answers, 1)
    assert server.denied.item() == 0

    # the same from the whole sequences at once
    for (x, p), answer, start in zip(prompts, answers, following.tolist()):
        whole = torch.cat([x, model.words[answer[:-1]]])
        at = ints(np.concatenate([p, np.tile(start + np.arange(steps - 1), (3, 1))], axis=1))
        again = model.prompt(whole, at, ints([0, len(whole)]))[-steps:]
        assert torch.equal(again, answer), (again, answer)
        print("%d cells and words -> words %s" % (len(x), " ".join(map(str, answer.tolist()))))
    server.release([1] * len(prompts))
    torch.cuda.synchronize()
    assert server.counts[0].item() == BLOCKS and sorted(server.free.tolist()) == list(range(BLOCKS))
    return answers


if __name__ == "__main__":
    main()
