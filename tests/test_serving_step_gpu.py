"""A server's steps made of the library's calls alone: pages taken, a norm, projections with 4-bit weights, keys into the cache, attention over it, the projection
back, the norm after the block with its gate and residual and the one before the next; forks of a prompt, slots that leave, a compaction in between.

Every call is compared with its definition in 64 bits on the inputs that it had (its own errors, not those of the calls before it), with the
tolerances of the operators' own tests; pages and lengths with the lists'."""
import pytest
import torch

from pages_helpers import Device, Model
from paged_helpers import attention_ref
from test_block_norm_gpu import check as check_norm, reference as norm_reference
from test_w4_gpu import check as check_w4, make, reference as w4_reference

pytestmark = pytest.mark.gpu

H, H_KV, D_H, PAGE, SLOTS, WIDTH, PAGES = 8, 2, 64, 16, 6, 8, 40
D = H * D_H
QKV = (H + 2 * H_KV) * D_H


class Layer:
    def __init__(self, pkg, seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.qkv, self.out = make(1, D, QKV, 64, True, seed)[1:], make(1, D, D, 128, False, seed + 1)[1:]
        self.w_qkv, self.w_out = pkg.w4_weight(*self.qkv), pkg.w4_weight(*self.out)
        vector = lambda: (1 + 0.1 * torch.randn(D, generator=gen, device="cuda")).half()  # noqa: E731
        self.before, self.after, self.gate = vector(), vector(), vector().reshape(1, D)


def step(pkg, dev, layers, x, starts, new, max_q, stream=None):
    """One step of all layers over the pool's first cache (each layer has its own pool of pages): what each call had and gave."""
    rows = x.shape[0]
    seen = []
    first = pkg.block_norm_params(D, eps=1e-5)
    between = pkg.block_norm_params(D, eps=1e-5, post=True, gate=pkg.GATE_SIGMOID, residual_scale=0.875, block_scale=0.5)
    h = torch.empty(rows, D, dtype=torch.float16, device="cuda")
    pkg.block_norm(x, None, None, h, rows, first, pre_w=layers[0].before, stream=stream)
    seen.append(("norm", first, (x.clone(), None, None, None, None, layers[0].before, None), None, h.clone()))
    for n, layer in enumerate(layers):
        qkv, o, y = (torch.empty(rows, w, dtype=torch.float16, device="cuda") for w in (QKV, D, D))
        pkg.project_w4(h, layer.w_qkv, qkv, rows, stream=stream)
        seen.append(("w4", layer.qkv, h.clone(), qkv.clone()))
        batch = pkg.paged_batch(starts, dev[n].kv, dev[n].pages, rows, max_q, WIDTH * PAGE)
        q, k, v = qkv, qkv[:, D:], qkv[:, D + H_KV * D_H:]
        pkg.cache_write(k, v, dev[n].cache, batch, stream=stream, head_stride=D_H, token_stride=QKV)
        ap = pkg.paged_attention_params(H, D_H, q_head_stride=D_H, q_token_stride=QKV)
        size = pkg.paged_attention_workspace(dev[n].cache, batch, ap)
        pkg.paged_attention(q, o, dev[n].cache, batch, ap, torch.empty(max(size, 16), dtype=torch.uint8, device="cuda"), stream=stream)
        seen.append(("attention", n, qkv.clone(), o.clone()))
        pkg.project_w4(o, layer.w_out, y, rows, stream=stream)
        seen.append(("w4", layer.out, o.clone(), y.clone()))
        after = layers[(n + 1) % len(layers)].before
        x_in = x.clone()
        pkg.block_norm(x, y, x, h, rows, between, layer.gate, layer.after, None, after, stream=stream)
        seen.append(("norm", between, (x_in, y, layer.gate, layer.after, None, after, None), x.clone(), h.clone()))
    return seen


def verify(pkg, dev, model, seen, starts):
    for what, *rest in seen:
        if what == "norm":
            bp, inputs, x_out, h = rest
            r, tr, hr, th = norm_reference(pkg, bp, *inputs)
            if x_out is not None:
                check_norm(x_out, r, tr, "x_out")
            check_norm(h, hr, th, "h")
        elif what == "w4":
            weights, X, out = rest
            check_w4(out, *w4_reference(X, *weights, torch.float16))
        else:
            n, qkv, o = rest
            for b in range(SLOTS):
                lo, hi, kv = starts[b], starts[b + 1], model.kv[b]
                if lo == hi:
                    continue
                at = torch.arange(kv)
                page, slot = torch.tensor(model.pages[b])[at // PAGE].cuda(), (at % PAGE).cuda()
                K, V = (p[page, :, slot].double().transpose(0, 1) for p in dev[n].parts[:2])
                new = qkv[lo:hi].double()
                # The new tokens' keys and values are the last ones, to the bit.
                assert torch.equal(K[:, kv - (hi - lo):], new[:, D:D + H_KV * D_H].reshape(hi - lo, H_KV, D_H).transpose(0, 1))
                assert torch.equal(V[:, kv - (hi - lo):], new[:, D + H_KV * D_H:].reshape(hi - lo, H_KV, D_H).transpose(0, 1))
                ref, tol = attention_ref(new[:, :D].reshape(hi - lo, H, D_H).transpose(0, 1), K, V, hi - lo, kv, D_H ** -0.5, 1)
                got = o[lo:hi].double().reshape(hi - lo, H, D_H).transpose(0, 1)
                assert torch.isfinite(got).all() and ((got - ref).abs() <= tol).all()


def test_prompts_forks_tokens_and_a_compaction(pkg, torch_cuda):
    pkg.kernel_status_reset()
    layers = [Layer(pkg, 10), Layer(pkg, 20)]
    dev = [Device(pkg, PAGES, PAGE, SLOTS, WIDTH, H=H_KV, d=D_H, seed=n) for n in range(2)]
    model = Model(PAGES, PAGE, SLOTS, WIDTH)
    for d in dev:
        d.load(model)
    gen = torch.Generator(device="cuda").manual_seed(1)

    def run(new):
        model.take(new)
        for d in dev:
            pkg.pages_take(d.pool, d.starts(new), d.ws)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        x = torch.randn(starts[-1], D, generator=gen, device="cuda").half()
        seen = step(pkg, dev, layers, x, dev[0].starts(new), new, max(new))
        for d in dev:
            d.same(model)
        verify(pkg, dev, model, seen, starts)

    run([37, 0, 20, 0, 0, 0])                                                # two prompts
    model.fork([0, 0, 2], [1, 4, 5])                                         # three more answers
    for d in dev:
        pkg.pages_fork(d.pool, d.cache, d.ints(0, 0, 2), d.ints(1, 4, 5), d.ws)
        d.same(model)
    for _ in range(13):                                                      # tokens of all five, across a page's end
        run([1, 1, 1, 0, 1, 1])
    model.free([0, 2])
    for d in dev:
        pkg.pages_free(d.pool, d.ints(0, 2))
    run([0, 1, 0, 25, 1, 2])                                                 # a new prompt among tokens, in pages that others left
    model.pages, model.refs, _, _ = model.compact()
    for d in dev:
        pkg.pages_compact(d.pool, d.cache, d.pages, d.refs, d.ints(*[0] * PAGES), d.ws)
        d.same(model)
    for _ in range(3):
        run([0, 1, 0, 1, 1, 1])
    assert pkg.kernel_status()[0] == 0


def test_a_captured_token_step(pkg, torch_cuda):
    """The step of single tokens as a graph, replayed while lengths and tables grow."""
    pkg.kernel_status_reset()
    layers, dev, model = [Layer(pkg, 30)], [Device(pkg, PAGES, PAGE, SLOTS, WIDTH, H=H_KV, d=D_H, seed=3)], Model(PAGES, PAGE, SLOTS, WIDTH)
    dev[0].load(model)
    x = torch.zeros(SLOTS, D, dtype=torch.float16, device="cuda")
    new, starts = [1] * SLOTS, list(range(SLOTS + 1))
    on_device = dev[0].starts(new)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(pkg, dev, layers, x, on_device, new, 1, stream=side)           # once outside of a capture, over empty slots
        torch.cuda.synchronize()
        dev[0].load(model)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            pkg.pages_take(dev[0].pool, on_device, dev[0].ws, stream=side)
            seen = step(pkg, dev, layers, x, on_device, new, 1, stream=side)
    gen = torch.Generator(device="cuda").manual_seed(4)
    for _ in range(20):
        fresh = torch.randn(SLOTS, D, generator=gen, device="cuda").half()
        x.copy_(fresh)
        model.take(new)
        graph.replay()
        dev[0].same(model)
        verify(pkg, dev, model, seen, starts)
    assert pkg.kernel_status()[0] == 0
