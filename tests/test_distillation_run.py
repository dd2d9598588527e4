"""The operators around a 4-bit student, together: a teacher's layer makes logits, its top alternatives are
kept, a layer with 4-bit weights makes the student's logits, one step gives loss and gradient, and the layer's
backward pass runs on the dequantised weights.  Each link is compared with its definition in float64, from what
the link before it has left; the tolerances are those of the operators' own tests."""
import threading

import numpy as np
import pytest

import test_logits_ops as logits
import test_mxfp4 as mx

FP32_TOL = 1e-5                                            # relative, Frobenius: that of the fp32 products' tests
RUNS = [(1, 64, 1500, 5, 1.0, 0.5), (70, 100, 5003, 16, 2.0, 0.7), (257, 784, 1030, 64, 4.0, 0.9),
        (9, 33, 900, 3, 1.5, 1.0), (300, 96, 33000, 20, 1.0, 0.25)]


class Run:
    """The buffers of a training step, and the step."""

    def __init__(self, g, batch, hidden, vocab, top, t, w, seed=0):
        self.g, self.size, self.t, self.w = g, (batch, hidden, vocab, top), t, w
        rng = np.random.default_rng(seed + batch * 31 + vocab)
        normal = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.x, self.teacher, self.student = normal(batch, hidden), normal(hidden, vocab), normal(hidden, vocab)
        self.bias = normal(vocab)
        self.labels = rng.integers(0, vocab, batch).astype(np.int32)
        self.labels[batch // 2] = -1
        f, e = g.Buffer.from_host, g.Buffer.empty
        self.b = dict(x=f(self.x), teacher=f(self.teacher), student=f(self.student), bias=f(self.bias),
                      labels=g.Buffer.from_host_int32(self.labels), z=e(batch * vocab * 4), top=e(batch * top * 4),
                      top_lp=e(batch * top * 4), entropy=e(batch * 4), packed=e(g.mxfp4_bytes(vocab, hidden)),
                      y=e(batch * vocab * 4), loss=e(batch * 4), grad=e(batch * vocab * 4), wq=e(hidden * vocab * 4),
                      wt=e(hidden * vocab * 4), dx=e(batch * hidden * 4), dw=e(hidden * vocab * 4), db=e(vocab * 4))

    def step(self):
        g, b, (batch, hidden, vocab, top) = self.g, self.b, self.size
        g.fused_linear_activation(b["x"], batch, hidden, b["teacher"], vocab, b["bias"], g.ACT_NONE, 0.0, b["z"])
        g.token_logprobs(b["z"], batch, vocab, entropy=b["entropy"], top_n=top, top_tokens=b["top"],
                         top_logprobs=b["top_lp"])
        g.mxfp4_quantize(b["student"], hidden, vocab, True, b["packed"])
        g.mxfp4_linear(b["x"], batch, hidden, b["packed"], vocab, b["bias"], g.ACT_NONE, 0.0, b["y"])
        g.distill_step(b["y"], batch, vocab, b["top"], b["top_lp"], top, b["labels"], self.t, self.w, loss=b["loss"],
                       grad=b["grad"], grad_scale=1.0 / batch)
        g.mxfp4_dequantize(b["packed"], vocab, hidden, b["wq"])
        g.transpose(b["wq"], (vocab, hidden), b["wt"])
        g.linear_backward(b["x"], b["wt"], b["grad"], None, batch, hidden, vocab, dx=b["dx"], dw=b["dw"], db=b["db"])

    def results(self):
        b, (batch, hidden, vocab, top) = self.b, self.size
        got = {k: b[k].retrieve(s) for k, s in dict(z=(batch, vocab), top_lp=(batch, top), entropy=(batch,),
                                                    y=(batch, vocab), loss=(batch,), grad=(batch, vocab),
                                                    wq=(vocab, hidden), dx=(batch, hidden), dw=(hidden, vocab),
                                                    db=(vocab,)).items()}
        return dict(got, top=b["top"].retrieve_int32((batch, top)))

    def check(self, r):
        batch, hidden, vocab, top = self.size
        x = self.x.astype(np.float64)
        best = np.argsort(-r["z"], axis=1, kind="stable")[:, :top]
        assert np.array_equal(r["top"], best)
        assert logits.close(r["top_lp"], np.take_along_axis(logits.logprobs64(r["z"]), best, 1),
                            logits.tol_logprob(r["z"], best))
        assert logits.close(r["entropy"], logits.entropy64(r["z"]), logits.tol_entropy(r["z"]))
        wq = mx.through(np.ascontiguousarray(self.student.T))
        assert np.array_equal(r["wq"], wq)
        xq = mx.through(self.x)
        mass = np.abs(xq) @ np.abs(wq.T) + np.abs(self.bias)
        assert np.all(np.abs(r["y"] - (xq @ wq.T + self.bias)) <= (hidden / 32 + 8) * 2.0 ** -23 * mass)
        loss, grad, tol_l, tol_g = logits.distill64(r["y"], r["top"], r["top_lp"], self.labels, self.t, self.w,
                                                    np.full(batch, np.float32(1.0 / batch), np.float64))
        assert logits.close(r["loss"], loss, tol_l) and logits.close(r["grad"], grad, tol_g)
        dy = r["grad"].astype(np.float64)
        for got, want in ((r["dx"], dy @ wq), (r["dw"], x.T @ dy)):
            assert np.linalg.norm(got - want) <= FP32_TOL * np.linalg.norm(want)
        assert np.all(np.abs(r["db"] - dy.sum(0)) <= batch * 2.0 ** -23 * np.abs(dy).sum(0))


@pytest.mark.gpu
@pytest.mark.parametrize("batch,hidden,vocab,top,t,w", RUNS)
def test_a_step_of_a_student(gpu, batch, hidden, vocab, top, t, w):
    """Without a wait in between, and a second time over the same buffers."""
    run = Run(gpu, batch, hidden, vocab, top, t, w)
    gpu.lib().gonngpu_set_blocking(0)
    try:
        run.step()
        gpu.synchronize()
        first = run.results()
        run.step()
        gpu.synchronize()
    finally:
        gpu.lib().gonngpu_set_blocking(1)
    again = run.results()
    run.check(first)
    assert all(np.array_equal(first[k], again[k]) for k in first)


@pytest.mark.gpu
def test_steps_of_several_callers(gpu):
    """Threads share the library's stream and its scratch."""
    runs = [Run(gpu, *RUNS[i % 4], seed=i) for i in range(4)]
    failed = []

    def work(run):
        try:
            for _ in range(3):
                run.step()
        except Exception as e:  # noqa: BLE001 - reported below
            failed.append(e)

    threads = [threading.Thread(target=work, args=(r,)) for r in runs]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed
    for run in runs:
        run.check(run.results())


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [5, 40])
def test_captured_and_replayed(gpu, batch):
    """The operators in a graph over the caller's own memory: replayed on new inputs, they give what the calls give."""
    import torch
    hidden, vocab, top = 96, 5003, 16
    g, dev = gpu, "cuda:0"
    gen = torch.Generator(device=dev).manual_seed(batch)
    new = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=dev)  # noqa: E731
    m = dict(x=new(batch, hidden), w=new(vocab, hidden), packed=new(g.mxfp4_bytes(vocab, hidden), dtype=torch.uint8),
             px=new(g.mxfp4_bytes(batch, hidden), dtype=torch.uint8), y=new(batch, vocab), lp=new(batch, top),
             tokens=new(batch, top, dtype=torch.int32), labels=new(batch, dtype=torch.int32), loss=new(batch),
             stats=new(batch, 3), grad=new(batch, vocab), back=new(batch, vocab), wq=new(vocab, hidden))
    b = {k: g.Buffer.wrap(v.data_ptr(), v.numel() * v.element_size(), v) for k, v in m.items()}

    def calls():
        g.mxfp4_quantize(b["w"], vocab, hidden, False, b["packed"])
        if batch <= 8:
            g.mxfp4_linear(b["x"], batch, hidden, b["packed"], vocab, None, g.ACT_NONE, 0.0, b["y"])
        else:
            g.mxfp4_quantize(b["x"], batch, hidden, False, b["px"])
            g.mxfp4_matmul(b["px"], batch, b["packed"], vocab, hidden, b["y"])
        g.token_logprobs(b["y"], batch, vocab, top_n=top, top_tokens=b["tokens"], top_logprobs=b["lp"])
        args = (b["y"], batch, vocab, b["tokens"], b["lp"], top, b["labels"], 2.0, 0.5)
        g.distill_forward(*args, loss=b["loss"], stats=b["stats"])
        g.distill_backward(*args, stats=b["stats"], grad=b["back"])
        g.distill_step(*args, loss=b["loss"], grad=b["grad"])
        g.mxfp4_dequantize(b["packed"], vocab, hidden, b["wq"])

    def fill():
        m["x"].normal_(generator=gen)
        m["w"].normal_(generator=gen)
        m["labels"].random_(0, vocab, generator=gen)
        torch.cuda.synchronize()

    results = ("y", "lp", "tokens", "loss", "stats", "grad", "back", "wq")
    stream = torch.cuda.ExternalStream(g.lib().gonngpu_stream())
    graph = torch.cuda.CUDAGraph()
    g.lib().gonngpu_set_blocking(0)
    try:
        fill()
        with torch.cuda.stream(stream):
            graph.capture_begin(capture_error_mode="thread_local")
            calls()
            if batch > 8:                                  # its scratch would outlive the capture
                with pytest.raises(g.GonnError) as e:
                    g.mxfp4_linear(b["x"], batch, hidden, b["packed"], vocab, None, g.ACT_NONE, 0.0, b["y"])
                assert e.value.code == -5 and "captured" in str(e.value)
            graph.capture_end()
        for _ in range(2):
            fill()
            with torch.cuda.stream(stream):
                graph.replay()
            torch.cuda.synchronize()
            replayed = {k: m[k].clone() for k in results}
            for k in results:
                m[k].zero_()
            torch.cuda.synchronize()
            calls()
            g.synchronize()
            assert all(torch.equal(replayed[k], m[k]) for k in results)
            assert bool((m["grad"] != 0).any()) and bool((m["loss"] > 0).all())
    finally:
        g.lib().gonngpu_set_blocking(1)


@pytest.mark.gpu
def test_memory_that_starts_between_words_is_refused(gpu):
    x, out = gpu.Buffer.empty(4096), gpu.Buffer.empty(64)
    odd = gpu.Buffer.wrap(x.device_address() + 2, 2048)
    mx.refused(gpu, lambda: gpu.token_logprobs(odd, 1, 100, entropy=out), -3)
    mx.refused(gpu, lambda: gpu.token_logprobs(x, 1, 100, entropy=odd), -3)
    p = gpu.Buffer.empty(gpu.mxfp4_bytes(1, 100))
    mx.refused(gpu, lambda: gpu.mxfp4_quantize(odd, 1, 100, False, p), -3)
    mx.refused(gpu, lambda: gpu.mxfp4_dequantize(p, 1, 100, odd), -3)
