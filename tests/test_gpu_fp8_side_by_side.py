"""Two engine threads, a context and a stream each, run a layer of the 8-bit operators at the same time.

Every pass starts from outputs full of a sentinel, and its outputs are compared on the device with what the layer gave
alone, so that a pass that did nothing or went wrong shows even where a later one did not."""
import threading

import numpy as np
import pytest

from test_gpu_fp8_layer import ROWS, Layer

pytestmark = pytest.mark.gpu
PASSES = 10


def _outputs(layer):
    return [*layer.c, *layer.s, layer.qkv, layer.q, layer.o, layer.att, layer.res, layer.gu, layer.y]


@pytest.mark.parametrize("kinds", [("prefill", "mixed"), ("decode", "prefill"), ("decode", "mixed")], ids="_".join)
def test_every_pass_beside_another_context(torch_mod, gsp, kinds):
    torch = torch_mod
    streams = [torch.cuda.Stream() for _ in kinds]
    layers, alone, pools = [], [], []
    for i, (kind, stream) in enumerate(zip(kinds, streams)):
        ctx = gsp.Context(0)
        ctx.set_stream(stream.cuda_stream)
        layer = Layer(torch, gsp, ctx, np.random.default_rng(40 + i), np.array(ROWS[kind]))
        layer.pack()
        layer.run()
        ctx.sync()
        layer.check()
        layers.append(layer)
        alone.append([t.clone() for t in _outputs(layer)])
        pools.append(layer.outputs()[-2:])
    torch.cuda.synchronize()
    bad = [torch.zeros(len(a), dtype=torch.int64, device="cuda") for a in alone]
    done, errors, start = [0, 0], [], threading.Barrier(2)

    def work(i):
        try:
            start.wait(30)
            with torch.cuda.stream(streams[i]):
                for _ in range(PASSES):
                    for t in _outputs(layers[i]):
                        t.fill_(77)
                    layers[i].run()
                    bad[i] += torch.stack([(t != w).any() for t, w in zip(_outputs(layers[i]), alone[i])])
                    done[i] += 1
            layers[i].ctx.sync()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,), daemon=True) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not any(t.is_alive() for t in threads) and not errors and done == [PASSES, PASSES]
    torch.cuda.synchronize()
    assert not any(b.any() for b in bad), [b.tolist() for b in bad]
    for layer, want, kv in zip(layers, alone, pools):
        assert all(torch.equal(t, w) for t, w in zip(_outputs(layer), want))
        assert all(np.array_equal(a, b) for a, b in zip(layer.outputs()[-2:], kv))
        layer.pool.destroy()
        layer.ctx.close()
