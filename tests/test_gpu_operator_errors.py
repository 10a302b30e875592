"""What a program that calls operators alone learns of a kernel whose wait ran out: cpde_operator_give_up lets one run out in some
microseconds and end as the products' kernels do."""
import pytest

torch = pytest.importorskip('torch')

from cpde_b200 import native, operators  # noqa: E402
from test_gpu_layers import BF16, made, same_bits, update  # noqa: E402

pytestmark = pytest.mark.gpu


def test_a_wait_that_ran_out_is_reported_once():
    torch.cuda.init()
    x, weight, matrix = made(1, 1500, 264, dtype=BF16), made(2, 600, 264, dtype=BF16), update(3, 40, 60)
    with native.Engine(0) as engine:
        operators.check(engine)
        want, _ = operators.linear(engine, x, weight)
        calls = [lambda: operators.linear(engine, x, weight), lambda: operators.linear_gradient(engine, want, x, weight),
                 lambda: operators.orthogonalize(engine, matrix), lambda: operators.muon(engine, matrix, matrix, matrix, 0.1),
                 lambda: operators.dropout(engine, x, 0.5, 1), lambda: operators.check(engine)]
        for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
            for call in calls:
                assert engine.lib.cpde_operator_give_up(engine.handle, stream.cuda_stream or 1) == native.OK
                torch.cuda.synchronize()
                with pytest.raises(native.EngineError, match='gave up') as error:
                    call()
                assert error.value.status == native.DEVICE_ERROR
                call()  # and the engine works on
        assert same_bits(operators.linear(engine, x, weight)[0], want)
        operators.check(engine)


def test_a_wait_of_a_graph_is_reported():
    torch.cuda.init()
    with native.Engine(0) as engine, native.Engine(0) as other:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            assert engine.lib.cpde_operator_give_up(engine.handle, torch.cuda.current_stream().cuda_stream) == native.OK
        operators.check(engine)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            operators.check(other)
            with pytest.raises(native.EngineError, match='gave up'):
                operators.check(engine)
