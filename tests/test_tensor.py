"""Tensors' descriptions, which need no GPU."""
import sys
import threading

import pytest

from affon_amd.core import Tensor


def described(shape, strides):
    return Tensor(None, None, "f32", shape, strides)


@pytest.mark.parametrize("shape,strides,contiguous", [
    ((3, 4), (4, 1), True), ((3, 4), (5, 1), False), ((3, 4), (1, 3), False), ((1, 4), (9, 1), True),
    ((3, 1), (1, 7), True), ((3, 1), (2, 1), False), ((), (), True), ((2, 3, 4), (12, 4, 1), True)])
def test_contiguous(shape, strides, contiguous):
    t = described(shape, strides)
    assert [t.is_contiguous(), t.is_contiguous()] == [contiguous] * 2


def test_contiguous_asked_by_two_threads():
    """A thread that asks while another one is at the strides is told what they say."""
    answers = []

    class Strides(tuple):
        asked = False

        def __reversed__(self):
            if not Strides.asked:
                Strides.asked = True
                other = threading.Thread(target=lambda: answers.append(t.is_contiguous()))
                other.start()
                other.join()
            return reversed(tuple(self))

    t = described((3, 4), (9, 1))
    t.strides = Strides(t.strides)
    answers.append(t.is_contiguous())
    assert answers == [False, False]


def test_contiguous_of_many_tensors_in_threads():
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        tensors, wrong = [described((8,) * 6, (1,) * 6) for _ in range(2000)], []

        def ask():
            wrong.extend(t for t in tensors if t.is_contiguous())
        threads = [threading.Thread(target=ask) for _ in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not wrong
    finally:
        sys.setswitchinterval(interval)


class Memory:
    ptr, nbytes = 1 << 20, 1 << 10


@pytest.mark.parametrize("shape,strides,values,message", [
    ((3, 4), (4, 1), [1, 2, 3], "shape"), ((3, 4), (5, 1), [[0] * 4] * 3, "contiguous"), ((2,), (1,), 5, "shape")])
def test_what_a_write_refuses(shape, strides, values, message):
    with pytest.raises(TypeError, match=message):
        Tensor(None, Memory, "u32", shape, strides).write(values)


def test_a_disposed_tensor_takes_no_values():
    t = Tensor(None, Memory, "f32", (2,), (1,))
    t.dispose()
    with pytest.raises(RuntimeError, match="disposed"):
        t.write([1, 2])
