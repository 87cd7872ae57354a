"""int8.tape8() belongs to the thread that entered it, and ends with its own block."""
import threading

from tf_depth_estimation_amd import int8


def test_threads_that_cross():
    """A enters, B enters, A leaves, B leaves: nobody else's networks are taped, and nothing stays on."""
    steps = [threading.Event() for _ in range(4)]
    seen = {}

    def a():
        with int8.tape8():
            seen["a in"] = int8.tape8_active()
            steps[0].set()
            assert steps[1].wait(10)
        seen["a out"] = int8.tape8_active()
        steps[2].set()

    def b():
        assert steps[0].wait(10)
        seen["b before"] = int8.tape8_active()
        with int8.tape8():
            steps[1].set()
            assert steps[2].wait(10)
            seen["b in"] = int8.tape8_active()
        seen["b out"] = int8.tape8_active()

    threads = [threading.Thread(target=f) for f in (a, b)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(20)
    assert seen == {"a in": True, "a out": False, "b before": False, "b in": True, "b out": False}
    assert not int8.tape8_active()


def test_a_thread_started_inside_is_outside():
    seen = []
    with int8.tape8():
        t = threading.Thread(target=lambda: seen.append(int8.tape8_active()))
        t.start()
        t.join(10)
        assert int8.tape8_active()
    assert seen == [False]


def test_blocks_left_in_another_order():
    first, second = int8.tape8(), int8.tape8()
    first.__enter__()
    second.__enter__()
    first.__exit__(None, None, None)
    assert int8.tape8_active()
    second.__exit__(None, None, None)
    assert not int8.tape8_active()
    off = int8.tape8(False)
    with int8.tape8():
        off.__enter__()
    assert not int8.tape8_active()
    off.__exit__(None, None, None)
    assert not int8.tape8_active()
