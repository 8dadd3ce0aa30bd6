"""CPU: the head's choice of products is the calling thread's own."""
import threading


def test_one_threads_choice_leaves_the_others_alone(M, rt):
    seen = []

    def other():
        seen.append(rt.malus_linear_xent_mode(1))
        seen.append(rt.malus_linear_xent_mode(0))
    assert rt.malus_linear_xent_mode(0) == -1
    t = threading.Thread(target=other)
    t.start()
    t.join()
    assert rt.malus_linear_xent_mode(-1) == 0
    assert seen == [-1, 1]
