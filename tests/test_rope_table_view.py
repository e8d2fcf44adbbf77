"""CPU: a rotary table over the caller's arrays frees nothing."""
from brasa_amd import RopeTable


class Buffer:
    ptr, freed = 4096, False

    def free(self):
        self.freed = True


def test_free_of_a_view():
    RopeTable.view(4096, 8192, 128, 10).free()  # (addresses)
    cos, sin = Buffer(), Buffer()
    RopeTable.view(cos, sin, 128, 10).free()
    assert not cos.freed and not sin.freed


def test_free_of_an_owned_table():
    t = RopeTable.__new__(RopeTable)
    t.cos, t.sin = Buffer(), Buffer()
    t.free()
    assert t.cos.freed and t.sin.freed
