"""Batches that take the rarer ways of the attention's launch rule (tests/paged_rule.py names them), and chunks of more pages
than a wave holds numbers of."""

# more tiles than places: even rounds; the rule's last candidate; chunks enlarged to the workspace's room
WAYS = {
    "few, rounds": dict(new=[1] * 32, kv=[24 + 150 * i for i in range(32)], hq=32, hk=32, d=(128, 256), page=16, columns=2048,
                        few=True, way="rounds"),
    "few, rounds of groups": dict(new=[3] * 40, kv=[5000 - 120 * i for i in range(40)], hq=64, hk=32, d=(128, 256), page=64,
                                  columns=512, few=True, way="rounds"),
    "few, room": dict(new=[16] * 40, kv=[5000 - 120 * i for i in range(40)], hq=32, hk=32, d=(64,), page=64,
                      columns=512, few=True, way="room"),
    "few, last": dict(new=[1] * 7, kv=[8023, 8007, 5007, 3003, 8051, 5036, 1510], hq=5, hk=5, d=(128,), page=16, columns=504,
                      few=True, way="last"),
    "few, too short": dict(new=[1] * 32, kv=[24 + 19 * i for i in range(32)], hq=32, hk=32, d=(64, 128), page=16,
                           columns=2048, few=True, way="whole"),
    "many, rounds": dict(new=[40] * 36, kv=[60 + 160 * i for i in range(36)], hq=8, hk=8, d=(64, 128), page=16,
                         columns=2048, few=False, way="rounds"),
    "many, rounds of 24": dict(new=[40] * 36, kv=[60 + 160 * i for i in range(36)], hq=8, hk=8, d=(64,), page=24,
                               columns=512, few=False, way="rounds"),
    "many, room": dict(new=[300] * 8 + [1] * 32, kv=[6000] * 8 + [100] * 32, hq=8, hk=8, d=(64, 128), page=16, columns=500,
                       few=False, way="room"),
    "many, room of wide heads": dict(new=[40] * 36, kv=[60 + 160 * i for i in range(36)], hq=8, hk=8, d=(256,), page=16,
                                     columns=2048, few=False, way="room"),
    "many, last": dict(new=[1, 70, 70, 40, 1], kv=[230, 3043, 3006, 1516, 3004], hq=3, hk=3, d=(64,), page=16, columns=191,
                       few=False, way="last"),
    "many, too short": dict(new=[200, 90, 150], kv=[200, 300, 150], hq=8, hk=8, d=(64, 128), page=16, columns=2048,
                            few=False, way="whole"),
}
# chunks (nch of the first sequence) over pages of 16: 64 page numbers sit on a wave's lanes, refilled so many times
WINDOWS = {
    "few, once": dict(new=[1], kv=[40000], hq=32, hk=32, d=64, page=16, columns=2500, few=True, nch=32, refills=1),
    "few, twice": dict(new=[1], kv=[70000], hq=32, hk=32, d=64, page=16, columns=4375, few=True, nch=31, refills=2),
    "few, whole": dict(new=[1] * 8, kv=[1100 - i for i in range(8)], hq=160, hk=160, d=64, page=16, columns=69, few=True,
                       nch=1, refills=1),
    "many, once": dict(new=[40], kv=[40000], hq=8, hk=8, d=64, page=16, columns=2500, few=False, nch=32, refills=1),
    "many, twice": dict(new=[40], kv=[70000], hq=8, hk=8, d=128, page=16, columns=4375, few=False, nch=32, refills=2),
}
