// Generated by gen_tile_asm.py -- do not edit; see that file for the register plan and the schedule.
// SK_TILE_ASM_LOADS / _LOADS_NN / _LOADS_TN: the 16 loads of one stage.  SK_TILE_ASM_LOOP(MF) / _LOOP_NN(MF) / _LOOP_TN(MF): the loop
// (_LOW: tiles of at most 128 rows) for the NT / NN / TN layout, MF = the MFMA mnemonic as a string literal.  SK_TILE_ASM_LOOP_F8(MF, MOD): fp8 operands, MOD =
// the format modifiers of the MFMA ("" for e4m3).  SK_TILE_ASM_STORE_x(CVT): the epilogue that leaves the stages alone.
#pragma once
#define SK_TILE_ASM_LOADS \
  "s_mov_b32 s83, %[ga]\n\t" \
  "s_add_u32 m0, %[lds], 0\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 4096\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 8192\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 12288\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 16384\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 20480\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 24576\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 28672\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_mov_b32 s83, %[gb]\n\t" \
  "s_add_u32 m0, %[lds], 32768\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 36864\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 40960\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 45056\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 49152\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 53248\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 57344\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 61440\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  ""
#define SK_TILE_ASM_LOADS_NN \
  "s_mov_b32 s83, %[ga]\n\t" \
  "s_add_u32 m0, %[lds], 0\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 4096\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 8192\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 12288\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 16384\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 20480\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 24576\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 28672\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_mov_b32 s83, %[gb]\n\t" \
  "s_add_u32 m0, %[lds], 32768\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 36864\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 40960\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 45056\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 49152\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 53248\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 57344\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 61440\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  ""
#define SK_TILE_ASM_LOADS_EARLY \
  "s_mov_b32 s83, %[ga]\n\t" \
  "s_add_u32 m0, %[lds], 0\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 4096\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas3]\n\t" \
  "s_add_u32 m0, %[lds], 16384\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 20480\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_mov_b32 s83, %[gb]\n\t" \
  "s_add_u32 m0, %[lds], 32768\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 36864\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, %[lds], 49152\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 53248\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  ""
#define SK_TILE_ASM_LOADS_EARLY_NN \
  "s_mov_b32 s83, %[ga]\n\t" \
  "s_add_u32 m0, %[lds], 0\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 4096\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas3]\n\t" \
  "s_add_u32 m0, %[lds], 16384\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 20480\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_mov_b32 s83, %[gb]\n\t" \
  "s_add_u32 m0, %[lds], 32768\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 36864\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 40960\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 45056\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 49152\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 53248\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 57344\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 61440\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  ""
#define SK_TILE_ASM_LOADS_TN \
  "s_mov_b32 s83, %[ga]\n\t" \
  "s_add_u32 m0, %[lds], 0\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 4096\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa1], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 8192\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 12288\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa1], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 16384\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 20480\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa1], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 24576\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 28672\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa1], %[rsa], s83 offen lds\n\t" \
  "s_mov_b32 s83, %[gb]\n\t" \
  "s_add_u32 m0, %[lds], 32768\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 36864\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 40960\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 45056\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 49152\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 53248\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 57344\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 61440\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  ""
#define SK_TILE_ASM_LOADS_EARLY_TN \
  "s_mov_b32 s83, %[ga]\n\t" \
  "s_add_u32 m0, %[lds], 0\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 4096\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa1], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 8192\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 12288\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa1], %[rsa], s83 offen lds\n\t" \
  "s_mov_b32 s83, %[gb]\n\t" \
  "s_add_u32 m0, %[lds], 32768\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 36864\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 40960\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 45056\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  ""
#define SK_TILE_ASM_LOADS_LOW \
  "s_mov_b32 s83, %[ga]\n\t" \
  "s_add_u32 m0, %[lds], 0\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 4096\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 16384\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 20480\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_mov_b32 s83, %[gb]\n\t" \
  "s_add_u32 m0, %[lds], 32768\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 36864\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 40960\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 45056\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 49152\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 53248\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 57344\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 61440\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  ""
#define SK_TILE_ASM_LOADS_EARLY_LOW \
  "s_mov_b32 s83, %[ga]\n\t" \
  "s_add_u32 m0, %[lds], 0\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 4096\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 16384\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 20480\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_mov_b32 s83, %[gb]\n\t" \
  "s_add_u32 m0, %[lds], 32768\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 36864\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, %[lds], 49152\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 53248\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  ""
#define SK_TILE_ASM_LOADS_LOW_NN \
  "s_mov_b32 s83, %[ga]\n\t" \
  "s_add_u32 m0, %[lds], 0\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 4096\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 16384\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 20480\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_mov_b32 s83, %[gb]\n\t" \
  "s_add_u32 m0, %[lds], 32768\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 36864\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 40960\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 45056\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 49152\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 53248\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 57344\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 61440\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  ""
#define SK_TILE_ASM_LOADS_EARLY_LOW_NN \
  "s_mov_b32 s83, %[ga]\n\t" \
  "s_add_u32 m0, %[lds], 0\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 4096\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 16384\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, %[lds], 20480\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[voa], %[rsa], s83 offen lds\n\t" \
  "s_mov_b32 s83, %[gb]\n\t" \
  "s_add_u32 m0, %[lds], 32768\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 36864\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 40960\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob], %[rsb], s83 offen lds\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, %[lds], 45056\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 %[vob1], %[rsb], s83 offen lds\n\t" \
  ""
#define SK_TILE_ASM_LOOP(MF) \
  "v_accvgpr_write_b32 a0, 0\n\t" \
  "v_accvgpr_write_b32 a1, 0\n\t" \
  "v_accvgpr_write_b32 a2, 0\n\t" \
  "v_accvgpr_write_b32 a3, 0\n\t" \
  "v_accvgpr_write_b32 a4, 0\n\t" \
  "v_accvgpr_write_b32 a5, 0\n\t" \
  "v_accvgpr_write_b32 a6, 0\n\t" \
  "v_accvgpr_write_b32 a7, 0\n\t" \
  "v_accvgpr_write_b32 a8, 0\n\t" \
  "v_accvgpr_write_b32 a9, 0\n\t" \
  "v_accvgpr_write_b32 a10, 0\n\t" \
  "v_accvgpr_write_b32 a11, 0\n\t" \
  "v_accvgpr_write_b32 a12, 0\n\t" \
  "v_accvgpr_write_b32 a13, 0\n\t" \
  "v_accvgpr_write_b32 a14, 0\n\t" \
  "v_accvgpr_write_b32 a15, 0\n\t" \
  "v_accvgpr_write_b32 a16, 0\n\t" \
  "v_accvgpr_write_b32 a17, 0\n\t" \
  "v_accvgpr_write_b32 a18, 0\n\t" \
  "v_accvgpr_write_b32 a19, 0\n\t" \
  "v_accvgpr_write_b32 a20, 0\n\t" \
  "v_accvgpr_write_b32 a21, 0\n\t" \
  "v_accvgpr_write_b32 a22, 0\n\t" \
  "v_accvgpr_write_b32 a23, 0\n\t" \
  "v_accvgpr_write_b32 a24, 0\n\t" \
  "v_accvgpr_write_b32 a25, 0\n\t" \
  "v_accvgpr_write_b32 a26, 0\n\t" \
  "v_accvgpr_write_b32 a27, 0\n\t" \
  "v_accvgpr_write_b32 a28, 0\n\t" \
  "v_accvgpr_write_b32 a29, 0\n\t" \
  "v_accvgpr_write_b32 a30, 0\n\t" \
  "v_accvgpr_write_b32 a31, 0\n\t" \
  "v_accvgpr_write_b32 a32, 0\n\t" \
  "v_accvgpr_write_b32 a33, 0\n\t" \
  "v_accvgpr_write_b32 a34, 0\n\t" \
  "v_accvgpr_write_b32 a35, 0\n\t" \
  "v_accvgpr_write_b32 a36, 0\n\t" \
  "v_accvgpr_write_b32 a37, 0\n\t" \
  "v_accvgpr_write_b32 a38, 0\n\t" \
  "v_accvgpr_write_b32 a39, 0\n\t" \
  "v_accvgpr_write_b32 a40, 0\n\t" \
  "v_accvgpr_write_b32 a41, 0\n\t" \
  "v_accvgpr_write_b32 a42, 0\n\t" \
  "v_accvgpr_write_b32 a43, 0\n\t" \
  "v_accvgpr_write_b32 a44, 0\n\t" \
  "v_accvgpr_write_b32 a45, 0\n\t" \
  "v_accvgpr_write_b32 a46, 0\n\t" \
  "v_accvgpr_write_b32 a47, 0\n\t" \
  "v_accvgpr_write_b32 a48, 0\n\t" \
  "v_accvgpr_write_b32 a49, 0\n\t" \
  "v_accvgpr_write_b32 a50, 0\n\t" \
  "v_accvgpr_write_b32 a51, 0\n\t" \
  "v_accvgpr_write_b32 a52, 0\n\t" \
  "v_accvgpr_write_b32 a53, 0\n\t" \
  "v_accvgpr_write_b32 a54, 0\n\t" \
  "v_accvgpr_write_b32 a55, 0\n\t" \
  "v_accvgpr_write_b32 a56, 0\n\t" \
  "v_accvgpr_write_b32 a57, 0\n\t" \
  "v_accvgpr_write_b32 a58, 0\n\t" \
  "v_accvgpr_write_b32 a59, 0\n\t" \
  "v_accvgpr_write_b32 a60, 0\n\t" \
  "v_accvgpr_write_b32 a61, 0\n\t" \
  "v_accvgpr_write_b32 a62, 0\n\t" \
  "v_accvgpr_write_b32 a63, 0\n\t" \
  "v_accvgpr_write_b32 a64, 0\n\t" \
  "v_accvgpr_write_b32 a65, 0\n\t" \
  "v_accvgpr_write_b32 a66, 0\n\t" \
  "v_accvgpr_write_b32 a67, 0\n\t" \
  "v_accvgpr_write_b32 a68, 0\n\t" \
  "v_accvgpr_write_b32 a69, 0\n\t" \
  "v_accvgpr_write_b32 a70, 0\n\t" \
  "v_accvgpr_write_b32 a71, 0\n\t" \
  "v_accvgpr_write_b32 a72, 0\n\t" \
  "v_accvgpr_write_b32 a73, 0\n\t" \
  "v_accvgpr_write_b32 a74, 0\n\t" \
  "v_accvgpr_write_b32 a75, 0\n\t" \
  "v_accvgpr_write_b32 a76, 0\n\t" \
  "v_accvgpr_write_b32 a77, 0\n\t" \
  "v_accvgpr_write_b32 a78, 0\n\t" \
  "v_accvgpr_write_b32 a79, 0\n\t" \
  "v_accvgpr_write_b32 a80, 0\n\t" \
  "v_accvgpr_write_b32 a81, 0\n\t" \
  "v_accvgpr_write_b32 a82, 0\n\t" \
  "v_accvgpr_write_b32 a83, 0\n\t" \
  "v_accvgpr_write_b32 a84, 0\n\t" \
  "v_accvgpr_write_b32 a85, 0\n\t" \
  "v_accvgpr_write_b32 a86, 0\n\t" \
  "v_accvgpr_write_b32 a87, 0\n\t" \
  "v_accvgpr_write_b32 a88, 0\n\t" \
  "v_accvgpr_write_b32 a89, 0\n\t" \
  "v_accvgpr_write_b32 a90, 0\n\t" \
  "v_accvgpr_write_b32 a91, 0\n\t" \
  "v_accvgpr_write_b32 a92, 0\n\t" \
  "v_accvgpr_write_b32 a93, 0\n\t" \
  "v_accvgpr_write_b32 a94, 0\n\t" \
  "v_accvgpr_write_b32 a95, 0\n\t" \
  "v_accvgpr_write_b32 a96, 0\n\t" \
  "v_accvgpr_write_b32 a97, 0\n\t" \
  "v_accvgpr_write_b32 a98, 0\n\t" \
  "v_accvgpr_write_b32 a99, 0\n\t" \
  "v_accvgpr_write_b32 a100, 0\n\t" \
  "v_accvgpr_write_b32 a101, 0\n\t" \
  "v_accvgpr_write_b32 a102, 0\n\t" \
  "v_accvgpr_write_b32 a103, 0\n\t" \
  "v_accvgpr_write_b32 a104, 0\n\t" \
  "v_accvgpr_write_b32 a105, 0\n\t" \
  "v_accvgpr_write_b32 a106, 0\n\t" \
  "v_accvgpr_write_b32 a107, 0\n\t" \
  "v_accvgpr_write_b32 a108, 0\n\t" \
  "v_accvgpr_write_b32 a109, 0\n\t" \
  "v_accvgpr_write_b32 a110, 0\n\t" \
  "v_accvgpr_write_b32 a111, 0\n\t" \
  "v_accvgpr_write_b32 a112, 0\n\t" \
  "v_accvgpr_write_b32 a113, 0\n\t" \
  "v_accvgpr_write_b32 a114, 0\n\t" \
  "v_accvgpr_write_b32 a115, 0\n\t" \
  "v_accvgpr_write_b32 a116, 0\n\t" \
  "v_accvgpr_write_b32 a117, 0\n\t" \
  "v_accvgpr_write_b32 a118, 0\n\t" \
  "v_accvgpr_write_b32 a119, 0\n\t" \
  "v_accvgpr_write_b32 a120, 0\n\t" \
  "v_accvgpr_write_b32 a121, 0\n\t" \
  "v_accvgpr_write_b32 a122, 0\n\t" \
  "v_accvgpr_write_b32 a123, 0\n\t" \
  "v_accvgpr_write_b32 a124, 0\n\t" \
  "v_accvgpr_write_b32 a125, 0\n\t" \
  "v_accvgpr_write_b32 a126, 0\n\t" \
  "v_accvgpr_write_b32 a127, 0\n\t" \
  "v_accvgpr_write_b32 a128, 0\n\t" \
  "v_accvgpr_write_b32 a129, 0\n\t" \
  "v_accvgpr_write_b32 a130, 0\n\t" \
  "v_accvgpr_write_b32 a131, 0\n\t" \
  "v_accvgpr_write_b32 a132, 0\n\t" \
  "v_accvgpr_write_b32 a133, 0\n\t" \
  "v_accvgpr_write_b32 a134, 0\n\t" \
  "v_accvgpr_write_b32 a135, 0\n\t" \
  "v_accvgpr_write_b32 a136, 0\n\t" \
  "v_accvgpr_write_b32 a137, 0\n\t" \
  "v_accvgpr_write_b32 a138, 0\n\t" \
  "v_accvgpr_write_b32 a139, 0\n\t" \
  "v_accvgpr_write_b32 a140, 0\n\t" \
  "v_accvgpr_write_b32 a141, 0\n\t" \
  "v_accvgpr_write_b32 a142, 0\n\t" \
  "v_accvgpr_write_b32 a143, 0\n\t" \
  "v_accvgpr_write_b32 a144, 0\n\t" \
  "v_accvgpr_write_b32 a145, 0\n\t" \
  "v_accvgpr_write_b32 a146, 0\n\t" \
  "v_accvgpr_write_b32 a147, 0\n\t" \
  "v_accvgpr_write_b32 a148, 0\n\t" \
  "v_accvgpr_write_b32 a149, 0\n\t" \
  "v_accvgpr_write_b32 a150, 0\n\t" \
  "v_accvgpr_write_b32 a151, 0\n\t" \
  "v_accvgpr_write_b32 a152, 0\n\t" \
  "v_accvgpr_write_b32 a153, 0\n\t" \
  "v_accvgpr_write_b32 a154, 0\n\t" \
  "v_accvgpr_write_b32 a155, 0\n\t" \
  "v_accvgpr_write_b32 a156, 0\n\t" \
  "v_accvgpr_write_b32 a157, 0\n\t" \
  "v_accvgpr_write_b32 a158, 0\n\t" \
  "v_accvgpr_write_b32 a159, 0\n\t" \
  "v_accvgpr_write_b32 a160, 0\n\t" \
  "v_accvgpr_write_b32 a161, 0\n\t" \
  "v_accvgpr_write_b32 a162, 0\n\t" \
  "v_accvgpr_write_b32 a163, 0\n\t" \
  "v_accvgpr_write_b32 a164, 0\n\t" \
  "v_accvgpr_write_b32 a165, 0\n\t" \
  "v_accvgpr_write_b32 a166, 0\n\t" \
  "v_accvgpr_write_b32 a167, 0\n\t" \
  "v_accvgpr_write_b32 a168, 0\n\t" \
  "v_accvgpr_write_b32 a169, 0\n\t" \
  "v_accvgpr_write_b32 a170, 0\n\t" \
  "v_accvgpr_write_b32 a171, 0\n\t" \
  "v_accvgpr_write_b32 a172, 0\n\t" \
  "v_accvgpr_write_b32 a173, 0\n\t" \
  "v_accvgpr_write_b32 a174, 0\n\t" \
  "v_accvgpr_write_b32 a175, 0\n\t" \
  "v_accvgpr_write_b32 a176, 0\n\t" \
  "v_accvgpr_write_b32 a177, 0\n\t" \
  "v_accvgpr_write_b32 a178, 0\n\t" \
  "v_accvgpr_write_b32 a179, 0\n\t" \
  "v_accvgpr_write_b32 a180, 0\n\t" \
  "v_accvgpr_write_b32 a181, 0\n\t" \
  "v_accvgpr_write_b32 a182, 0\n\t" \
  "v_accvgpr_write_b32 a183, 0\n\t" \
  "v_accvgpr_write_b32 a184, 0\n\t" \
  "v_accvgpr_write_b32 a185, 0\n\t" \
  "v_accvgpr_write_b32 a186, 0\n\t" \
  "v_accvgpr_write_b32 a187, 0\n\t" \
  "v_accvgpr_write_b32 a188, 0\n\t" \
  "v_accvgpr_write_b32 a189, 0\n\t" \
  "v_accvgpr_write_b32 a190, 0\n\t" \
  "v_accvgpr_write_b32 a191, 0\n\t" \
  "v_accvgpr_write_b32 a192, 0\n\t" \
  "v_accvgpr_write_b32 a193, 0\n\t" \
  "v_accvgpr_write_b32 a194, 0\n\t" \
  "v_accvgpr_write_b32 a195, 0\n\t" \
  "v_accvgpr_write_b32 a196, 0\n\t" \
  "v_accvgpr_write_b32 a197, 0\n\t" \
  "v_accvgpr_write_b32 a198, 0\n\t" \
  "v_accvgpr_write_b32 a199, 0\n\t" \
  "v_accvgpr_write_b32 a200, 0\n\t" \
  "v_accvgpr_write_b32 a201, 0\n\t" \
  "v_accvgpr_write_b32 a202, 0\n\t" \
  "v_accvgpr_write_b32 a203, 0\n\t" \
  "v_accvgpr_write_b32 a204, 0\n\t" \
  "v_accvgpr_write_b32 a205, 0\n\t" \
  "v_accvgpr_write_b32 a206, 0\n\t" \
  "v_accvgpr_write_b32 a207, 0\n\t" \
  "v_accvgpr_write_b32 a208, 0\n\t" \
  "v_accvgpr_write_b32 a209, 0\n\t" \
  "v_accvgpr_write_b32 a210, 0\n\t" \
  "v_accvgpr_write_b32 a211, 0\n\t" \
  "v_accvgpr_write_b32 a212, 0\n\t" \
  "v_accvgpr_write_b32 a213, 0\n\t" \
  "v_accvgpr_write_b32 a214, 0\n\t" \
  "v_accvgpr_write_b32 a215, 0\n\t" \
  "v_accvgpr_write_b32 a216, 0\n\t" \
  "v_accvgpr_write_b32 a217, 0\n\t" \
  "v_accvgpr_write_b32 a218, 0\n\t" \
  "v_accvgpr_write_b32 a219, 0\n\t" \
  "v_accvgpr_write_b32 a220, 0\n\t" \
  "v_accvgpr_write_b32 a221, 0\n\t" \
  "v_accvgpr_write_b32 a222, 0\n\t" \
  "v_accvgpr_write_b32 a223, 0\n\t" \
  "v_accvgpr_write_b32 a224, 0\n\t" \
  "v_accvgpr_write_b32 a225, 0\n\t" \
  "v_accvgpr_write_b32 a226, 0\n\t" \
  "v_accvgpr_write_b32 a227, 0\n\t" \
  "v_accvgpr_write_b32 a228, 0\n\t" \
  "v_accvgpr_write_b32 a229, 0\n\t" \
  "v_accvgpr_write_b32 a230, 0\n\t" \
  "v_accvgpr_write_b32 a231, 0\n\t" \
  "v_accvgpr_write_b32 a232, 0\n\t" \
  "v_accvgpr_write_b32 a233, 0\n\t" \
  "v_accvgpr_write_b32 a234, 0\n\t" \
  "v_accvgpr_write_b32 a235, 0\n\t" \
  "v_accvgpr_write_b32 a236, 0\n\t" \
  "v_accvgpr_write_b32 a237, 0\n\t" \
  "v_accvgpr_write_b32 a238, 0\n\t" \
  "v_accvgpr_write_b32 a239, 0\n\t" \
  "v_accvgpr_write_b32 a240, 0\n\t" \
  "v_accvgpr_write_b32 a241, 0\n\t" \
  "v_accvgpr_write_b32 a242, 0\n\t" \
  "v_accvgpr_write_b32 a243, 0\n\t" \
  "v_accvgpr_write_b32 a244, 0\n\t" \
  "v_accvgpr_write_b32 a245, 0\n\t" \
  "v_accvgpr_write_b32 a246, 0\n\t" \
  "v_accvgpr_write_b32 a247, 0\n\t" \
  "v_accvgpr_write_b32 a248, 0\n\t" \
  "v_accvgpr_write_b32 a249, 0\n\t" \
  "v_accvgpr_write_b32 a250, 0\n\t" \
  "v_accvgpr_write_b32 a251, 0\n\t" \
  "v_accvgpr_write_b32 a252, 0\n\t" \
  "v_accvgpr_write_b32 a253, 0\n\t" \
  "v_accvgpr_write_b32 a254, 0\n\t" \
  "v_accvgpr_write_b32 a255, 0\n\t" \
  "s_mov_b32 s80, 0\n\t" \
  "s_xor_b32 s86, %[lds], 0x10000\n\t" \
  "s_add_u32 s81, %[ga0], 128\n\t" \
  "s_add_u32 s82, %[gb0], 128\n\t" \
  "s_add_u32 s87, s80, 1\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "v_or_b32 v120, s84, %[voa]\n\t" \
  "v_or_b32 v121, s84, %[vob]\n\t" \
  "s_waitcnt vmcnt(8)\n\t" \
  "s_barrier\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  "ds_read_b128 v[160:163], %[rb0] offset:0\n\t" \
  "ds_read_b128 v[164:167], %[rb0] offset:2048\n\t" \
  "ds_read_b128 v[168:171], %[rb0] offset:4096\n\t" \
  "ds_read_b128 v[172:175], %[rb0] offset:6144\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  "s_nop 7\n\t" \
  "L_sk_loop%=:\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[0:3], v[160:163], v[128:131], a[0:3]\n\t" \
  "ds_read_b128 v[176:179], %[rb0] offset:8192\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[4:7], v[164:167], v[128:131], a[4:7]\n\t" \
  "ds_read_b128 v[180:183], %[rb0] offset:10240\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[8:11], v[168:171], v[128:131], a[8:11]\n\t" \
  "ds_read_b128 v[184:187], %[rb0] offset:12288\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[12:15], v[172:175], v[128:131], a[12:15]\n\t" \
  "ds_read_b128 v[188:191], %[rb0] offset:14336\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[44:47], v[172:175], v[132:135], a[44:47]\n\t" \
  "ds_read_b128 v[144:147], %[ra0] offset:8192\n\t" \
  MF " a[40:43], v[168:171], v[132:135], a[40:43]\n\t" \
  "ds_read_b128 v[148:151], %[ra0] offset:10240\n\t" \
  MF " a[36:39], v[164:167], v[132:135], a[36:39]\n\t" \
  "ds_read_b128 v[152:155], %[ra0] offset:12288\n\t" \
  MF " a[32:35], v[160:163], v[132:135], a[32:35]\n\t" \
  "ds_read_b128 v[156:159], %[ra0] offset:14336\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[64:67], v[160:163], v[136:139], a[64:67]\n\t" \
  "s_add_u32 s83, s81, %[gas2]\n\t" \
  "s_add_u32 m0, s86, 8192\n\t" \
  MF " a[68:71], v[164:167], v[136:139], a[68:71]\n\t" \
  "ds_read_b128 v[192:195], %[ra1] offset:0\n\t" \
  MF " a[72:75], v[168:171], v[136:139], a[72:75]\n\t" \
  "v_xor_b32 %[ra0], 0x10000, %[ra0]\n\t" \
  MF " a[76:79], v[172:175], v[136:139], a[76:79]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[108:111], v[172:175], v[140:143], a[108:111]\n\t" \
  MF " a[104:107], v[168:171], v[140:143], a[104:107]\n\t" \
  MF " a[100:103], v[164:167], v[140:143], a[100:103]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 12288\n\t" \
  MF " a[96:99], v[160:163], v[140:143], a[96:99]\n\t" \
  "ds_read_b128 v[224:227], %[rb1] offset:0\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[112:115], v[176:179], v[140:143], a[112:115]\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  MF " a[116:119], v[180:183], v[140:143], a[116:119]\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[120:123], v[184:187], v[140:143], a[120:123]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[124:127], v[188:191], v[140:143], a[124:127]\n\t" \
  MF " a[92:95], v[188:191], v[136:139], a[92:95]\n\t" \
  "ds_read_b128 v[228:231], %[rb1] offset:2048\n\t" \
  MF " a[88:91], v[184:187], v[136:139], a[88:91]\n\t" \
  "s_add_u32 s83, s83, %[gas3]\n\t" \
  "s_add_u32 m0, s86, 24576\n\t" \
  MF " a[84:87], v[180:183], v[136:139], a[84:87]\n\t" \
  MF " a[80:83], v[176:179], v[136:139], a[80:83]\n\t" \
  MF " a[48:51], v[176:179], v[132:135], a[48:51]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[52:55], v[180:183], v[132:135], a[52:55]\n\t" \
  MF " a[56:59], v[184:187], v[132:135], a[56:59]\n\t" \
  "ds_read_b128 v[232:235], %[rb1] offset:4096\n\t" \
  MF " a[60:63], v[188:191], v[132:135], a[60:63]\n\t" \
  MF " a[28:31], v[188:191], v[128:131], a[28:31]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 28672\n\t" \
  MF " a[24:27], v[184:187], v[128:131], a[24:27]\n\t" \
  MF " a[20:23], v[180:183], v[128:131], a[20:23]\n\t" \
  MF " a[16:19], v[176:179], v[128:131], a[16:19]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[144:147], v[176:179], v[144:147], a[144:147]\n\t" \
  "ds_read_b128 v[236:239], %[rb1] offset:6144\n\t" \
  MF " a[148:151], v[180:183], v[144:147], a[148:151]\n\t" \
  MF " a[152:155], v[184:187], v[144:147], a[152:155]\n\t" \
  MF " a[156:159], v[188:191], v[144:147], a[156:159]\n\t" \
  "s_add_u32 s83, s82, %[gbs2]\n\t" \
  "s_add_u32 m0, s86, 40960\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[188:191], v[188:191], v[148:151], a[188:191]\n\t" \
  MF " a[184:187], v[184:187], v[148:151], a[184:187]\n\t" \
  "ds_read_b128 v[196:199], %[ra1] offset:2048\n\t" \
  MF " a[180:183], v[180:183], v[148:151], a[180:183]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[176:179], v[176:179], v[148:151], a[176:179]\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[208:211], v[176:179], v[152:155], a[208:211]\n\t" \
  "v_xor_b32 %[rb0], 0x10000, %[rb0]\n\t" \
  MF " a[212:215], v[180:183], v[152:155], a[212:215]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 45056\n\t" \
  MF " a[216:219], v[184:187], v[152:155], a[216:219]\n\t" \
  MF " a[220:223], v[188:191], v[152:155], a[220:223]\n\t" \
  "ds_read_b128 v[200:203], %[ra1] offset:4096\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[252:255], v[188:191], v[156:159], a[252:255]\n\t" \
  MF " a[248:251], v[184:187], v[156:159], a[248:251]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[244:247], v[180:183], v[156:159], a[244:247]\n\t" \
  MF " a[240:243], v[176:179], v[156:159], a[240:243]\n\t" \
  MF " a[236:239], v[172:175], v[156:159], a[236:239]\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 57344\n\t" \
  MF " a[232:235], v[168:171], v[156:159], a[232:235]\n\t" \
  "ds_read_b128 v[204:207], %[ra1] offset:6144\n\t" \
  MF " a[228:231], v[164:167], v[156:159], a[228:231]\n\t" \
  MF " a[224:227], v[160:163], v[156:159], a[224:227]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[192:195], v[160:163], v[152:155], a[192:195]\n\t" \
  MF " a[196:199], v[164:167], v[152:155], a[196:199]\n\t" \
  MF " a[200:203], v[168:171], v[152:155], a[200:203]\n\t" \
  MF " a[204:207], v[172:175], v[152:155], a[204:207]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 61440\n\t" \
  MF " a[172:175], v[172:175], v[148:151], a[172:175]\n\t" \
  MF " a[168:171], v[168:171], v[148:151], a[168:171]\n\t" \
  MF " a[164:167], v[164:167], v[148:151], a[164:167]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[160:163], v[160:163], v[148:151], a[160:163]\n\t" \
  MF " a[128:131], v[160:163], v[144:147], a[128:131]\n\t" \
  MF " a[132:135], v[164:167], v[144:147], a[132:135]\n\t" \
  MF " a[136:139], v[168:171], v[144:147], a[136:139]\n\t" \
  MF " a[140:143], v[172:175], v[144:147], a[140:143]\n\t" \
  "s_waitcnt vmcnt(8) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  MF " a[0:3], v[224:227], v[192:195], a[0:3]\n\t" \
  "ds_read_b128 v[240:243], %[rb1] offset:8192\n\t" \
  MF " a[4:7], v[228:231], v[192:195], a[4:7]\n\t" \
  "ds_read_b128 v[244:247], %[rb1] offset:10240\n\t" \
  MF " a[8:11], v[232:235], v[192:195], a[8:11]\n\t" \
  "ds_read_b128 v[248:251], %[rb1] offset:12288\n\t" \
  MF " a[12:15], v[236:239], v[192:195], a[12:15]\n\t" \
  "ds_read_b128 v[252:255], %[rb1] offset:14336\n\t" \
  MF " a[44:47], v[236:239], v[196:199], a[44:47]\n\t" \
  "ds_read_b128 v[208:211], %[ra1] offset:8192\n\t" \
  MF " a[40:43], v[232:235], v[196:199], a[40:43]\n\t" \
  "ds_read_b128 v[212:215], %[ra1] offset:10240\n\t" \
  MF " a[36:39], v[228:231], v[196:199], a[36:39]\n\t" \
  "ds_read_b128 v[216:219], %[ra1] offset:12288\n\t" \
  MF " a[32:35], v[224:227], v[196:199], a[32:35]\n\t" \
  "ds_read_b128 v[220:223], %[ra1] offset:14336\n\t" \
  MF " a[64:67], v[224:227], v[200:203], a[64:67]\n\t" \
  "s_add_u32 s81, s81, 128\n\t" \
  "s_add_u32 s82, s82, 128\n\t" \
  MF " a[68:71], v[228:231], v[200:203], a[68:71]\n\t" \
  "s_xor_b32 s86, s86, 0x10000\n\t" \
  "s_add_u32 s87, s80, 2\n\t" \
  MF " a[72:75], v[232:235], v[200:203], a[72:75]\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  MF " a[76:79], v[236:239], v[200:203], a[76:79]\n\t" \
  "v_or_b32 v120, s84, %[voa]\n\t" \
  MF " a[108:111], v[236:239], v[204:207], a[108:111]\n\t" \
  "v_or_b32 v121, s84, %[vob]\n\t" \
  MF " a[104:107], v[232:235], v[204:207], a[104:107]\n\t" \
  "s_mov_b32 s83, s81\n\t" \
  "s_add_u32 m0, s86, 0\n\t" \
  MF " a[100:103], v[228:231], v[204:207], a[100:103]\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  MF " a[96:99], v[224:227], v[204:207], a[96:99]\n\t" \
  "v_xor_b32 %[ra1], 0x10000, %[ra1]\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  MF " a[112:115], v[240:243], v[204:207], a[112:115]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[116:119], v[244:247], v[204:207], a[116:119]\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[120:123], v[248:251], v[204:207], a[120:123]\n\t" \
  "ds_read_b128 v[160:163], %[rb0] offset:0\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[124:127], v[252:255], v[204:207], a[124:127]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 4096\n\t" \
  MF " a[92:95], v[252:255], v[200:203], a[92:95]\n\t" \
  MF " a[88:91], v[248:251], v[200:203], a[88:91]\n\t" \
  MF " a[84:87], v[244:247], v[200:203], a[84:87]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[80:83], v[240:243], v[200:203], a[80:83]\n\t" \
  "ds_read_b128 v[164:167], %[rb0] offset:2048\n\t" \
  MF " a[48:51], v[240:243], v[196:199], a[48:51]\n\t" \
  MF " a[52:55], v[244:247], v[196:199], a[52:55]\n\t" \
  "s_add_u32 s83, s83, %[gas3]\n\t" \
  "s_add_u32 m0, s86, 16384\n\t" \
  MF " a[56:59], v[248:251], v[196:199], a[56:59]\n\t" \
  MF " a[60:63], v[252:255], v[196:199], a[60:63]\n\t" \
  MF " a[28:31], v[252:255], v[192:195], a[28:31]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[24:27], v[248:251], v[192:195], a[24:27]\n\t" \
  "ds_read_b128 v[168:171], %[rb0] offset:4096\n\t" \
  MF " a[20:23], v[244:247], v[192:195], a[20:23]\n\t" \
  MF " a[16:19], v[240:243], v[192:195], a[16:19]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 20480\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[144:147], v[240:243], v[208:211], a[144:147]\n\t" \
  MF " a[148:151], v[244:247], v[208:211], a[148:151]\n\t" \
  "ds_read_b128 v[172:175], %[rb0] offset:6144\n\t" \
  MF " a[152:155], v[248:251], v[208:211], a[152:155]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[156:159], v[252:255], v[208:211], a[156:159]\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[188:191], v[252:255], v[212:215], a[188:191]\n\t" \
  MF " a[184:187], v[248:251], v[212:215], a[184:187]\n\t" \
  "s_mov_b32 s83, s82\n\t" \
  "s_add_u32 m0, s86, 32768\n\t" \
  MF " a[180:183], v[244:247], v[212:215], a[180:183]\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  MF " a[176:179], v[240:243], v[212:215], a[176:179]\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[208:211], v[240:243], v[216:219], a[208:211]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[212:215], v[244:247], v[216:219], a[212:215]\n\t" \
  MF " a[216:219], v[248:251], v[216:219], a[216:219]\n\t" \
  "v_xor_b32 %[rb1], 0x10000, %[rb1]\n\t" \
  MF " a[220:223], v[252:255], v[216:219], a[220:223]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 36864\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[252:255], v[252:255], v[220:223], a[252:255]\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  MF " a[248:251], v[248:251], v[220:223], a[248:251]\n\t" \
  MF " a[244:247], v[244:247], v[220:223], a[244:247]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[240:243], v[240:243], v[220:223], a[240:243]\n\t" \
  MF " a[236:239], v[236:239], v[220:223], a[236:239]\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  MF " a[232:235], v[232:235], v[220:223], a[232:235]\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 49152\n\t" \
  MF " a[228:231], v[228:231], v[220:223], a[228:231]\n\t" \
  MF " a[224:227], v[224:227], v[220:223], a[224:227]\n\t" \
  MF " a[192:195], v[224:227], v[216:219], a[192:195]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[196:199], v[228:231], v[216:219], a[196:199]\n\t" \
  MF " a[200:203], v[232:235], v[216:219], a[200:203]\n\t" \
  MF " a[204:207], v[236:239], v[216:219], a[204:207]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 53248\n\t" \
  MF " a[172:175], v[236:239], v[212:215], a[172:175]\n\t" \
  MF " a[168:171], v[232:235], v[212:215], a[168:171]\n\t" \
  MF " a[164:167], v[228:231], v[212:215], a[164:167]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[160:163], v[224:227], v[212:215], a[160:163]\n\t" \
  MF " a[128:131], v[224:227], v[208:211], a[128:131]\n\t" \
  MF " a[132:135], v[228:231], v[208:211], a[132:135]\n\t" \
  MF " a[136:139], v[232:235], v[208:211], a[136:139]\n\t" \
  MF " a[140:143], v[236:239], v[208:211], a[140:143]\n\t" \
  "s_add_u32 s80, s80, 1\n\t" \
  "s_waitcnt vmcnt(8) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "s_cmp_lt_u32 s80, %[n]\n\t" \
  "s_cbranch_scc1 L_sk_loop%=\n\t" \
  "s_waitcnt vmcnt(0) lgkmcnt(0)\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  ""
#define SK_TILE_ASM_LOOP_WRAP(MF) \
  "v_accvgpr_write_b32 a0, 0\n\t" \
  "v_accvgpr_write_b32 a1, 0\n\t" \
  "v_accvgpr_write_b32 a2, 0\n\t" \
  "v_accvgpr_write_b32 a3, 0\n\t" \
  "v_accvgpr_write_b32 a4, 0\n\t" \
  "v_accvgpr_write_b32 a5, 0\n\t" \
  "v_accvgpr_write_b32 a6, 0\n\t" \
  "v_accvgpr_write_b32 a7, 0\n\t" \
  "v_accvgpr_write_b32 a8, 0\n\t" \
  "v_accvgpr_write_b32 a9, 0\n\t" \
  "v_accvgpr_write_b32 a10, 0\n\t" \
  "v_accvgpr_write_b32 a11, 0\n\t" \
  "v_accvgpr_write_b32 a12, 0\n\t" \
  "v_accvgpr_write_b32 a13, 0\n\t" \
  "v_accvgpr_write_b32 a14, 0\n\t" \
  "v_accvgpr_write_b32 a15, 0\n\t" \
  "v_accvgpr_write_b32 a16, 0\n\t" \
  "v_accvgpr_write_b32 a17, 0\n\t" \
  "v_accvgpr_write_b32 a18, 0\n\t" \
  "v_accvgpr_write_b32 a19, 0\n\t" \
  "v_accvgpr_write_b32 a20, 0\n\t" \
  "v_accvgpr_write_b32 a21, 0\n\t" \
  "v_accvgpr_write_b32 a22, 0\n\t" \
  "v_accvgpr_write_b32 a23, 0\n\t" \
  "v_accvgpr_write_b32 a24, 0\n\t" \
  "v_accvgpr_write_b32 a25, 0\n\t" \
  "v_accvgpr_write_b32 a26, 0\n\t" \
  "v_accvgpr_write_b32 a27, 0\n\t" \
  "v_accvgpr_write_b32 a28, 0\n\t" \
  "v_accvgpr_write_b32 a29, 0\n\t" \
  "v_accvgpr_write_b32 a30, 0\n\t" \
  "v_accvgpr_write_b32 a31, 0\n\t" \
  "v_accvgpr_write_b32 a32, 0\n\t" \
  "v_accvgpr_write_b32 a33, 0\n\t" \
  "v_accvgpr_write_b32 a34, 0\n\t" \
  "v_accvgpr_write_b32 a35, 0\n\t" \
  "v_accvgpr_write_b32 a36, 0\n\t" \
  "v_accvgpr_write_b32 a37, 0\n\t" \
  "v_accvgpr_write_b32 a38, 0\n\t" \
  "v_accvgpr_write_b32 a39, 0\n\t" \
  "v_accvgpr_write_b32 a40, 0\n\t" \
  "v_accvgpr_write_b32 a41, 0\n\t" \
  "v_accvgpr_write_b32 a42, 0\n\t" \
  "v_accvgpr_write_b32 a43, 0\n\t" \
  "v_accvgpr_write_b32 a44, 0\n\t" \
  "v_accvgpr_write_b32 a45, 0\n\t" \
  "v_accvgpr_write_b32 a46, 0\n\t" \
  "v_accvgpr_write_b32 a47, 0\n\t" \
  "v_accvgpr_write_b32 a48, 0\n\t" \
  "v_accvgpr_write_b32 a49, 0\n\t" \
  "v_accvgpr_write_b32 a50, 0\n\t" \
  "v_accvgpr_write_b32 a51, 0\n\t" \
  "v_accvgpr_write_b32 a52, 0\n\t" \
  "v_accvgpr_write_b32 a53, 0\n\t" \
  "v_accvgpr_write_b32 a54, 0\n\t" \
  "v_accvgpr_write_b32 a55, 0\n\t" \
  "v_accvgpr_write_b32 a56, 0\n\t" \
  "v_accvgpr_write_b32 a57, 0\n\t" \
  "v_accvgpr_write_b32 a58, 0\n\t" \
  "v_accvgpr_write_b32 a59, 0\n\t" \
  "v_accvgpr_write_b32 a60, 0\n\t" \
  "v_accvgpr_write_b32 a61, 0\n\t" \
  "v_accvgpr_write_b32 a62, 0\n\t" \
  "v_accvgpr_write_b32 a63, 0\n\t" \
  "v_accvgpr_write_b32 a64, 0\n\t" \
  "v_accvgpr_write_b32 a65, 0\n\t" \
  "v_accvgpr_write_b32 a66, 0\n\t" \
  "v_accvgpr_write_b32 a67, 0\n\t" \
  "v_accvgpr_write_b32 a68, 0\n\t" \
  "v_accvgpr_write_b32 a69, 0\n\t" \
  "v_accvgpr_write_b32 a70, 0\n\t" \
  "v_accvgpr_write_b32 a71, 0\n\t" \
  "v_accvgpr_write_b32 a72, 0\n\t" \
  "v_accvgpr_write_b32 a73, 0\n\t" \
  "v_accvgpr_write_b32 a74, 0\n\t" \
  "v_accvgpr_write_b32 a75, 0\n\t" \
  "v_accvgpr_write_b32 a76, 0\n\t" \
  "v_accvgpr_write_b32 a77, 0\n\t" \
  "v_accvgpr_write_b32 a78, 0\n\t" \
  "v_accvgpr_write_b32 a79, 0\n\t" \
  "v_accvgpr_write_b32 a80, 0\n\t" \
  "v_accvgpr_write_b32 a81, 0\n\t" \
  "v_accvgpr_write_b32 a82, 0\n\t" \
  "v_accvgpr_write_b32 a83, 0\n\t" \
  "v_accvgpr_write_b32 a84, 0\n\t" \
  "v_accvgpr_write_b32 a85, 0\n\t" \
  "v_accvgpr_write_b32 a86, 0\n\t" \
  "v_accvgpr_write_b32 a87, 0\n\t" \
  "v_accvgpr_write_b32 a88, 0\n\t" \
  "v_accvgpr_write_b32 a89, 0\n\t" \
  "v_accvgpr_write_b32 a90, 0\n\t" \
  "v_accvgpr_write_b32 a91, 0\n\t" \
  "v_accvgpr_write_b32 a92, 0\n\t" \
  "v_accvgpr_write_b32 a93, 0\n\t" \
  "v_accvgpr_write_b32 a94, 0\n\t" \
  "v_accvgpr_write_b32 a95, 0\n\t" \
  "v_accvgpr_write_b32 a96, 0\n\t" \
  "v_accvgpr_write_b32 a97, 0\n\t" \
  "v_accvgpr_write_b32 a98, 0\n\t" \
  "v_accvgpr_write_b32 a99, 0\n\t" \
  "v_accvgpr_write_b32 a100, 0\n\t" \
  "v_accvgpr_write_b32 a101, 0\n\t" \
  "v_accvgpr_write_b32 a102, 0\n\t" \
  "v_accvgpr_write_b32 a103, 0\n\t" \
  "v_accvgpr_write_b32 a104, 0\n\t" \
  "v_accvgpr_write_b32 a105, 0\n\t" \
  "v_accvgpr_write_b32 a106, 0\n\t" \
  "v_accvgpr_write_b32 a107, 0\n\t" \
  "v_accvgpr_write_b32 a108, 0\n\t" \
  "v_accvgpr_write_b32 a109, 0\n\t" \
  "v_accvgpr_write_b32 a110, 0\n\t" \
  "v_accvgpr_write_b32 a111, 0\n\t" \
  "v_accvgpr_write_b32 a112, 0\n\t" \
  "v_accvgpr_write_b32 a113, 0\n\t" \
  "v_accvgpr_write_b32 a114, 0\n\t" \
  "v_accvgpr_write_b32 a115, 0\n\t" \
  "v_accvgpr_write_b32 a116, 0\n\t" \
  "v_accvgpr_write_b32 a117, 0\n\t" \
  "v_accvgpr_write_b32 a118, 0\n\t" \
  "v_accvgpr_write_b32 a119, 0\n\t" \
  "v_accvgpr_write_b32 a120, 0\n\t" \
  "v_accvgpr_write_b32 a121, 0\n\t" \
  "v_accvgpr_write_b32 a122, 0\n\t" \
  "v_accvgpr_write_b32 a123, 0\n\t" \
  "v_accvgpr_write_b32 a124, 0\n\t" \
  "v_accvgpr_write_b32 a125, 0\n\t" \
  "v_accvgpr_write_b32 a126, 0\n\t" \
  "v_accvgpr_write_b32 a127, 0\n\t" \
  "v_accvgpr_write_b32 a128, 0\n\t" \
  "v_accvgpr_write_b32 a129, 0\n\t" \
  "v_accvgpr_write_b32 a130, 0\n\t" \
  "v_accvgpr_write_b32 a131, 0\n\t" \
  "v_accvgpr_write_b32 a132, 0\n\t" \
  "v_accvgpr_write_b32 a133, 0\n\t" \
  "v_accvgpr_write_b32 a134, 0\n\t" \
  "v_accvgpr_write_b32 a135, 0\n\t" \
  "v_accvgpr_write_b32 a136, 0\n\t" \
  "v_accvgpr_write_b32 a137, 0\n\t" \
  "v_accvgpr_write_b32 a138, 0\n\t" \
  "v_accvgpr_write_b32 a139, 0\n\t" \
  "v_accvgpr_write_b32 a140, 0\n\t" \
  "v_accvgpr_write_b32 a141, 0\n\t" \
  "v_accvgpr_write_b32 a142, 0\n\t" \
  "v_accvgpr_write_b32 a143, 0\n\t" \
  "v_accvgpr_write_b32 a144, 0\n\t" \
  "v_accvgpr_write_b32 a145, 0\n\t" \
  "v_accvgpr_write_b32 a146, 0\n\t" \
  "v_accvgpr_write_b32 a147, 0\n\t" \
  "v_accvgpr_write_b32 a148, 0\n\t" \
  "v_accvgpr_write_b32 a149, 0\n\t" \
  "v_accvgpr_write_b32 a150, 0\n\t" \
  "v_accvgpr_write_b32 a151, 0\n\t" \
  "v_accvgpr_write_b32 a152, 0\n\t" \
  "v_accvgpr_write_b32 a153, 0\n\t" \
  "v_accvgpr_write_b32 a154, 0\n\t" \
  "v_accvgpr_write_b32 a155, 0\n\t" \
  "v_accvgpr_write_b32 a156, 0\n\t" \
  "v_accvgpr_write_b32 a157, 0\n\t" \
  "v_accvgpr_write_b32 a158, 0\n\t" \
  "v_accvgpr_write_b32 a159, 0\n\t" \
  "v_accvgpr_write_b32 a160, 0\n\t" \
  "v_accvgpr_write_b32 a161, 0\n\t" \
  "v_accvgpr_write_b32 a162, 0\n\t" \
  "v_accvgpr_write_b32 a163, 0\n\t" \
  "v_accvgpr_write_b32 a164, 0\n\t" \
  "v_accvgpr_write_b32 a165, 0\n\t" \
  "v_accvgpr_write_b32 a166, 0\n\t" \
  "v_accvgpr_write_b32 a167, 0\n\t" \
  "v_accvgpr_write_b32 a168, 0\n\t" \
  "v_accvgpr_write_b32 a169, 0\n\t" \
  "v_accvgpr_write_b32 a170, 0\n\t" \
  "v_accvgpr_write_b32 a171, 0\n\t" \
  "v_accvgpr_write_b32 a172, 0\n\t" \
  "v_accvgpr_write_b32 a173, 0\n\t" \
  "v_accvgpr_write_b32 a174, 0\n\t" \
  "v_accvgpr_write_b32 a175, 0\n\t" \
  "v_accvgpr_write_b32 a176, 0\n\t" \
  "v_accvgpr_write_b32 a177, 0\n\t" \
  "v_accvgpr_write_b32 a178, 0\n\t" \
  "v_accvgpr_write_b32 a179, 0\n\t" \
  "v_accvgpr_write_b32 a180, 0\n\t" \
  "v_accvgpr_write_b32 a181, 0\n\t" \
  "v_accvgpr_write_b32 a182, 0\n\t" \
  "v_accvgpr_write_b32 a183, 0\n\t" \
  "v_accvgpr_write_b32 a184, 0\n\t" \
  "v_accvgpr_write_b32 a185, 0\n\t" \
  "v_accvgpr_write_b32 a186, 0\n\t" \
  "v_accvgpr_write_b32 a187, 0\n\t" \
  "v_accvgpr_write_b32 a188, 0\n\t" \
  "v_accvgpr_write_b32 a189, 0\n\t" \
  "v_accvgpr_write_b32 a190, 0\n\t" \
  "v_accvgpr_write_b32 a191, 0\n\t" \
  "v_accvgpr_write_b32 a192, 0\n\t" \
  "v_accvgpr_write_b32 a193, 0\n\t" \
  "v_accvgpr_write_b32 a194, 0\n\t" \
  "v_accvgpr_write_b32 a195, 0\n\t" \
  "v_accvgpr_write_b32 a196, 0\n\t" \
  "v_accvgpr_write_b32 a197, 0\n\t" \
  "v_accvgpr_write_b32 a198, 0\n\t" \
  "v_accvgpr_write_b32 a199, 0\n\t" \
  "v_accvgpr_write_b32 a200, 0\n\t" \
  "v_accvgpr_write_b32 a201, 0\n\t" \
  "v_accvgpr_write_b32 a202, 0\n\t" \
  "v_accvgpr_write_b32 a203, 0\n\t" \
  "v_accvgpr_write_b32 a204, 0\n\t" \
  "v_accvgpr_write_b32 a205, 0\n\t" \
  "v_accvgpr_write_b32 a206, 0\n\t" \
  "v_accvgpr_write_b32 a207, 0\n\t" \
  "v_accvgpr_write_b32 a208, 0\n\t" \
  "v_accvgpr_write_b32 a209, 0\n\t" \
  "v_accvgpr_write_b32 a210, 0\n\t" \
  "v_accvgpr_write_b32 a211, 0\n\t" \
  "v_accvgpr_write_b32 a212, 0\n\t" \
  "v_accvgpr_write_b32 a213, 0\n\t" \
  "v_accvgpr_write_b32 a214, 0\n\t" \
  "v_accvgpr_write_b32 a215, 0\n\t" \
  "v_accvgpr_write_b32 a216, 0\n\t" \
  "v_accvgpr_write_b32 a217, 0\n\t" \
  "v_accvgpr_write_b32 a218, 0\n\t" \
  "v_accvgpr_write_b32 a219, 0\n\t" \
  "v_accvgpr_write_b32 a220, 0\n\t" \
  "v_accvgpr_write_b32 a221, 0\n\t" \
  "v_accvgpr_write_b32 a222, 0\n\t" \
  "v_accvgpr_write_b32 a223, 0\n\t" \
  "v_accvgpr_write_b32 a224, 0\n\t" \
  "v_accvgpr_write_b32 a225, 0\n\t" \
  "v_accvgpr_write_b32 a226, 0\n\t" \
  "v_accvgpr_write_b32 a227, 0\n\t" \
  "v_accvgpr_write_b32 a228, 0\n\t" \
  "v_accvgpr_write_b32 a229, 0\n\t" \
  "v_accvgpr_write_b32 a230, 0\n\t" \
  "v_accvgpr_write_b32 a231, 0\n\t" \
  "v_accvgpr_write_b32 a232, 0\n\t" \
  "v_accvgpr_write_b32 a233, 0\n\t" \
  "v_accvgpr_write_b32 a234, 0\n\t" \
  "v_accvgpr_write_b32 a235, 0\n\t" \
  "v_accvgpr_write_b32 a236, 0\n\t" \
  "v_accvgpr_write_b32 a237, 0\n\t" \
  "v_accvgpr_write_b32 a238, 0\n\t" \
  "v_accvgpr_write_b32 a239, 0\n\t" \
  "v_accvgpr_write_b32 a240, 0\n\t" \
  "v_accvgpr_write_b32 a241, 0\n\t" \
  "v_accvgpr_write_b32 a242, 0\n\t" \
  "v_accvgpr_write_b32 a243, 0\n\t" \
  "v_accvgpr_write_b32 a244, 0\n\t" \
  "v_accvgpr_write_b32 a245, 0\n\t" \
  "v_accvgpr_write_b32 a246, 0\n\t" \
  "v_accvgpr_write_b32 a247, 0\n\t" \
  "v_accvgpr_write_b32 a248, 0\n\t" \
  "v_accvgpr_write_b32 a249, 0\n\t" \
  "v_accvgpr_write_b32 a250, 0\n\t" \
  "v_accvgpr_write_b32 a251, 0\n\t" \
  "v_accvgpr_write_b32 a252, 0\n\t" \
  "v_accvgpr_write_b32 a253, 0\n\t" \
  "v_accvgpr_write_b32 a254, 0\n\t" \
  "v_accvgpr_write_b32 a255, 0\n\t" \
  "s_mov_b32 s80, 0\n\t" \
  "s_xor_b32 s86, %[lds], 0x10000\n\t" \
  "s_cmp_eq_u32 %[wrap], 1\n\t" \
  "s_cselect_b32 s85, %[back], 128\n\t" \
  "s_add_u32 s81, %[ga0], s85\n\t" \
  "s_add_u32 s82, %[gb0], s85\n\t" \
  "s_add_u32 s87, s80, 1\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "v_or_b32 v120, s84, %[voa]\n\t" \
  "v_or_b32 v121, s84, %[vob]\n\t" \
  "s_waitcnt vmcnt(8)\n\t" \
  "s_barrier\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  "ds_read_b128 v[160:163], %[rb0] offset:0\n\t" \
  "ds_read_b128 v[164:167], %[rb0] offset:2048\n\t" \
  "ds_read_b128 v[168:171], %[rb0] offset:4096\n\t" \
  "ds_read_b128 v[172:175], %[rb0] offset:6144\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  "s_nop 7\n\t" \
  "L_sk_loop%=:\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[0:3], v[160:163], v[128:131], a[0:3]\n\t" \
  "ds_read_b128 v[176:179], %[rb0] offset:8192\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[4:7], v[164:167], v[128:131], a[4:7]\n\t" \
  "ds_read_b128 v[180:183], %[rb0] offset:10240\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[8:11], v[168:171], v[128:131], a[8:11]\n\t" \
  "ds_read_b128 v[184:187], %[rb0] offset:12288\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[12:15], v[172:175], v[128:131], a[12:15]\n\t" \
  "ds_read_b128 v[188:191], %[rb0] offset:14336\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[44:47], v[172:175], v[132:135], a[44:47]\n\t" \
  "ds_read_b128 v[144:147], %[ra0] offset:8192\n\t" \
  MF " a[40:43], v[168:171], v[132:135], a[40:43]\n\t" \
  "ds_read_b128 v[148:151], %[ra0] offset:10240\n\t" \
  MF " a[36:39], v[164:167], v[132:135], a[36:39]\n\t" \
  "ds_read_b128 v[152:155], %[ra0] offset:12288\n\t" \
  MF " a[32:35], v[160:163], v[132:135], a[32:35]\n\t" \
  "ds_read_b128 v[156:159], %[ra0] offset:14336\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[64:67], v[160:163], v[136:139], a[64:67]\n\t" \
  "s_add_u32 s83, s81, %[gas2]\n\t" \
  "s_add_u32 m0, s86, 8192\n\t" \
  MF " a[68:71], v[164:167], v[136:139], a[68:71]\n\t" \
  "ds_read_b128 v[192:195], %[ra1] offset:0\n\t" \
  MF " a[72:75], v[168:171], v[136:139], a[72:75]\n\t" \
  "v_xor_b32 %[ra0], 0x10000, %[ra0]\n\t" \
  MF " a[76:79], v[172:175], v[136:139], a[76:79]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[108:111], v[172:175], v[140:143], a[108:111]\n\t" \
  MF " a[104:107], v[168:171], v[140:143], a[104:107]\n\t" \
  MF " a[100:103], v[164:167], v[140:143], a[100:103]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 12288\n\t" \
  MF " a[96:99], v[160:163], v[140:143], a[96:99]\n\t" \
  "ds_read_b128 v[224:227], %[rb1] offset:0\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[112:115], v[176:179], v[140:143], a[112:115]\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  MF " a[116:119], v[180:183], v[140:143], a[116:119]\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[120:123], v[184:187], v[140:143], a[120:123]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[124:127], v[188:191], v[140:143], a[124:127]\n\t" \
  MF " a[92:95], v[188:191], v[136:139], a[92:95]\n\t" \
  "ds_read_b128 v[228:231], %[rb1] offset:2048\n\t" \
  MF " a[88:91], v[184:187], v[136:139], a[88:91]\n\t" \
  "s_add_u32 s83, s83, %[gas3]\n\t" \
  "s_add_u32 m0, s86, 24576\n\t" \
  MF " a[84:87], v[180:183], v[136:139], a[84:87]\n\t" \
  MF " a[80:83], v[176:179], v[136:139], a[80:83]\n\t" \
  MF " a[48:51], v[176:179], v[132:135], a[48:51]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[52:55], v[180:183], v[132:135], a[52:55]\n\t" \
  MF " a[56:59], v[184:187], v[132:135], a[56:59]\n\t" \
  "ds_read_b128 v[232:235], %[rb1] offset:4096\n\t" \
  MF " a[60:63], v[188:191], v[132:135], a[60:63]\n\t" \
  MF " a[28:31], v[188:191], v[128:131], a[28:31]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 28672\n\t" \
  MF " a[24:27], v[184:187], v[128:131], a[24:27]\n\t" \
  MF " a[20:23], v[180:183], v[128:131], a[20:23]\n\t" \
  MF " a[16:19], v[176:179], v[128:131], a[16:19]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[144:147], v[176:179], v[144:147], a[144:147]\n\t" \
  "ds_read_b128 v[236:239], %[rb1] offset:6144\n\t" \
  MF " a[148:151], v[180:183], v[144:147], a[148:151]\n\t" \
  MF " a[152:155], v[184:187], v[144:147], a[152:155]\n\t" \
  MF " a[156:159], v[188:191], v[144:147], a[156:159]\n\t" \
  "s_add_u32 s83, s82, %[gbs2]\n\t" \
  "s_add_u32 m0, s86, 40960\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[188:191], v[188:191], v[148:151], a[188:191]\n\t" \
  MF " a[184:187], v[184:187], v[148:151], a[184:187]\n\t" \
  "ds_read_b128 v[196:199], %[ra1] offset:2048\n\t" \
  MF " a[180:183], v[180:183], v[148:151], a[180:183]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[176:179], v[176:179], v[148:151], a[176:179]\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[208:211], v[176:179], v[152:155], a[208:211]\n\t" \
  "v_xor_b32 %[rb0], 0x10000, %[rb0]\n\t" \
  MF " a[212:215], v[180:183], v[152:155], a[212:215]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 45056\n\t" \
  MF " a[216:219], v[184:187], v[152:155], a[216:219]\n\t" \
  MF " a[220:223], v[188:191], v[152:155], a[220:223]\n\t" \
  "ds_read_b128 v[200:203], %[ra1] offset:4096\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[252:255], v[188:191], v[156:159], a[252:255]\n\t" \
  MF " a[248:251], v[184:187], v[156:159], a[248:251]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[244:247], v[180:183], v[156:159], a[244:247]\n\t" \
  MF " a[240:243], v[176:179], v[156:159], a[240:243]\n\t" \
  MF " a[236:239], v[172:175], v[156:159], a[236:239]\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 57344\n\t" \
  MF " a[232:235], v[168:171], v[156:159], a[232:235]\n\t" \
  "ds_read_b128 v[204:207], %[ra1] offset:6144\n\t" \
  MF " a[228:231], v[164:167], v[156:159], a[228:231]\n\t" \
  MF " a[224:227], v[160:163], v[156:159], a[224:227]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[192:195], v[160:163], v[152:155], a[192:195]\n\t" \
  MF " a[196:199], v[164:167], v[152:155], a[196:199]\n\t" \
  MF " a[200:203], v[168:171], v[152:155], a[200:203]\n\t" \
  MF " a[204:207], v[172:175], v[152:155], a[204:207]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 61440\n\t" \
  MF " a[172:175], v[172:175], v[148:151], a[172:175]\n\t" \
  MF " a[168:171], v[168:171], v[148:151], a[168:171]\n\t" \
  MF " a[164:167], v[164:167], v[148:151], a[164:167]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[160:163], v[160:163], v[148:151], a[160:163]\n\t" \
  MF " a[128:131], v[160:163], v[144:147], a[128:131]\n\t" \
  MF " a[132:135], v[164:167], v[144:147], a[132:135]\n\t" \
  MF " a[136:139], v[168:171], v[144:147], a[136:139]\n\t" \
  MF " a[140:143], v[172:175], v[144:147], a[140:143]\n\t" \
  "s_waitcnt vmcnt(8) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  MF " a[0:3], v[224:227], v[192:195], a[0:3]\n\t" \
  "ds_read_b128 v[240:243], %[rb1] offset:8192\n\t" \
  MF " a[4:7], v[228:231], v[192:195], a[4:7]\n\t" \
  "ds_read_b128 v[244:247], %[rb1] offset:10240\n\t" \
  MF " a[8:11], v[232:235], v[192:195], a[8:11]\n\t" \
  "ds_read_b128 v[248:251], %[rb1] offset:12288\n\t" \
  MF " a[12:15], v[236:239], v[192:195], a[12:15]\n\t" \
  "ds_read_b128 v[252:255], %[rb1] offset:14336\n\t" \
  MF " a[44:47], v[236:239], v[196:199], a[44:47]\n\t" \
  "ds_read_b128 v[208:211], %[ra1] offset:8192\n\t" \
  MF " a[40:43], v[232:235], v[196:199], a[40:43]\n\t" \
  "ds_read_b128 v[212:215], %[ra1] offset:10240\n\t" \
  MF " a[36:39], v[228:231], v[196:199], a[36:39]\n\t" \
  "ds_read_b128 v[216:219], %[ra1] offset:12288\n\t" \
  MF " a[32:35], v[224:227], v[196:199], a[32:35]\n\t" \
  "ds_read_b128 v[220:223], %[ra1] offset:14336\n\t" \
  MF " a[64:67], v[224:227], v[200:203], a[64:67]\n\t" \
  "s_add_u32 s87, s80, 2\n\t" \
  "s_cmp_eq_u32 s87, %[wrap]\n\t" \
  "s_cselect_b32 s85, %[back], 128\n\t" \
  MF " a[68:71], v[228:231], v[200:203], a[68:71]\n\t" \
  "s_add_u32 s81, s81, s85\n\t" \
  "s_add_u32 s82, s82, s85\n\t" \
  MF " a[72:75], v[232:235], v[200:203], a[72:75]\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "s_xor_b32 s86, s86, 0x10000\n\t" \
  MF " a[76:79], v[236:239], v[200:203], a[76:79]\n\t" \
  "v_or_b32 v120, s84, %[voa]\n\t" \
  MF " a[108:111], v[236:239], v[204:207], a[108:111]\n\t" \
  "v_or_b32 v121, s84, %[vob]\n\t" \
  MF " a[104:107], v[232:235], v[204:207], a[104:107]\n\t" \
  "s_mov_b32 s83, s81\n\t" \
  "s_add_u32 m0, s86, 0\n\t" \
  MF " a[100:103], v[228:231], v[204:207], a[100:103]\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  MF " a[96:99], v[224:227], v[204:207], a[96:99]\n\t" \
  "v_xor_b32 %[ra1], 0x10000, %[ra1]\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  MF " a[112:115], v[240:243], v[204:207], a[112:115]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[116:119], v[244:247], v[204:207], a[116:119]\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[120:123], v[248:251], v[204:207], a[120:123]\n\t" \
  "ds_read_b128 v[160:163], %[rb0] offset:0\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[124:127], v[252:255], v[204:207], a[124:127]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 4096\n\t" \
  MF " a[92:95], v[252:255], v[200:203], a[92:95]\n\t" \
  MF " a[88:91], v[248:251], v[200:203], a[88:91]\n\t" \
  MF " a[84:87], v[244:247], v[200:203], a[84:87]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[80:83], v[240:243], v[200:203], a[80:83]\n\t" \
  "ds_read_b128 v[164:167], %[rb0] offset:2048\n\t" \
  MF " a[48:51], v[240:243], v[196:199], a[48:51]\n\t" \
  MF " a[52:55], v[244:247], v[196:199], a[52:55]\n\t" \
  "s_add_u32 s83, s83, %[gas3]\n\t" \
  "s_add_u32 m0, s86, 16384\n\t" \
  MF " a[56:59], v[248:251], v[196:199], a[56:59]\n\t" \
  MF " a[60:63], v[252:255], v[196:199], a[60:63]\n\t" \
  MF " a[28:31], v[252:255], v[192:195], a[28:31]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[24:27], v[248:251], v[192:195], a[24:27]\n\t" \
  "ds_read_b128 v[168:171], %[rb0] offset:4096\n\t" \
  MF " a[20:23], v[244:247], v[192:195], a[20:23]\n\t" \
  MF " a[16:19], v[240:243], v[192:195], a[16:19]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 20480\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[144:147], v[240:243], v[208:211], a[144:147]\n\t" \
  MF " a[148:151], v[244:247], v[208:211], a[148:151]\n\t" \
  "ds_read_b128 v[172:175], %[rb0] offset:6144\n\t" \
  MF " a[152:155], v[248:251], v[208:211], a[152:155]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[156:159], v[252:255], v[208:211], a[156:159]\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[188:191], v[252:255], v[212:215], a[188:191]\n\t" \
  MF " a[184:187], v[248:251], v[212:215], a[184:187]\n\t" \
  "s_mov_b32 s83, s82\n\t" \
  "s_add_u32 m0, s86, 32768\n\t" \
  MF " a[180:183], v[244:247], v[212:215], a[180:183]\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  MF " a[176:179], v[240:243], v[212:215], a[176:179]\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[208:211], v[240:243], v[216:219], a[208:211]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[212:215], v[244:247], v[216:219], a[212:215]\n\t" \
  MF " a[216:219], v[248:251], v[216:219], a[216:219]\n\t" \
  "v_xor_b32 %[rb1], 0x10000, %[rb1]\n\t" \
  MF " a[220:223], v[252:255], v[216:219], a[220:223]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 36864\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[252:255], v[252:255], v[220:223], a[252:255]\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  MF " a[248:251], v[248:251], v[220:223], a[248:251]\n\t" \
  MF " a[244:247], v[244:247], v[220:223], a[244:247]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[240:243], v[240:243], v[220:223], a[240:243]\n\t" \
  MF " a[236:239], v[236:239], v[220:223], a[236:239]\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  MF " a[232:235], v[232:235], v[220:223], a[232:235]\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 49152\n\t" \
  MF " a[228:231], v[228:231], v[220:223], a[228:231]\n\t" \
  MF " a[224:227], v[224:227], v[220:223], a[224:227]\n\t" \
  MF " a[192:195], v[224:227], v[216:219], a[192:195]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[196:199], v[228:231], v[216:219], a[196:199]\n\t" \
  MF " a[200:203], v[232:235], v[216:219], a[200:203]\n\t" \
  MF " a[204:207], v[236:239], v[216:219], a[204:207]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 53248\n\t" \
  MF " a[172:175], v[236:239], v[212:215], a[172:175]\n\t" \
  MF " a[168:171], v[232:235], v[212:215], a[168:171]\n\t" \
  MF " a[164:167], v[228:231], v[212:215], a[164:167]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[160:163], v[224:227], v[212:215], a[160:163]\n\t" \
  MF " a[128:131], v[224:227], v[208:211], a[128:131]\n\t" \
  MF " a[132:135], v[228:231], v[208:211], a[132:135]\n\t" \
  MF " a[136:139], v[232:235], v[208:211], a[136:139]\n\t" \
  MF " a[140:143], v[236:239], v[208:211], a[140:143]\n\t" \
  "s_add_u32 s80, s80, 1\n\t" \
  "s_waitcnt vmcnt(8) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "s_cmp_lt_u32 s80, %[n]\n\t" \
  "s_cbranch_scc1 L_sk_loop%=\n\t" \
  "s_waitcnt vmcnt(0) lgkmcnt(0)\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  ""
#define SK_TILE_ASM_LOOP_LOW(MF) \
  "v_accvgpr_write_b32 a0, 0\n\t" \
  "v_accvgpr_write_b32 a1, 0\n\t" \
  "v_accvgpr_write_b32 a2, 0\n\t" \
  "v_accvgpr_write_b32 a3, 0\n\t" \
  "v_accvgpr_write_b32 a4, 0\n\t" \
  "v_accvgpr_write_b32 a5, 0\n\t" \
  "v_accvgpr_write_b32 a6, 0\n\t" \
  "v_accvgpr_write_b32 a7, 0\n\t" \
  "v_accvgpr_write_b32 a8, 0\n\t" \
  "v_accvgpr_write_b32 a9, 0\n\t" \
  "v_accvgpr_write_b32 a10, 0\n\t" \
  "v_accvgpr_write_b32 a11, 0\n\t" \
  "v_accvgpr_write_b32 a12, 0\n\t" \
  "v_accvgpr_write_b32 a13, 0\n\t" \
  "v_accvgpr_write_b32 a14, 0\n\t" \
  "v_accvgpr_write_b32 a15, 0\n\t" \
  "v_accvgpr_write_b32 a16, 0\n\t" \
  "v_accvgpr_write_b32 a17, 0\n\t" \
  "v_accvgpr_write_b32 a18, 0\n\t" \
  "v_accvgpr_write_b32 a19, 0\n\t" \
  "v_accvgpr_write_b32 a20, 0\n\t" \
  "v_accvgpr_write_b32 a21, 0\n\t" \
  "v_accvgpr_write_b32 a22, 0\n\t" \
  "v_accvgpr_write_b32 a23, 0\n\t" \
  "v_accvgpr_write_b32 a24, 0\n\t" \
  "v_accvgpr_write_b32 a25, 0\n\t" \
  "v_accvgpr_write_b32 a26, 0\n\t" \
  "v_accvgpr_write_b32 a27, 0\n\t" \
  "v_accvgpr_write_b32 a28, 0\n\t" \
  "v_accvgpr_write_b32 a29, 0\n\t" \
  "v_accvgpr_write_b32 a30, 0\n\t" \
  "v_accvgpr_write_b32 a31, 0\n\t" \
  "v_accvgpr_write_b32 a32, 0\n\t" \
  "v_accvgpr_write_b32 a33, 0\n\t" \
  "v_accvgpr_write_b32 a34, 0\n\t" \
  "v_accvgpr_write_b32 a35, 0\n\t" \
  "v_accvgpr_write_b32 a36, 0\n\t" \
  "v_accvgpr_write_b32 a37, 0\n\t" \
  "v_accvgpr_write_b32 a38, 0\n\t" \
  "v_accvgpr_write_b32 a39, 0\n\t" \
  "v_accvgpr_write_b32 a40, 0\n\t" \
  "v_accvgpr_write_b32 a41, 0\n\t" \
  "v_accvgpr_write_b32 a42, 0\n\t" \
  "v_accvgpr_write_b32 a43, 0\n\t" \
  "v_accvgpr_write_b32 a44, 0\n\t" \
  "v_accvgpr_write_b32 a45, 0\n\t" \
  "v_accvgpr_write_b32 a46, 0\n\t" \
  "v_accvgpr_write_b32 a47, 0\n\t" \
  "v_accvgpr_write_b32 a48, 0\n\t" \
  "v_accvgpr_write_b32 a49, 0\n\t" \
  "v_accvgpr_write_b32 a50, 0\n\t" \
  "v_accvgpr_write_b32 a51, 0\n\t" \
  "v_accvgpr_write_b32 a52, 0\n\t" \
  "v_accvgpr_write_b32 a53, 0\n\t" \
  "v_accvgpr_write_b32 a54, 0\n\t" \
  "v_accvgpr_write_b32 a55, 0\n\t" \
  "v_accvgpr_write_b32 a56, 0\n\t" \
  "v_accvgpr_write_b32 a57, 0\n\t" \
  "v_accvgpr_write_b32 a58, 0\n\t" \
  "v_accvgpr_write_b32 a59, 0\n\t" \
  "v_accvgpr_write_b32 a60, 0\n\t" \
  "v_accvgpr_write_b32 a61, 0\n\t" \
  "v_accvgpr_write_b32 a62, 0\n\t" \
  "v_accvgpr_write_b32 a63, 0\n\t" \
  "v_accvgpr_write_b32 a64, 0\n\t" \
  "v_accvgpr_write_b32 a65, 0\n\t" \
  "v_accvgpr_write_b32 a66, 0\n\t" \
  "v_accvgpr_write_b32 a67, 0\n\t" \
  "v_accvgpr_write_b32 a68, 0\n\t" \
  "v_accvgpr_write_b32 a69, 0\n\t" \
  "v_accvgpr_write_b32 a70, 0\n\t" \
  "v_accvgpr_write_b32 a71, 0\n\t" \
  "v_accvgpr_write_b32 a72, 0\n\t" \
  "v_accvgpr_write_b32 a73, 0\n\t" \
  "v_accvgpr_write_b32 a74, 0\n\t" \
  "v_accvgpr_write_b32 a75, 0\n\t" \
  "v_accvgpr_write_b32 a76, 0\n\t" \
  "v_accvgpr_write_b32 a77, 0\n\t" \
  "v_accvgpr_write_b32 a78, 0\n\t" \
  "v_accvgpr_write_b32 a79, 0\n\t" \
  "v_accvgpr_write_b32 a80, 0\n\t" \
  "v_accvgpr_write_b32 a81, 0\n\t" \
  "v_accvgpr_write_b32 a82, 0\n\t" \
  "v_accvgpr_write_b32 a83, 0\n\t" \
  "v_accvgpr_write_b32 a84, 0\n\t" \
  "v_accvgpr_write_b32 a85, 0\n\t" \
  "v_accvgpr_write_b32 a86, 0\n\t" \
  "v_accvgpr_write_b32 a87, 0\n\t" \
  "v_accvgpr_write_b32 a88, 0\n\t" \
  "v_accvgpr_write_b32 a89, 0\n\t" \
  "v_accvgpr_write_b32 a90, 0\n\t" \
  "v_accvgpr_write_b32 a91, 0\n\t" \
  "v_accvgpr_write_b32 a92, 0\n\t" \
  "v_accvgpr_write_b32 a93, 0\n\t" \
  "v_accvgpr_write_b32 a94, 0\n\t" \
  "v_accvgpr_write_b32 a95, 0\n\t" \
  "v_accvgpr_write_b32 a96, 0\n\t" \
  "v_accvgpr_write_b32 a97, 0\n\t" \
  "v_accvgpr_write_b32 a98, 0\n\t" \
  "v_accvgpr_write_b32 a99, 0\n\t" \
  "v_accvgpr_write_b32 a100, 0\n\t" \
  "v_accvgpr_write_b32 a101, 0\n\t" \
  "v_accvgpr_write_b32 a102, 0\n\t" \
  "v_accvgpr_write_b32 a103, 0\n\t" \
  "v_accvgpr_write_b32 a104, 0\n\t" \
  "v_accvgpr_write_b32 a105, 0\n\t" \
  "v_accvgpr_write_b32 a106, 0\n\t" \
  "v_accvgpr_write_b32 a107, 0\n\t" \
  "v_accvgpr_write_b32 a108, 0\n\t" \
  "v_accvgpr_write_b32 a109, 0\n\t" \
  "v_accvgpr_write_b32 a110, 0\n\t" \
  "v_accvgpr_write_b32 a111, 0\n\t" \
  "v_accvgpr_write_b32 a112, 0\n\t" \
  "v_accvgpr_write_b32 a113, 0\n\t" \
  "v_accvgpr_write_b32 a114, 0\n\t" \
  "v_accvgpr_write_b32 a115, 0\n\t" \
  "v_accvgpr_write_b32 a116, 0\n\t" \
  "v_accvgpr_write_b32 a117, 0\n\t" \
  "v_accvgpr_write_b32 a118, 0\n\t" \
  "v_accvgpr_write_b32 a119, 0\n\t" \
  "v_accvgpr_write_b32 a120, 0\n\t" \
  "v_accvgpr_write_b32 a121, 0\n\t" \
  "v_accvgpr_write_b32 a122, 0\n\t" \
  "v_accvgpr_write_b32 a123, 0\n\t" \
  "v_accvgpr_write_b32 a124, 0\n\t" \
  "v_accvgpr_write_b32 a125, 0\n\t" \
  "v_accvgpr_write_b32 a126, 0\n\t" \
  "v_accvgpr_write_b32 a127, 0\n\t" \
  "s_mov_b32 s80, 0\n\t" \
  "s_xor_b32 s86, %[lds], 0x10000\n\t" \
  "s_cmp_eq_u32 %[wrap], 1\n\t" \
  "s_cselect_b32 s85, %[back], 128\n\t" \
  "s_add_u32 s81, %[ga0], s85\n\t" \
  "s_add_u32 s82, %[gb0], s85\n\t" \
  "s_add_u32 s87, s80, 1\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "v_or_b32 v120, s84, %[voa]\n\t" \
  "v_or_b32 v121, s84, %[vob]\n\t" \
  "s_waitcnt vmcnt(8)\n\t" \
  "s_barrier\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  "ds_read_b128 v[160:163], %[rb0] offset:0\n\t" \
  "ds_read_b128 v[164:167], %[rb0] offset:2048\n\t" \
  "ds_read_b128 v[168:171], %[rb0] offset:4096\n\t" \
  "ds_read_b128 v[172:175], %[rb0] offset:6144\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  "s_nop 7\n\t" \
  "L_sk_loop%=:\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[0:3], v[160:163], v[128:131], a[0:3]\n\t" \
  "ds_read_b128 v[176:179], %[rb0] offset:8192\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[4:7], v[164:167], v[128:131], a[4:7]\n\t" \
  "ds_read_b128 v[180:183], %[rb0] offset:10240\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[8:11], v[168:171], v[128:131], a[8:11]\n\t" \
  "ds_read_b128 v[184:187], %[rb0] offset:12288\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[12:15], v[172:175], v[128:131], a[12:15]\n\t" \
  "ds_read_b128 v[188:191], %[rb0] offset:14336\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[44:47], v[172:175], v[132:135], a[44:47]\n\t" \
  "s_add_u32 s83, s82, %[gbs2]\n\t" \
  "s_add_u32 m0, s86, 40960\n\t" \
  MF " a[40:43], v[168:171], v[132:135], a[40:43]\n\t" \
  "ds_read_b128 v[192:195], %[ra1] offset:0\n\t" \
  MF " a[36:39], v[164:167], v[132:135], a[36:39]\n\t" \
  "v_xor_b32 %[ra0], 0x10000, %[ra0]\n\t" \
  MF " a[32:35], v[160:163], v[132:135], a[32:35]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[64:67], v[160:163], v[136:139], a[64:67]\n\t" \
  "ds_read_b128 v[224:227], %[rb1] offset:0\n\t" \
  MF " a[68:71], v[164:167], v[136:139], a[68:71]\n\t" \
  MF " a[72:75], v[168:171], v[136:139], a[72:75]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 45056\n\t" \
  MF " a[76:79], v[172:175], v[136:139], a[76:79]\n\t" \
  "ds_read_b128 v[228:231], %[rb1] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[108:111], v[172:175], v[140:143], a[108:111]\n\t" \
  MF " a[104:107], v[168:171], v[140:143], a[104:107]\n\t" \
  "ds_read_b128 v[232:235], %[rb1] offset:4096\n\t" \
  MF " a[100:103], v[164:167], v[140:143], a[100:103]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[96:99], v[160:163], v[140:143], a[96:99]\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[112:115], v[176:179], v[140:143], a[112:115]\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[116:119], v[180:183], v[140:143], a[116:119]\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 57344\n\t" \
  "s_waitcnt lgkmcnt(5)\n\t" \
  MF " a[120:123], v[184:187], v[140:143], a[120:123]\n\t" \
  "ds_read_b128 v[236:239], %[rb1] offset:6144\n\t" \
  "s_waitcnt lgkmcnt(5)\n\t" \
  MF " a[124:127], v[188:191], v[140:143], a[124:127]\n\t" \
  MF " a[92:95], v[188:191], v[136:139], a[92:95]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[88:91], v[184:187], v[136:139], a[88:91]\n\t" \
  "ds_read_b128 v[196:199], %[ra1] offset:2048\n\t" \
  MF " a[84:87], v[180:183], v[136:139], a[84:87]\n\t" \
  "v_xor_b32 %[rb0], 0x10000, %[rb0]\n\t" \
  MF " a[80:83], v[176:179], v[136:139], a[80:83]\n\t" \
  "ds_read_b128 v[200:203], %[ra1] offset:4096\n\t" \
  MF " a[48:51], v[176:179], v[132:135], a[48:51]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 61440\n\t" \
  MF " a[52:55], v[180:183], v[132:135], a[52:55]\n\t" \
  MF " a[56:59], v[184:187], v[132:135], a[56:59]\n\t" \
  "ds_read_b128 v[204:207], %[ra1] offset:6144\n\t" \
  MF " a[60:63], v[188:191], v[132:135], a[60:63]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[28:31], v[188:191], v[128:131], a[28:31]\n\t" \
  MF " a[24:27], v[184:187], v[128:131], a[24:27]\n\t" \
  MF " a[20:23], v[180:183], v[128:131], a[20:23]\n\t" \
  MF " a[16:19], v[176:179], v[128:131], a[16:19]\n\t" \
  "s_waitcnt vmcnt(4) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  MF " a[0:3], v[224:227], v[192:195], a[0:3]\n\t" \
  "ds_read_b128 v[240:243], %[rb1] offset:8192\n\t" \
  "s_add_u32 s87, s80, 2\n\t" \
  "s_cmp_eq_u32 s87, %[wrap]\n\t" \
  "s_cselect_b32 s85, %[back], 128\n\t" \
  MF " a[4:7], v[228:231], v[192:195], a[4:7]\n\t" \
  "ds_read_b128 v[244:247], %[rb1] offset:10240\n\t" \
  "s_add_u32 s81, s81, s85\n\t" \
  "s_add_u32 s82, s82, s85\n\t" \
  MF " a[8:11], v[232:235], v[192:195], a[8:11]\n\t" \
  "ds_read_b128 v[248:251], %[rb1] offset:12288\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "s_xor_b32 s86, s86, 0x10000\n\t" \
  MF " a[12:15], v[236:239], v[192:195], a[12:15]\n\t" \
  "ds_read_b128 v[252:255], %[rb1] offset:14336\n\t" \
  "v_or_b32 v120, s84, %[voa]\n\t" \
  MF " a[44:47], v[236:239], v[196:199], a[44:47]\n\t" \
  "v_or_b32 v121, s84, %[vob]\n\t" \
  MF " a[40:43], v[232:235], v[196:199], a[40:43]\n\t" \
  "s_mov_b32 s83, s81\n\t" \
  "s_add_u32 m0, s86, 0\n\t" \
  MF " a[36:39], v[228:231], v[196:199], a[36:39]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[32:35], v[224:227], v[196:199], a[32:35]\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  MF " a[64:67], v[224:227], v[200:203], a[64:67]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 4096\n\t" \
  MF " a[68:71], v[228:231], v[200:203], a[68:71]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[72:75], v[232:235], v[200:203], a[72:75]\n\t" \
  "ds_read_b128 v[160:163], %[rb0] offset:0\n\t" \
  MF " a[76:79], v[236:239], v[200:203], a[76:79]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 16384\n\t" \
  MF " a[108:111], v[236:239], v[204:207], a[108:111]\n\t" \
  "ds_read_b128 v[164:167], %[rb0] offset:2048\n\t" \
  MF " a[104:107], v[232:235], v[204:207], a[104:107]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[100:103], v[228:231], v[204:207], a[100:103]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 20480\n\t" \
  MF " a[96:99], v[224:227], v[204:207], a[96:99]\n\t" \
  "ds_read_b128 v[168:171], %[rb0] offset:4096\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[112:115], v[240:243], v[204:207], a[112:115]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[116:119], v[244:247], v[204:207], a[116:119]\n\t" \
  "ds_read_b128 v[172:175], %[rb0] offset:6144\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[120:123], v[248:251], v[204:207], a[120:123]\n\t" \
  "s_mov_b32 s83, s82\n\t" \
  "s_add_u32 m0, s86, 32768\n\t" \
  "s_waitcnt lgkmcnt(5)\n\t" \
  MF " a[124:127], v[252:255], v[204:207], a[124:127]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[92:95], v[252:255], v[200:203], a[92:95]\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  MF " a[88:91], v[248:251], v[200:203], a[88:91]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 36864\n\t" \
  MF " a[84:87], v[244:247], v[200:203], a[84:87]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[80:83], v[240:243], v[200:203], a[80:83]\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  MF " a[48:51], v[240:243], v[196:199], a[48:51]\n\t" \
  "s_add_u32 s83, s83, %[gbs3]\n\t" \
  "s_add_u32 m0, s86, 49152\n\t" \
  MF " a[52:55], v[244:247], v[196:199], a[52:55]\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  MF " a[56:59], v[248:251], v[196:199], a[56:59]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[60:63], v[252:255], v[196:199], a[60:63]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 53248\n\t" \
  MF " a[28:31], v[252:255], v[192:195], a[28:31]\n\t" \
  "v_xor_b32 %[ra1], 0x10000, %[ra1]\n\t" \
  MF " a[24:27], v[248:251], v[192:195], a[24:27]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[20:23], v[244:247], v[192:195], a[20:23]\n\t" \
  "v_xor_b32 %[rb1], 0x10000, %[rb1]\n\t" \
  MF " a[16:19], v[240:243], v[192:195], a[16:19]\n\t" \
  "s_add_u32 s80, s80, 1\n\t" \
  "s_waitcnt vmcnt(8) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "s_cmp_lt_u32 s80, %[n]\n\t" \
  "s_cbranch_scc1 L_sk_loop%=\n\t" \
  "s_waitcnt vmcnt(0) lgkmcnt(0)\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  ""
#define SK_TILE_ASM_LOOP_LOW_NN(MF) \
  "v_accvgpr_write_b32 a0, 0\n\t" \
  "v_accvgpr_write_b32 a1, 0\n\t" \
  "v_accvgpr_write_b32 a2, 0\n\t" \
  "v_accvgpr_write_b32 a3, 0\n\t" \
  "v_accvgpr_write_b32 a4, 0\n\t" \
  "v_accvgpr_write_b32 a5, 0\n\t" \
  "v_accvgpr_write_b32 a6, 0\n\t" \
  "v_accvgpr_write_b32 a7, 0\n\t" \
  "v_accvgpr_write_b32 a8, 0\n\t" \
  "v_accvgpr_write_b32 a9, 0\n\t" \
  "v_accvgpr_write_b32 a10, 0\n\t" \
  "v_accvgpr_write_b32 a11, 0\n\t" \
  "v_accvgpr_write_b32 a12, 0\n\t" \
  "v_accvgpr_write_b32 a13, 0\n\t" \
  "v_accvgpr_write_b32 a14, 0\n\t" \
  "v_accvgpr_write_b32 a15, 0\n\t" \
  "v_accvgpr_write_b32 a16, 0\n\t" \
  "v_accvgpr_write_b32 a17, 0\n\t" \
  "v_accvgpr_write_b32 a18, 0\n\t" \
  "v_accvgpr_write_b32 a19, 0\n\t" \
  "v_accvgpr_write_b32 a20, 0\n\t" \
  "v_accvgpr_write_b32 a21, 0\n\t" \
  "v_accvgpr_write_b32 a22, 0\n\t" \
  "v_accvgpr_write_b32 a23, 0\n\t" \
  "v_accvgpr_write_b32 a24, 0\n\t" \
  "v_accvgpr_write_b32 a25, 0\n\t" \
  "v_accvgpr_write_b32 a26, 0\n\t" \
  "v_accvgpr_write_b32 a27, 0\n\t" \
  "v_accvgpr_write_b32 a28, 0\n\t" \
  "v_accvgpr_write_b32 a29, 0\n\t" \
  "v_accvgpr_write_b32 a30, 0\n\t" \
  "v_accvgpr_write_b32 a31, 0\n\t" \
  "v_accvgpr_write_b32 a32, 0\n\t" \
  "v_accvgpr_write_b32 a33, 0\n\t" \
  "v_accvgpr_write_b32 a34, 0\n\t" \
  "v_accvgpr_write_b32 a35, 0\n\t" \
  "v_accvgpr_write_b32 a36, 0\n\t" \
  "v_accvgpr_write_b32 a37, 0\n\t" \
  "v_accvgpr_write_b32 a38, 0\n\t" \
  "v_accvgpr_write_b32 a39, 0\n\t" \
  "v_accvgpr_write_b32 a40, 0\n\t" \
  "v_accvgpr_write_b32 a41, 0\n\t" \
  "v_accvgpr_write_b32 a42, 0\n\t" \
  "v_accvgpr_write_b32 a43, 0\n\t" \
  "v_accvgpr_write_b32 a44, 0\n\t" \
  "v_accvgpr_write_b32 a45, 0\n\t" \
  "v_accvgpr_write_b32 a46, 0\n\t" \
  "v_accvgpr_write_b32 a47, 0\n\t" \
  "v_accvgpr_write_b32 a48, 0\n\t" \
  "v_accvgpr_write_b32 a49, 0\n\t" \
  "v_accvgpr_write_b32 a50, 0\n\t" \
  "v_accvgpr_write_b32 a51, 0\n\t" \
  "v_accvgpr_write_b32 a52, 0\n\t" \
  "v_accvgpr_write_b32 a53, 0\n\t" \
  "v_accvgpr_write_b32 a54, 0\n\t" \
  "v_accvgpr_write_b32 a55, 0\n\t" \
  "v_accvgpr_write_b32 a56, 0\n\t" \
  "v_accvgpr_write_b32 a57, 0\n\t" \
  "v_accvgpr_write_b32 a58, 0\n\t" \
  "v_accvgpr_write_b32 a59, 0\n\t" \
  "v_accvgpr_write_b32 a60, 0\n\t" \
  "v_accvgpr_write_b32 a61, 0\n\t" \
  "v_accvgpr_write_b32 a62, 0\n\t" \
  "v_accvgpr_write_b32 a63, 0\n\t" \
  "v_accvgpr_write_b32 a64, 0\n\t" \
  "v_accvgpr_write_b32 a65, 0\n\t" \
  "v_accvgpr_write_b32 a66, 0\n\t" \
  "v_accvgpr_write_b32 a67, 0\n\t" \
  "v_accvgpr_write_b32 a68, 0\n\t" \
  "v_accvgpr_write_b32 a69, 0\n\t" \
  "v_accvgpr_write_b32 a70, 0\n\t" \
  "v_accvgpr_write_b32 a71, 0\n\t" \
  "v_accvgpr_write_b32 a72, 0\n\t" \
  "v_accvgpr_write_b32 a73, 0\n\t" \
  "v_accvgpr_write_b32 a74, 0\n\t" \
  "v_accvgpr_write_b32 a75, 0\n\t" \
  "v_accvgpr_write_b32 a76, 0\n\t" \
  "v_accvgpr_write_b32 a77, 0\n\t" \
  "v_accvgpr_write_b32 a78, 0\n\t" \
  "v_accvgpr_write_b32 a79, 0\n\t" \
  "v_accvgpr_write_b32 a80, 0\n\t" \
  "v_accvgpr_write_b32 a81, 0\n\t" \
  "v_accvgpr_write_b32 a82, 0\n\t" \
  "v_accvgpr_write_b32 a83, 0\n\t" \
  "v_accvgpr_write_b32 a84, 0\n\t" \
  "v_accvgpr_write_b32 a85, 0\n\t" \
  "v_accvgpr_write_b32 a86, 0\n\t" \
  "v_accvgpr_write_b32 a87, 0\n\t" \
  "v_accvgpr_write_b32 a88, 0\n\t" \
  "v_accvgpr_write_b32 a89, 0\n\t" \
  "v_accvgpr_write_b32 a90, 0\n\t" \
  "v_accvgpr_write_b32 a91, 0\n\t" \
  "v_accvgpr_write_b32 a92, 0\n\t" \
  "v_accvgpr_write_b32 a93, 0\n\t" \
  "v_accvgpr_write_b32 a94, 0\n\t" \
  "v_accvgpr_write_b32 a95, 0\n\t" \
  "v_accvgpr_write_b32 a96, 0\n\t" \
  "v_accvgpr_write_b32 a97, 0\n\t" \
  "v_accvgpr_write_b32 a98, 0\n\t" \
  "v_accvgpr_write_b32 a99, 0\n\t" \
  "v_accvgpr_write_b32 a100, 0\n\t" \
  "v_accvgpr_write_b32 a101, 0\n\t" \
  "v_accvgpr_write_b32 a102, 0\n\t" \
  "v_accvgpr_write_b32 a103, 0\n\t" \
  "v_accvgpr_write_b32 a104, 0\n\t" \
  "v_accvgpr_write_b32 a105, 0\n\t" \
  "v_accvgpr_write_b32 a106, 0\n\t" \
  "v_accvgpr_write_b32 a107, 0\n\t" \
  "v_accvgpr_write_b32 a108, 0\n\t" \
  "v_accvgpr_write_b32 a109, 0\n\t" \
  "v_accvgpr_write_b32 a110, 0\n\t" \
  "v_accvgpr_write_b32 a111, 0\n\t" \
  "v_accvgpr_write_b32 a112, 0\n\t" \
  "v_accvgpr_write_b32 a113, 0\n\t" \
  "v_accvgpr_write_b32 a114, 0\n\t" \
  "v_accvgpr_write_b32 a115, 0\n\t" \
  "v_accvgpr_write_b32 a116, 0\n\t" \
  "v_accvgpr_write_b32 a117, 0\n\t" \
  "v_accvgpr_write_b32 a118, 0\n\t" \
  "v_accvgpr_write_b32 a119, 0\n\t" \
  "v_accvgpr_write_b32 a120, 0\n\t" \
  "v_accvgpr_write_b32 a121, 0\n\t" \
  "v_accvgpr_write_b32 a122, 0\n\t" \
  "v_accvgpr_write_b32 a123, 0\n\t" \
  "v_accvgpr_write_b32 a124, 0\n\t" \
  "v_accvgpr_write_b32 a125, 0\n\t" \
  "v_accvgpr_write_b32 a126, 0\n\t" \
  "v_accvgpr_write_b32 a127, 0\n\t" \
  "s_mov_b32 s80, 0\n\t" \
  "s_xor_b32 s86, %[lds], 0x10000\n\t" \
  "s_add_u32 s81, %[ga0], 128\n\t" \
  "s_add_u32 s82, %[gb0], %[kbs]\n\t" \
  "s_add_u32 s87, s80, 1\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "v_or_b32 v120, s84, %[voa]\n\t" \
  "v_or_b32 v121, s84, %[vob]\n\t" \
  "v_or_b32 v122, s84, %[vob1]\n\t" \
  "s_waitcnt vmcnt(8)\n\t" \
  "s_barrier\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[160:161], %[rbt0] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[162:163], %[rbt0] offset:2048\n\t" \
  "ds_read_b64_tr_b16 v[164:165], %[rbt1] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[166:167], %[rbt1] offset:2048\n\t" \
  "ds_read_b64_tr_b16 v[168:169], %[rbt2] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[170:171], %[rbt2] offset:2048\n\t" \
  "ds_read_b64_tr_b16 v[172:173], %[rbt3] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[174:175], %[rbt3] offset:2048\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  "s_nop 7\n\t" \
  "L_sk_loop%=:\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[0:3], v[160:163], v[128:131], a[0:3]\n\t" \
  "ds_read_b64_tr_b16 v[176:177], %[rbt4] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[178:179], %[rbt4] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[4:7], v[164:167], v[128:131], a[4:7]\n\t" \
  "ds_read_b64_tr_b16 v[180:181], %[rbt5] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[182:183], %[rbt5] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[8:11], v[168:171], v[128:131], a[8:11]\n\t" \
  "ds_read_b64_tr_b16 v[184:185], %[rbt6] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[186:187], %[rbt6] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[12:15], v[172:175], v[128:131], a[12:15]\n\t" \
  "ds_read_b64_tr_b16 v[188:189], %[rbt7] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[190:191], %[rbt7] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  MF " a[44:47], v[172:175], v[132:135], a[44:47]\n\t" \
  "s_add_u32 s83, s82, %[gbs4]\n\t" \
  "s_add_u32 m0, s86, 49152\n\t" \
  MF " a[40:43], v[168:171], v[132:135], a[40:43]\n\t" \
  "ds_read_b128 v[192:195], %[ra1] offset:0\n\t" \
  MF " a[36:39], v[164:167], v[132:135], a[36:39]\n\t" \
  "v_xor_b32 %[ra0], 0x10000, %[ra0]\n\t" \
  MF " a[32:35], v[160:163], v[132:135], a[32:35]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  MF " a[64:67], v[160:163], v[136:139], a[64:67]\n\t" \
  "ds_read_b64_tr_b16 v[224:225], %[rbt0] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[226:227], %[rbt0] offset:18432\n\t" \
  MF " a[68:71], v[164:167], v[136:139], a[68:71]\n\t" \
  MF " a[72:75], v[168:171], v[136:139], a[72:75]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 53248\n\t" \
  MF " a[76:79], v[172:175], v[136:139], a[76:79]\n\t" \
  "ds_read_b64_tr_b16 v[228:229], %[rbt1] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[230:231], %[rbt1] offset:18432\n\t" \
  "s_waitcnt lgkmcnt(13)\n\t" \
  MF " a[108:111], v[172:175], v[140:143], a[108:111]\n\t" \
  MF " a[104:107], v[168:171], v[140:143], a[104:107]\n\t" \
  MF " a[100:103], v[164:167], v[140:143], a[100:103]\n\t" \
  "buffer_load_dwordx4 v122, %[rsb], s83 offen lds\n\t" \
  MF " a[96:99], v[160:163], v[140:143], a[96:99]\n\t" \
  "ds_read_b64_tr_b16 v[232:233], %[rbt2] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[234:235], %[rbt2] offset:18432\n\t" \
  "s_waitcnt lgkmcnt(13)\n\t" \
  MF " a[112:115], v[176:179], v[140:143], a[112:115]\n\t" \
  "s_waitcnt lgkmcnt(11)\n\t" \
  MF " a[116:119], v[180:183], v[140:143], a[116:119]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 57344\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[120:123], v[184:187], v[140:143], a[120:123]\n\t" \
  "ds_read_b64_tr_b16 v[236:237], %[rbt3] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[238:239], %[rbt3] offset:18432\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[124:127], v[188:191], v[140:143], a[124:127]\n\t" \
  MF " a[92:95], v[188:191], v[136:139], a[92:95]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[88:91], v[184:187], v[136:139], a[88:91]\n\t" \
  "ds_read_b128 v[196:199], %[ra1] offset:2048\n\t" \
  MF " a[84:87], v[180:183], v[136:139], a[84:87]\n\t" \
  MF " a[80:83], v[176:179], v[136:139], a[80:83]\n\t" \
  MF " a[48:51], v[176:179], v[132:135], a[48:51]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 61440\n\t" \
  MF " a[52:55], v[180:183], v[132:135], a[52:55]\n\t" \
  "ds_read_b128 v[200:203], %[ra1] offset:4096\n\t" \
  MF " a[56:59], v[184:187], v[132:135], a[56:59]\n\t" \
  MF " a[60:63], v[188:191], v[132:135], a[60:63]\n\t" \
  "buffer_load_dwordx4 v122, %[rsb], s83 offen lds\n\t" \
  MF " a[28:31], v[188:191], v[128:131], a[28:31]\n\t" \
  "ds_read_b128 v[204:207], %[ra1] offset:6144\n\t" \
  MF " a[24:27], v[184:187], v[128:131], a[24:27]\n\t" \
  MF " a[20:23], v[180:183], v[128:131], a[20:23]\n\t" \
  MF " a[16:19], v[176:179], v[128:131], a[16:19]\n\t" \
  "s_waitcnt vmcnt(4) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  MF " a[0:3], v[224:227], v[192:195], a[0:3]\n\t" \
  "ds_read_b64_tr_b16 v[240:241], %[rbt4] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[242:243], %[rbt4] offset:18432\n\t" \
  "s_add_u32 s81, s81, 128\n\t" \
  "s_add_u32 s82, s82, %[kbs]\n\t" \
  MF " a[4:7], v[228:231], v[192:195], a[4:7]\n\t" \
  "ds_read_b64_tr_b16 v[244:245], %[rbt5] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[246:247], %[rbt5] offset:18432\n\t" \
  "s_xor_b32 s86, s86, 0x10000\n\t" \
  "s_add_u32 s87, s80, 2\n\t" \
  MF " a[8:11], v[232:235], v[192:195], a[8:11]\n\t" \
  "ds_read_b64_tr_b16 v[248:249], %[rbt6] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[250:251], %[rbt6] offset:18432\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  MF " a[12:15], v[236:239], v[192:195], a[12:15]\n\t" \
  "ds_read_b64_tr_b16 v[252:253], %[rbt7] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[254:255], %[rbt7] offset:18432\n\t" \
  "v_or_b32 v120, s84, %[voa]\n\t" \
  MF " a[44:47], v[236:239], v[196:199], a[44:47]\n\t" \
  "v_or_b32 v121, s84, %[vob]\n\t" \
  "v_or_b32 v122, s84, %[vob1]\n\t" \
  "v_xor_b32 %[rbt0], 0x10000, %[rbt0]\n\t" \
  "v_xor_b32 %[rbt1], 0x10000, %[rbt1]\n\t" \
  MF " a[40:43], v[232:235], v[196:199], a[40:43]\n\t" \
  "v_xor_b32 %[rbt2], 0x10000, %[rbt2]\n\t" \
  "v_xor_b32 %[rbt3], 0x10000, %[rbt3]\n\t" \
  "v_xor_b32 %[ra1], 0x10000, %[ra1]\n\t" \
  "v_xor_b32 %[rbt4], 0x10000, %[rbt4]\n\t" \
  MF " a[36:39], v[228:231], v[196:199], a[36:39]\n\t" \
  "v_xor_b32 %[rbt5], 0x10000, %[rbt5]\n\t" \
  "v_xor_b32 %[rbt6], 0x10000, %[rbt6]\n\t" \
  "v_xor_b32 %[rbt7], 0x10000, %[rbt7]\n\t" \
  MF " a[32:35], v[224:227], v[196:199], a[32:35]\n\t" \
  "s_mov_b32 s83, s81\n\t" \
  "s_add_u32 m0, s86, 0\n\t" \
  MF " a[64:67], v[224:227], v[200:203], a[64:67]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[68:71], v[228:231], v[200:203], a[68:71]\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  MF " a[72:75], v[232:235], v[200:203], a[72:75]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 4096\n\t" \
  MF " a[76:79], v[236:239], v[200:203], a[76:79]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[108:111], v[236:239], v[204:207], a[108:111]\n\t" \
  "ds_read_b64_tr_b16 v[160:161], %[rbt0] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[162:163], %[rbt0] offset:2048\n\t" \
  MF " a[104:107], v[232:235], v[204:207], a[104:107]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 16384\n\t" \
  MF " a[100:103], v[228:231], v[204:207], a[100:103]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[96:99], v[224:227], v[204:207], a[96:99]\n\t" \
  "ds_read_b64_tr_b16 v[164:165], %[rbt1] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[166:167], %[rbt1] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(11)\n\t" \
  MF " a[112:115], v[240:243], v[204:207], a[112:115]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 20480\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[116:119], v[244:247], v[204:207], a[116:119]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[120:123], v[248:251], v[204:207], a[120:123]\n\t" \
  "ds_read_b64_tr_b16 v[168:169], %[rbt2] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[170:171], %[rbt2] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[124:127], v[252:255], v[204:207], a[124:127]\n\t" \
  "s_mov_b32 s83, s82\n\t" \
  "s_add_u32 m0, s86, 32768\n\t" \
  MF " a[92:95], v[252:255], v[200:203], a[92:95]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[88:91], v[248:251], v[200:203], a[88:91]\n\t" \
  "ds_read_b64_tr_b16 v[172:173], %[rbt3] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[174:175], %[rbt3] offset:2048\n\t" \
  MF " a[84:87], v[244:247], v[200:203], a[84:87]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 36864\n\t" \
  MF " a[80:83], v[240:243], v[200:203], a[80:83]\n\t" \
  "buffer_load_dwordx4 v122, %[rsb], s83 offen lds\n\t" \
  MF " a[48:51], v[240:243], v[196:199], a[48:51]\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  MF " a[52:55], v[244:247], v[196:199], a[52:55]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 40960\n\t" \
  MF " a[56:59], v[248:251], v[196:199], a[56:59]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[60:63], v[252:255], v[196:199], a[60:63]\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  MF " a[28:31], v[252:255], v[192:195], a[28:31]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 45056\n\t" \
  MF " a[24:27], v[248:251], v[192:195], a[24:27]\n\t" \
  "buffer_load_dwordx4 v122, %[rsb], s83 offen lds\n\t" \
  MF " a[20:23], v[244:247], v[192:195], a[20:23]\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  MF " a[16:19], v[240:243], v[192:195], a[16:19]\n\t" \
  "s_add_u32 s80, s80, 1\n\t" \
  "s_waitcnt vmcnt(8) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "s_cmp_lt_u32 s80, %[n]\n\t" \
  "s_cbranch_scc1 L_sk_loop%=\n\t" \
  "s_waitcnt vmcnt(0) lgkmcnt(0)\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  ""
#define SK_TILE_ASM_LOOP_NN(MF) \
  "v_accvgpr_write_b32 a0, 0\n\t" \
  "v_accvgpr_write_b32 a1, 0\n\t" \
  "v_accvgpr_write_b32 a2, 0\n\t" \
  "v_accvgpr_write_b32 a3, 0\n\t" \
  "v_accvgpr_write_b32 a4, 0\n\t" \
  "v_accvgpr_write_b32 a5, 0\n\t" \
  "v_accvgpr_write_b32 a6, 0\n\t" \
  "v_accvgpr_write_b32 a7, 0\n\t" \
  "v_accvgpr_write_b32 a8, 0\n\t" \
  "v_accvgpr_write_b32 a9, 0\n\t" \
  "v_accvgpr_write_b32 a10, 0\n\t" \
  "v_accvgpr_write_b32 a11, 0\n\t" \
  "v_accvgpr_write_b32 a12, 0\n\t" \
  "v_accvgpr_write_b32 a13, 0\n\t" \
  "v_accvgpr_write_b32 a14, 0\n\t" \
  "v_accvgpr_write_b32 a15, 0\n\t" \
  "v_accvgpr_write_b32 a16, 0\n\t" \
  "v_accvgpr_write_b32 a17, 0\n\t" \
  "v_accvgpr_write_b32 a18, 0\n\t" \
  "v_accvgpr_write_b32 a19, 0\n\t" \
  "v_accvgpr_write_b32 a20, 0\n\t" \
  "v_accvgpr_write_b32 a21, 0\n\t" \
  "v_accvgpr_write_b32 a22, 0\n\t" \
  "v_accvgpr_write_b32 a23, 0\n\t" \
  "v_accvgpr_write_b32 a24, 0\n\t" \
  "v_accvgpr_write_b32 a25, 0\n\t" \
  "v_accvgpr_write_b32 a26, 0\n\t" \
  "v_accvgpr_write_b32 a27, 0\n\t" \
  "v_accvgpr_write_b32 a28, 0\n\t" \
  "v_accvgpr_write_b32 a29, 0\n\t" \
  "v_accvgpr_write_b32 a30, 0\n\t" \
  "v_accvgpr_write_b32 a31, 0\n\t" \
  "v_accvgpr_write_b32 a32, 0\n\t" \
  "v_accvgpr_write_b32 a33, 0\n\t" \
  "v_accvgpr_write_b32 a34, 0\n\t" \
  "v_accvgpr_write_b32 a35, 0\n\t" \
  "v_accvgpr_write_b32 a36, 0\n\t" \
  "v_accvgpr_write_b32 a37, 0\n\t" \
  "v_accvgpr_write_b32 a38, 0\n\t" \
  "v_accvgpr_write_b32 a39, 0\n\t" \
  "v_accvgpr_write_b32 a40, 0\n\t" \
  "v_accvgpr_write_b32 a41, 0\n\t" \
  "v_accvgpr_write_b32 a42, 0\n\t" \
  "v_accvgpr_write_b32 a43, 0\n\t" \
  "v_accvgpr_write_b32 a44, 0\n\t" \
  "v_accvgpr_write_b32 a45, 0\n\t" \
  "v_accvgpr_write_b32 a46, 0\n\t" \
  "v_accvgpr_write_b32 a47, 0\n\t" \
  "v_accvgpr_write_b32 a48, 0\n\t" \
  "v_accvgpr_write_b32 a49, 0\n\t" \
  "v_accvgpr_write_b32 a50, 0\n\t" \
  "v_accvgpr_write_b32 a51, 0\n\t" \
  "v_accvgpr_write_b32 a52, 0\n\t" \
  "v_accvgpr_write_b32 a53, 0\n\t" \
  "v_accvgpr_write_b32 a54, 0\n\t" \
  "v_accvgpr_write_b32 a55, 0\n\t" \
  "v_accvgpr_write_b32 a56, 0\n\t" \
  "v_accvgpr_write_b32 a57, 0\n\t" \
  "v_accvgpr_write_b32 a58, 0\n\t" \
  "v_accvgpr_write_b32 a59, 0\n\t" \
  "v_accvgpr_write_b32 a60, 0\n\t" \
  "v_accvgpr_write_b32 a61, 0\n\t" \
  "v_accvgpr_write_b32 a62, 0\n\t" \
  "v_accvgpr_write_b32 a63, 0\n\t" \
  "v_accvgpr_write_b32 a64, 0\n\t" \
  "v_accvgpr_write_b32 a65, 0\n\t" \
  "v_accvgpr_write_b32 a66, 0\n\t" \
  "v_accvgpr_write_b32 a67, 0\n\t" \
  "v_accvgpr_write_b32 a68, 0\n\t" \
  "v_accvgpr_write_b32 a69, 0\n\t" \
  "v_accvgpr_write_b32 a70, 0\n\t" \
  "v_accvgpr_write_b32 a71, 0\n\t" \
  "v_accvgpr_write_b32 a72, 0\n\t" \
  "v_accvgpr_write_b32 a73, 0\n\t" \
  "v_accvgpr_write_b32 a74, 0\n\t" \
  "v_accvgpr_write_b32 a75, 0\n\t" \
  "v_accvgpr_write_b32 a76, 0\n\t" \
  "v_accvgpr_write_b32 a77, 0\n\t" \
  "v_accvgpr_write_b32 a78, 0\n\t" \
  "v_accvgpr_write_b32 a79, 0\n\t" \
  "v_accvgpr_write_b32 a80, 0\n\t" \
  "v_accvgpr_write_b32 a81, 0\n\t" \
  "v_accvgpr_write_b32 a82, 0\n\t" \
  "v_accvgpr_write_b32 a83, 0\n\t" \
  "v_accvgpr_write_b32 a84, 0\n\t" \
  "v_accvgpr_write_b32 a85, 0\n\t" \
  "v_accvgpr_write_b32 a86, 0\n\t" \
  "v_accvgpr_write_b32 a87, 0\n\t" \
  "v_accvgpr_write_b32 a88, 0\n\t" \
  "v_accvgpr_write_b32 a89, 0\n\t" \
  "v_accvgpr_write_b32 a90, 0\n\t" \
  "v_accvgpr_write_b32 a91, 0\n\t" \
  "v_accvgpr_write_b32 a92, 0\n\t" \
  "v_accvgpr_write_b32 a93, 0\n\t" \
  "v_accvgpr_write_b32 a94, 0\n\t" \
  "v_accvgpr_write_b32 a95, 0\n\t" \
  "v_accvgpr_write_b32 a96, 0\n\t" \
  "v_accvgpr_write_b32 a97, 0\n\t" \
  "v_accvgpr_write_b32 a98, 0\n\t" \
  "v_accvgpr_write_b32 a99, 0\n\t" \
  "v_accvgpr_write_b32 a100, 0\n\t" \
  "v_accvgpr_write_b32 a101, 0\n\t" \
  "v_accvgpr_write_b32 a102, 0\n\t" \
  "v_accvgpr_write_b32 a103, 0\n\t" \
  "v_accvgpr_write_b32 a104, 0\n\t" \
  "v_accvgpr_write_b32 a105, 0\n\t" \
  "v_accvgpr_write_b32 a106, 0\n\t" \
  "v_accvgpr_write_b32 a107, 0\n\t" \
  "v_accvgpr_write_b32 a108, 0\n\t" \
  "v_accvgpr_write_b32 a109, 0\n\t" \
  "v_accvgpr_write_b32 a110, 0\n\t" \
  "v_accvgpr_write_b32 a111, 0\n\t" \
  "v_accvgpr_write_b32 a112, 0\n\t" \
  "v_accvgpr_write_b32 a113, 0\n\t" \
  "v_accvgpr_write_b32 a114, 0\n\t" \
  "v_accvgpr_write_b32 a115, 0\n\t" \
  "v_accvgpr_write_b32 a116, 0\n\t" \
  "v_accvgpr_write_b32 a117, 0\n\t" \
  "v_accvgpr_write_b32 a118, 0\n\t" \
  "v_accvgpr_write_b32 a119, 0\n\t" \
  "v_accvgpr_write_b32 a120, 0\n\t" \
  "v_accvgpr_write_b32 a121, 0\n\t" \
  "v_accvgpr_write_b32 a122, 0\n\t" \
  "v_accvgpr_write_b32 a123, 0\n\t" \
  "v_accvgpr_write_b32 a124, 0\n\t" \
  "v_accvgpr_write_b32 a125, 0\n\t" \
  "v_accvgpr_write_b32 a126, 0\n\t" \
  "v_accvgpr_write_b32 a127, 0\n\t" \
  "v_accvgpr_write_b32 a128, 0\n\t" \
  "v_accvgpr_write_b32 a129, 0\n\t" \
  "v_accvgpr_write_b32 a130, 0\n\t" \
  "v_accvgpr_write_b32 a131, 0\n\t" \
  "v_accvgpr_write_b32 a132, 0\n\t" \
  "v_accvgpr_write_b32 a133, 0\n\t" \
  "v_accvgpr_write_b32 a134, 0\n\t" \
  "v_accvgpr_write_b32 a135, 0\n\t" \
  "v_accvgpr_write_b32 a136, 0\n\t" \
  "v_accvgpr_write_b32 a137, 0\n\t" \
  "v_accvgpr_write_b32 a138, 0\n\t" \
  "v_accvgpr_write_b32 a139, 0\n\t" \
  "v_accvgpr_write_b32 a140, 0\n\t" \
  "v_accvgpr_write_b32 a141, 0\n\t" \
  "v_accvgpr_write_b32 a142, 0\n\t" \
  "v_accvgpr_write_b32 a143, 0\n\t" \
  "v_accvgpr_write_b32 a144, 0\n\t" \
  "v_accvgpr_write_b32 a145, 0\n\t" \
  "v_accvgpr_write_b32 a146, 0\n\t" \
  "v_accvgpr_write_b32 a147, 0\n\t" \
  "v_accvgpr_write_b32 a148, 0\n\t" \
  "v_accvgpr_write_b32 a149, 0\n\t" \
  "v_accvgpr_write_b32 a150, 0\n\t" \
  "v_accvgpr_write_b32 a151, 0\n\t" \
  "v_accvgpr_write_b32 a152, 0\n\t" \
  "v_accvgpr_write_b32 a153, 0\n\t" \
  "v_accvgpr_write_b32 a154, 0\n\t" \
  "v_accvgpr_write_b32 a155, 0\n\t" \
  "v_accvgpr_write_b32 a156, 0\n\t" \
  "v_accvgpr_write_b32 a157, 0\n\t" \
  "v_accvgpr_write_b32 a158, 0\n\t" \
  "v_accvgpr_write_b32 a159, 0\n\t" \
  "v_accvgpr_write_b32 a160, 0\n\t" \
  "v_accvgpr_write_b32 a161, 0\n\t" \
  "v_accvgpr_write_b32 a162, 0\n\t" \
  "v_accvgpr_write_b32 a163, 0\n\t" \
  "v_accvgpr_write_b32 a164, 0\n\t" \
  "v_accvgpr_write_b32 a165, 0\n\t" \
  "v_accvgpr_write_b32 a166, 0\n\t" \
  "v_accvgpr_write_b32 a167, 0\n\t" \
  "v_accvgpr_write_b32 a168, 0\n\t" \
  "v_accvgpr_write_b32 a169, 0\n\t" \
  "v_accvgpr_write_b32 a170, 0\n\t" \
  "v_accvgpr_write_b32 a171, 0\n\t" \
  "v_accvgpr_write_b32 a172, 0\n\t" \
  "v_accvgpr_write_b32 a173, 0\n\t" \
  "v_accvgpr_write_b32 a174, 0\n\t" \
  "v_accvgpr_write_b32 a175, 0\n\t" \
  "v_accvgpr_write_b32 a176, 0\n\t" \
  "v_accvgpr_write_b32 a177, 0\n\t" \
  "v_accvgpr_write_b32 a178, 0\n\t" \
  "v_accvgpr_write_b32 a179, 0\n\t" \
  "v_accvgpr_write_b32 a180, 0\n\t" \
  "v_accvgpr_write_b32 a181, 0\n\t" \
  "v_accvgpr_write_b32 a182, 0\n\t" \
  "v_accvgpr_write_b32 a183, 0\n\t" \
  "v_accvgpr_write_b32 a184, 0\n\t" \
  "v_accvgpr_write_b32 a185, 0\n\t" \
  "v_accvgpr_write_b32 a186, 0\n\t" \
  "v_accvgpr_write_b32 a187, 0\n\t" \
  "v_accvgpr_write_b32 a188, 0\n\t" \
  "v_accvgpr_write_b32 a189, 0\n\t" \
  "v_accvgpr_write_b32 a190, 0\n\t" \
  "v_accvgpr_write_b32 a191, 0\n\t" \
  "v_accvgpr_write_b32 a192, 0\n\t" \
  "v_accvgpr_write_b32 a193, 0\n\t" \
  "v_accvgpr_write_b32 a194, 0\n\t" \
  "v_accvgpr_write_b32 a195, 0\n\t" \
  "v_accvgpr_write_b32 a196, 0\n\t" \
  "v_accvgpr_write_b32 a197, 0\n\t" \
  "v_accvgpr_write_b32 a198, 0\n\t" \
  "v_accvgpr_write_b32 a199, 0\n\t" \
  "v_accvgpr_write_b32 a200, 0\n\t" \
  "v_accvgpr_write_b32 a201, 0\n\t" \
  "v_accvgpr_write_b32 a202, 0\n\t" \
  "v_accvgpr_write_b32 a203, 0\n\t" \
  "v_accvgpr_write_b32 a204, 0\n\t" \
  "v_accvgpr_write_b32 a205, 0\n\t" \
  "v_accvgpr_write_b32 a206, 0\n\t" \
  "v_accvgpr_write_b32 a207, 0\n\t" \
  "v_accvgpr_write_b32 a208, 0\n\t" \
  "v_accvgpr_write_b32 a209, 0\n\t" \
  "v_accvgpr_write_b32 a210, 0\n\t" \
  "v_accvgpr_write_b32 a211, 0\n\t" \
  "v_accvgpr_write_b32 a212, 0\n\t" \
  "v_accvgpr_write_b32 a213, 0\n\t" \
  "v_accvgpr_write_b32 a214, 0\n\t" \
  "v_accvgpr_write_b32 a215, 0\n\t" \
  "v_accvgpr_write_b32 a216, 0\n\t" \
  "v_accvgpr_write_b32 a217, 0\n\t" \
  "v_accvgpr_write_b32 a218, 0\n\t" \
  "v_accvgpr_write_b32 a219, 0\n\t" \
  "v_accvgpr_write_b32 a220, 0\n\t" \
  "v_accvgpr_write_b32 a221, 0\n\t" \
  "v_accvgpr_write_b32 a222, 0\n\t" \
  "v_accvgpr_write_b32 a223, 0\n\t" \
  "v_accvgpr_write_b32 a224, 0\n\t" \
  "v_accvgpr_write_b32 a225, 0\n\t" \
  "v_accvgpr_write_b32 a226, 0\n\t" \
  "v_accvgpr_write_b32 a227, 0\n\t" \
  "v_accvgpr_write_b32 a228, 0\n\t" \
  "v_accvgpr_write_b32 a229, 0\n\t" \
  "v_accvgpr_write_b32 a230, 0\n\t" \
  "v_accvgpr_write_b32 a231, 0\n\t" \
  "v_accvgpr_write_b32 a232, 0\n\t" \
  "v_accvgpr_write_b32 a233, 0\n\t" \
  "v_accvgpr_write_b32 a234, 0\n\t" \
  "v_accvgpr_write_b32 a235, 0\n\t" \
  "v_accvgpr_write_b32 a236, 0\n\t" \
  "v_accvgpr_write_b32 a237, 0\n\t" \
  "v_accvgpr_write_b32 a238, 0\n\t" \
  "v_accvgpr_write_b32 a239, 0\n\t" \
  "v_accvgpr_write_b32 a240, 0\n\t" \
  "v_accvgpr_write_b32 a241, 0\n\t" \
  "v_accvgpr_write_b32 a242, 0\n\t" \
  "v_accvgpr_write_b32 a243, 0\n\t" \
  "v_accvgpr_write_b32 a244, 0\n\t" \
  "v_accvgpr_write_b32 a245, 0\n\t" \
  "v_accvgpr_write_b32 a246, 0\n\t" \
  "v_accvgpr_write_b32 a247, 0\n\t" \
  "v_accvgpr_write_b32 a248, 0\n\t" \
  "v_accvgpr_write_b32 a249, 0\n\t" \
  "v_accvgpr_write_b32 a250, 0\n\t" \
  "v_accvgpr_write_b32 a251, 0\n\t" \
  "v_accvgpr_write_b32 a252, 0\n\t" \
  "v_accvgpr_write_b32 a253, 0\n\t" \
  "v_accvgpr_write_b32 a254, 0\n\t" \
  "v_accvgpr_write_b32 a255, 0\n\t" \
  "s_mov_b32 s80, 0\n\t" \
  "s_xor_b32 s86, %[lds], 0x10000\n\t" \
  "s_add_u32 s81, %[ga0], 128\n\t" \
  "s_add_u32 s82, %[gb0], %[kbs]\n\t" \
  "s_add_u32 s87, s80, 1\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "v_or_b32 v120, s84, %[voa]\n\t" \
  "v_or_b32 v121, s84, %[vob]\n\t" \
  "v_or_b32 v122, s84, %[vob1]\n\t" \
  "s_waitcnt vmcnt(12)\n\t" \
  "s_barrier\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[160:161], %[rbt0] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[162:163], %[rbt0] offset:2048\n\t" \
  "ds_read_b64_tr_b16 v[164:165], %[rbt1] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[166:167], %[rbt1] offset:2048\n\t" \
  "ds_read_b64_tr_b16 v[168:169], %[rbt2] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[170:171], %[rbt2] offset:2048\n\t" \
  "ds_read_b64_tr_b16 v[172:173], %[rbt3] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[174:175], %[rbt3] offset:2048\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  "s_nop 7\n\t" \
  "L_sk_loop%=:\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[0:3], v[160:163], v[128:131], a[0:3]\n\t" \
  "ds_read_b64_tr_b16 v[176:177], %[rbt4] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[178:179], %[rbt4] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[4:7], v[164:167], v[128:131], a[4:7]\n\t" \
  "ds_read_b64_tr_b16 v[180:181], %[rbt5] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[182:183], %[rbt5] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[8:11], v[168:171], v[128:131], a[8:11]\n\t" \
  "ds_read_b64_tr_b16 v[184:185], %[rbt6] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[186:187], %[rbt6] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[12:15], v[172:175], v[128:131], a[12:15]\n\t" \
  "ds_read_b64_tr_b16 v[188:189], %[rbt7] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[190:191], %[rbt7] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  MF " a[44:47], v[172:175], v[132:135], a[44:47]\n\t" \
  "ds_read_b128 v[144:147], %[ra0] offset:8192\n\t" \
  MF " a[40:43], v[168:171], v[132:135], a[40:43]\n\t" \
  "ds_read_b128 v[148:151], %[ra0] offset:10240\n\t" \
  MF " a[36:39], v[164:167], v[132:135], a[36:39]\n\t" \
  "ds_read_b128 v[152:155], %[ra0] offset:12288\n\t" \
  MF " a[32:35], v[160:163], v[132:135], a[32:35]\n\t" \
  "ds_read_b128 v[156:159], %[ra0] offset:14336\n\t" \
  "s_waitcnt lgkmcnt(13)\n\t" \
  MF " a[64:67], v[160:163], v[136:139], a[64:67]\n\t" \
  "s_add_u32 s83, s81, %[gas2]\n\t" \
  "s_add_u32 m0, s86, 8192\n\t" \
  MF " a[68:71], v[164:167], v[136:139], a[68:71]\n\t" \
  "ds_read_b128 v[192:195], %[ra1] offset:0\n\t" \
  MF " a[72:75], v[168:171], v[136:139], a[72:75]\n\t" \
  "v_xor_b32 %[ra0], 0x10000, %[ra0]\n\t" \
  MF " a[76:79], v[172:175], v[136:139], a[76:79]\n\t" \
  "s_waitcnt lgkmcnt(13)\n\t" \
  MF " a[108:111], v[172:175], v[140:143], a[108:111]\n\t" \
  MF " a[104:107], v[168:171], v[140:143], a[104:107]\n\t" \
  "ds_read_b64_tr_b16 v[224:225], %[rbt0] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[226:227], %[rbt0] offset:18432\n\t" \
  MF " a[100:103], v[164:167], v[140:143], a[100:103]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[96:99], v[160:163], v[140:143], a[96:99]\n\t" \
  "s_waitcnt lgkmcnt(13)\n\t" \
  MF " a[112:115], v[176:179], v[140:143], a[112:115]\n\t" \
  "s_waitcnt lgkmcnt(11)\n\t" \
  MF " a[116:119], v[180:183], v[140:143], a[116:119]\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[120:123], v[184:187], v[140:143], a[120:123]\n\t" \
  "s_waitcnt lgkmcnt(7)\n\t" \
  MF " a[124:127], v[188:191], v[140:143], a[124:127]\n\t" \
  "ds_read_b64_tr_b16 v[228:229], %[rbt1] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[230:231], %[rbt1] offset:18432\n\t" \
  MF " a[92:95], v[188:191], v[136:139], a[92:95]\n\t" \
  MF " a[88:91], v[184:187], v[136:139], a[88:91]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 12288\n\t" \
  MF " a[84:87], v[180:183], v[136:139], a[84:87]\n\t" \
  MF " a[80:83], v[176:179], v[136:139], a[80:83]\n\t" \
  MF " a[48:51], v[176:179], v[132:135], a[48:51]\n\t" \
  MF " a[52:55], v[180:183], v[132:135], a[52:55]\n\t" \
  "ds_read_b64_tr_b16 v[232:233], %[rbt2] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[234:235], %[rbt2] offset:18432\n\t" \
  MF " a[56:59], v[184:187], v[132:135], a[56:59]\n\t" \
  MF " a[60:63], v[188:191], v[132:135], a[60:63]\n\t" \
  MF " a[28:31], v[188:191], v[128:131], a[28:31]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[24:27], v[184:187], v[128:131], a[24:27]\n\t" \
  MF " a[20:23], v[180:183], v[128:131], a[20:23]\n\t" \
  MF " a[16:19], v[176:179], v[128:131], a[16:19]\n\t" \
  "ds_read_b64_tr_b16 v[236:237], %[rbt3] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[238:239], %[rbt3] offset:18432\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  MF " a[144:147], v[176:179], v[144:147], a[144:147]\n\t" \
  MF " a[148:151], v[180:183], v[144:147], a[148:151]\n\t" \
  MF " a[152:155], v[184:187], v[144:147], a[152:155]\n\t" \
  MF " a[156:159], v[188:191], v[144:147], a[156:159]\n\t" \
  "s_add_u32 s83, s83, %[gas3]\n\t" \
  "s_add_u32 m0, s86, 24576\n\t" \
  "s_waitcnt lgkmcnt(11)\n\t" \
  MF " a[188:191], v[188:191], v[148:151], a[188:191]\n\t" \
  MF " a[184:187], v[184:187], v[148:151], a[184:187]\n\t" \
  "ds_read_b128 v[196:199], %[ra1] offset:2048\n\t" \
  MF " a[180:183], v[180:183], v[148:151], a[180:183]\n\t" \
  MF " a[176:179], v[176:179], v[148:151], a[176:179]\n\t" \
  "s_waitcnt lgkmcnt(11)\n\t" \
  MF " a[208:211], v[176:179], v[152:155], a[208:211]\n\t" \
  MF " a[212:215], v[180:183], v[152:155], a[212:215]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[216:219], v[184:187], v[152:155], a[216:219]\n\t" \
  MF " a[220:223], v[188:191], v[152:155], a[220:223]\n\t" \
  "ds_read_b128 v[200:203], %[ra1] offset:4096\n\t" \
  "s_waitcnt lgkmcnt(11)\n\t" \
  MF " a[252:255], v[188:191], v[156:159], a[252:255]\n\t" \
  MF " a[248:251], v[184:187], v[156:159], a[248:251]\n\t" \
  MF " a[244:247], v[180:183], v[156:159], a[244:247]\n\t" \
  MF " a[240:243], v[176:179], v[156:159], a[240:243]\n\t" \
  MF " a[236:239], v[172:175], v[156:159], a[236:239]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 28672\n\t" \
  MF " a[232:235], v[168:171], v[156:159], a[232:235]\n\t" \
  "ds_read_b128 v[204:207], %[ra1] offset:6144\n\t" \
  MF " a[228:231], v[164:167], v[156:159], a[228:231]\n\t" \
  MF " a[224:227], v[160:163], v[156:159], a[224:227]\n\t" \
  MF " a[192:195], v[160:163], v[152:155], a[192:195]\n\t" \
  MF " a[196:199], v[164:167], v[152:155], a[196:199]\n\t" \
  MF " a[200:203], v[168:171], v[152:155], a[200:203]\n\t" \
  MF " a[204:207], v[172:175], v[152:155], a[204:207]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[172:175], v[172:175], v[148:151], a[172:175]\n\t" \
  MF " a[168:171], v[168:171], v[148:151], a[168:171]\n\t" \
  MF " a[164:167], v[164:167], v[148:151], a[164:167]\n\t" \
  MF " a[160:163], v[160:163], v[148:151], a[160:163]\n\t" \
  MF " a[128:131], v[160:163], v[144:147], a[128:131]\n\t" \
  MF " a[132:135], v[164:167], v[144:147], a[132:135]\n\t" \
  MF " a[136:139], v[168:171], v[144:147], a[136:139]\n\t" \
  MF " a[140:143], v[172:175], v[144:147], a[140:143]\n\t" \
  "s_waitcnt vmcnt(4) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  MF " a[0:3], v[224:227], v[192:195], a[0:3]\n\t" \
  "ds_read_b64_tr_b16 v[240:241], %[rbt4] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[242:243], %[rbt4] offset:18432\n\t" \
  MF " a[4:7], v[228:231], v[192:195], a[4:7]\n\t" \
  "ds_read_b64_tr_b16 v[244:245], %[rbt5] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[246:247], %[rbt5] offset:18432\n\t" \
  MF " a[8:11], v[232:235], v[192:195], a[8:11]\n\t" \
  "ds_read_b64_tr_b16 v[248:249], %[rbt6] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[250:251], %[rbt6] offset:18432\n\t" \
  MF " a[12:15], v[236:239], v[192:195], a[12:15]\n\t" \
  "ds_read_b64_tr_b16 v[252:253], %[rbt7] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[254:255], %[rbt7] offset:18432\n\t" \
  MF " a[44:47], v[236:239], v[196:199], a[44:47]\n\t" \
  "ds_read_b128 v[208:211], %[ra1] offset:8192\n\t" \
  MF " a[40:43], v[232:235], v[196:199], a[40:43]\n\t" \
  "ds_read_b128 v[212:215], %[ra1] offset:10240\n\t" \
  MF " a[36:39], v[228:231], v[196:199], a[36:39]\n\t" \
  "ds_read_b128 v[216:219], %[ra1] offset:12288\n\t" \
  MF " a[32:35], v[224:227], v[196:199], a[32:35]\n\t" \
  "ds_read_b128 v[220:223], %[ra1] offset:14336\n\t" \
  MF " a[64:67], v[224:227], v[200:203], a[64:67]\n\t" \
  "s_add_u32 s81, s81, 128\n\t" \
  "s_add_u32 s82, s82, %[kbs]\n\t" \
  MF " a[68:71], v[228:231], v[200:203], a[68:71]\n\t" \
  "s_xor_b32 s86, s86, 0x10000\n\t" \
  "s_add_u32 s87, s80, 2\n\t" \
  MF " a[72:75], v[232:235], v[200:203], a[72:75]\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  MF " a[76:79], v[236:239], v[200:203], a[76:79]\n\t" \
  "v_or_b32 v120, s84, %[voa]\n\t" \
  MF " a[108:111], v[236:239], v[204:207], a[108:111]\n\t" \
  "v_or_b32 v121, s84, %[vob]\n\t" \
  MF " a[104:107], v[232:235], v[204:207], a[104:107]\n\t" \
  "v_or_b32 v122, s84, %[vob1]\n\t" \
  MF " a[100:103], v[228:231], v[204:207], a[100:103]\n\t" \
  "v_xor_b32 %[rbt0], 0x10000, %[rbt0]\n\t" \
  MF " a[96:99], v[224:227], v[204:207], a[96:99]\n\t" \
  "v_xor_b32 %[rbt1], 0x10000, %[rbt1]\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  MF " a[112:115], v[240:243], v[204:207], a[112:115]\n\t" \
  "v_xor_b32 %[rbt2], 0x10000, %[rbt2]\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  MF " a[116:119], v[244:247], v[204:207], a[116:119]\n\t" \
  "v_xor_b32 %[rbt3], 0x10000, %[rbt3]\n\t" \
  "s_waitcnt lgkmcnt(6)\n\t" \
  MF " a[120:123], v[248:251], v[204:207], a[120:123]\n\t" \
  "s_mov_b32 s83, s81\n\t" \
  "s_add_u32 m0, s86, 0\n\t" \
  "s_waitcnt lgkmcnt(4)\n\t" \
  MF " a[124:127], v[252:255], v[204:207], a[124:127]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[92:95], v[252:255], v[200:203], a[92:95]\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  MF " a[88:91], v[248:251], v[200:203], a[88:91]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 4096\n\t" \
  MF " a[84:87], v[244:247], v[200:203], a[84:87]\n\t" \
  "v_xor_b32 %[ra1], 0x10000, %[ra1]\n\t" \
  MF " a[80:83], v[240:243], v[200:203], a[80:83]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[48:51], v[240:243], v[196:199], a[48:51]\n\t" \
  "ds_read_b64_tr_b16 v[160:161], %[rbt0] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[162:163], %[rbt0] offset:2048\n\t" \
  MF " a[52:55], v[244:247], v[196:199], a[52:55]\n\t" \
  "s_add_u32 s83, s83, %[gas3]\n\t" \
  "s_add_u32 m0, s86, 16384\n\t" \
  MF " a[56:59], v[248:251], v[196:199], a[56:59]\n\t" \
  MF " a[60:63], v[252:255], v[196:199], a[60:63]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[28:31], v[252:255], v[192:195], a[28:31]\n\t" \
  "ds_read_b64_tr_b16 v[164:165], %[rbt1] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[166:167], %[rbt1] offset:2048\n\t" \
  MF " a[24:27], v[248:251], v[192:195], a[24:27]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 20480\n\t" \
  MF " a[20:23], v[244:247], v[192:195], a[20:23]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[16:19], v[240:243], v[192:195], a[16:19]\n\t" \
  "v_xor_b32 %[rbt4], 0x10000, %[rbt4]\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  MF " a[144:147], v[240:243], v[208:211], a[144:147]\n\t" \
  "s_mov_b32 s83, s82\n\t" \
  "s_add_u32 m0, s86, 32768\n\t" \
  MF " a[148:151], v[244:247], v[208:211], a[148:151]\n\t" \
  "ds_read_b64_tr_b16 v[168:169], %[rbt2] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[170:171], %[rbt2] offset:2048\n\t" \
  MF " a[152:155], v[248:251], v[208:211], a[152:155]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[156:159], v[252:255], v[208:211], a[156:159]\n\t" \
  "s_waitcnt lgkmcnt(9)\n\t" \
  MF " a[188:191], v[252:255], v[212:215], a[188:191]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 36864\n\t" \
  MF " a[184:187], v[248:251], v[212:215], a[184:187]\n\t" \
  "ds_read_b64_tr_b16 v[172:173], %[rbt3] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[174:175], %[rbt3] offset:2048\n\t" \
  MF " a[180:183], v[244:247], v[212:215], a[180:183]\n\t" \
  "buffer_load_dwordx4 v122, %[rsb], s83 offen lds\n\t" \
  MF " a[176:179], v[240:243], v[212:215], a[176:179]\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  MF " a[208:211], v[240:243], v[216:219], a[208:211]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 40960\n\t" \
  MF " a[212:215], v[244:247], v[216:219], a[212:215]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[216:219], v[248:251], v[216:219], a[216:219]\n\t" \
  "ds_read_b128 v[132:135], %[ra0] offset:2048\n\t" \
  MF " a[220:223], v[252:255], v[216:219], a[220:223]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 45056\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  MF " a[252:255], v[252:255], v[220:223], a[252:255]\n\t" \
  "v_xor_b32 %[rbt5], 0x10000, %[rbt5]\n\t" \
  MF " a[248:251], v[248:251], v[220:223], a[248:251]\n\t" \
  "buffer_load_dwordx4 v122, %[rsb], s83 offen lds\n\t" \
  MF " a[244:247], v[244:247], v[220:223], a[244:247]\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:4096\n\t" \
  MF " a[240:243], v[240:243], v[220:223], a[240:243]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 49152\n\t" \
  MF " a[236:239], v[236:239], v[220:223], a[236:239]\n\t" \
  MF " a[232:235], v[232:235], v[220:223], a[232:235]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[228:231], v[228:231], v[220:223], a[228:231]\n\t" \
  "ds_read_b128 v[140:143], %[ra0] offset:6144\n\t" \
  MF " a[224:227], v[224:227], v[220:223], a[224:227]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 53248\n\t" \
  MF " a[192:195], v[224:227], v[216:219], a[192:195]\n\t" \
  "buffer_load_dwordx4 v122, %[rsb], s83 offen lds\n\t" \
  MF " a[196:199], v[228:231], v[216:219], a[196:199]\n\t" \
  "v_xor_b32 %[rbt6], 0x10000, %[rbt6]\n\t" \
  MF " a[200:203], v[232:235], v[216:219], a[200:203]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 57344\n\t" \
  MF " a[204:207], v[236:239], v[216:219], a[204:207]\n\t" \
  MF " a[172:175], v[236:239], v[212:215], a[172:175]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[168:171], v[232:235], v[212:215], a[168:171]\n\t" \
  MF " a[164:167], v[228:231], v[212:215], a[164:167]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 61440\n\t" \
  MF " a[160:163], v[224:227], v[212:215], a[160:163]\n\t" \
  "v_xor_b32 %[rbt7], 0x10000, %[rbt7]\n\t" \
  MF " a[128:131], v[224:227], v[208:211], a[128:131]\n\t" \
  "buffer_load_dwordx4 v122, %[rsb], s83 offen lds\n\t" \
  MF " a[132:135], v[228:231], v[208:211], a[132:135]\n\t" \
  MF " a[136:139], v[232:235], v[208:211], a[136:139]\n\t" \
  MF " a[140:143], v[236:239], v[208:211], a[140:143]\n\t" \
  "s_add_u32 s80, s80, 1\n\t" \
  "s_waitcnt vmcnt(12) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "s_cmp_lt_u32 s80, %[n]\n\t" \
  "s_cbranch_scc1 L_sk_loop%=\n\t" \
  "s_waitcnt vmcnt(0) lgkmcnt(0)\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  ""
#define SK_TILE_ASM_LOOP_TN(MF) \
  "v_accvgpr_write_b32 a0, 0\n\t" \
  "v_accvgpr_write_b32 a1, 0\n\t" \
  "v_accvgpr_write_b32 a2, 0\n\t" \
  "v_accvgpr_write_b32 a3, 0\n\t" \
  "v_accvgpr_write_b32 a4, 0\n\t" \
  "v_accvgpr_write_b32 a5, 0\n\t" \
  "v_accvgpr_write_b32 a6, 0\n\t" \
  "v_accvgpr_write_b32 a7, 0\n\t" \
  "v_accvgpr_write_b32 a8, 0\n\t" \
  "v_accvgpr_write_b32 a9, 0\n\t" \
  "v_accvgpr_write_b32 a10, 0\n\t" \
  "v_accvgpr_write_b32 a11, 0\n\t" \
  "v_accvgpr_write_b32 a12, 0\n\t" \
  "v_accvgpr_write_b32 a13, 0\n\t" \
  "v_accvgpr_write_b32 a14, 0\n\t" \
  "v_accvgpr_write_b32 a15, 0\n\t" \
  "v_accvgpr_write_b32 a16, 0\n\t" \
  "v_accvgpr_write_b32 a17, 0\n\t" \
  "v_accvgpr_write_b32 a18, 0\n\t" \
  "v_accvgpr_write_b32 a19, 0\n\t" \
  "v_accvgpr_write_b32 a20, 0\n\t" \
  "v_accvgpr_write_b32 a21, 0\n\t" \
  "v_accvgpr_write_b32 a22, 0\n\t" \
  "v_accvgpr_write_b32 a23, 0\n\t" \
  "v_accvgpr_write_b32 a24, 0\n\t" \
  "v_accvgpr_write_b32 a25, 0\n\t" \
  "v_accvgpr_write_b32 a26, 0\n\t" \
  "v_accvgpr_write_b32 a27, 0\n\t" \
  "v_accvgpr_write_b32 a28, 0\n\t" \
  "v_accvgpr_write_b32 a29, 0\n\t" \
  "v_accvgpr_write_b32 a30, 0\n\t" \
  "v_accvgpr_write_b32 a31, 0\n\t" \
  "v_accvgpr_write_b32 a32, 0\n\t" \
  "v_accvgpr_write_b32 a33, 0\n\t" \
  "v_accvgpr_write_b32 a34, 0\n\t" \
  "v_accvgpr_write_b32 a35, 0\n\t" \
  "v_accvgpr_write_b32 a36, 0\n\t" \
  "v_accvgpr_write_b32 a37, 0\n\t" \
  "v_accvgpr_write_b32 a38, 0\n\t" \
  "v_accvgpr_write_b32 a39, 0\n\t" \
  "v_accvgpr_write_b32 a40, 0\n\t" \
  "v_accvgpr_write_b32 a41, 0\n\t" \
  "v_accvgpr_write_b32 a42, 0\n\t" \
  "v_accvgpr_write_b32 a43, 0\n\t" \
  "v_accvgpr_write_b32 a44, 0\n\t" \
  "v_accvgpr_write_b32 a45, 0\n\t" \
  "v_accvgpr_write_b32 a46, 0\n\t" \
  "v_accvgpr_write_b32 a47, 0\n\t" \
  "v_accvgpr_write_b32 a48, 0\n\t" \
  "v_accvgpr_write_b32 a49, 0\n\t" \
  "v_accvgpr_write_b32 a50, 0\n\t" \
  "v_accvgpr_write_b32 a51, 0\n\t" \
  "v_accvgpr_write_b32 a52, 0\n\t" \
  "v_accvgpr_write_b32 a53, 0\n\t" \
  "v_accvgpr_write_b32 a54, 0\n\t" \
  "v_accvgpr_write_b32 a55, 0\n\t" \
  "v_accvgpr_write_b32 a56, 0\n\t" \
  "v_accvgpr_write_b32 a57, 0\n\t" \
  "v_accvgpr_write_b32 a58, 0\n\t" \
  "v_accvgpr_write_b32 a59, 0\n\t" \
  "v_accvgpr_write_b32 a60, 0\n\t" \
  "v_accvgpr_write_b32 a61, 0\n\t" \
  "v_accvgpr_write_b32 a62, 0\n\t" \
  "v_accvgpr_write_b32 a63, 0\n\t" \
  "v_accvgpr_write_b32 a64, 0\n\t" \
  "v_accvgpr_write_b32 a65, 0\n\t" \
  "v_accvgpr_write_b32 a66, 0\n\t" \
  "v_accvgpr_write_b32 a67, 0\n\t" \
  "v_accvgpr_write_b32 a68, 0\n\t" \
  "v_accvgpr_write_b32 a69, 0\n\t" \
  "v_accvgpr_write_b32 a70, 0\n\t" \
  "v_accvgpr_write_b32 a71, 0\n\t" \
  "v_accvgpr_write_b32 a72, 0\n\t" \
  "v_accvgpr_write_b32 a73, 0\n\t" \
  "v_accvgpr_write_b32 a74, 0\n\t" \
  "v_accvgpr_write_b32 a75, 0\n\t" \
  "v_accvgpr_write_b32 a76, 0\n\t" \
  "v_accvgpr_write_b32 a77, 0\n\t" \
  "v_accvgpr_write_b32 a78, 0\n\t" \
  "v_accvgpr_write_b32 a79, 0\n\t" \
  "v_accvgpr_write_b32 a80, 0\n\t" \
  "v_accvgpr_write_b32 a81, 0\n\t" \
  "v_accvgpr_write_b32 a82, 0\n\t" \
  "v_accvgpr_write_b32 a83, 0\n\t" \
  "v_accvgpr_write_b32 a84, 0\n\t" \
  "v_accvgpr_write_b32 a85, 0\n\t" \
  "v_accvgpr_write_b32 a86, 0\n\t" \
  "v_accvgpr_write_b32 a87, 0\n\t" \
  "v_accvgpr_write_b32 a88, 0\n\t" \
  "v_accvgpr_write_b32 a89, 0\n\t" \
  "v_accvgpr_write_b32 a90, 0\n\t" \
  "v_accvgpr_write_b32 a91, 0\n\t" \
  "v_accvgpr_write_b32 a92, 0\n\t" \
  "v_accvgpr_write_b32 a93, 0\n\t" \
  "v_accvgpr_write_b32 a94, 0\n\t" \
  "v_accvgpr_write_b32 a95, 0\n\t" \
  "v_accvgpr_write_b32 a96, 0\n\t" \
  "v_accvgpr_write_b32 a97, 0\n\t" \
  "v_accvgpr_write_b32 a98, 0\n\t" \
  "v_accvgpr_write_b32 a99, 0\n\t" \
  "v_accvgpr_write_b32 a100, 0\n\t" \
  "v_accvgpr_write_b32 a101, 0\n\t" \
  "v_accvgpr_write_b32 a102, 0\n\t" \
  "v_accvgpr_write_b32 a103, 0\n\t" \
  "v_accvgpr_write_b32 a104, 0\n\t" \
  "v_accvgpr_write_b32 a105, 0\n\t" \
  "v_accvgpr_write_b32 a106, 0\n\t" \
  "v_accvgpr_write_b32 a107, 0\n\t" \
  "v_accvgpr_write_b32 a108, 0\n\t" \
  "v_accvgpr_write_b32 a109, 0\n\t" \
  "v_accvgpr_write_b32 a110, 0\n\t" \
  "v_accvgpr_write_b32 a111, 0\n\t" \
  "v_accvgpr_write_b32 a112, 0\n\t" \
  "v_accvgpr_write_b32 a113, 0\n\t" \
  "v_accvgpr_write_b32 a114, 0\n\t" \
  "v_accvgpr_write_b32 a115, 0\n\t" \
  "v_accvgpr_write_b32 a116, 0\n\t" \
  "v_accvgpr_write_b32 a117, 0\n\t" \
  "v_accvgpr_write_b32 a118, 0\n\t" \
  "v_accvgpr_write_b32 a119, 0\n\t" \
  "v_accvgpr_write_b32 a120, 0\n\t" \
  "v_accvgpr_write_b32 a121, 0\n\t" \
  "v_accvgpr_write_b32 a122, 0\n\t" \
  "v_accvgpr_write_b32 a123, 0\n\t" \
  "v_accvgpr_write_b32 a124, 0\n\t" \
  "v_accvgpr_write_b32 a125, 0\n\t" \
  "v_accvgpr_write_b32 a126, 0\n\t" \
  "v_accvgpr_write_b32 a127, 0\n\t" \
  "v_accvgpr_write_b32 a128, 0\n\t" \
  "v_accvgpr_write_b32 a129, 0\n\t" \
  "v_accvgpr_write_b32 a130, 0\n\t" \
  "v_accvgpr_write_b32 a131, 0\n\t" \
  "v_accvgpr_write_b32 a132, 0\n\t" \
  "v_accvgpr_write_b32 a133, 0\n\t" \
  "v_accvgpr_write_b32 a134, 0\n\t" \
  "v_accvgpr_write_b32 a135, 0\n\t" \
  "v_accvgpr_write_b32 a136, 0\n\t" \
  "v_accvgpr_write_b32 a137, 0\n\t" \
  "v_accvgpr_write_b32 a138, 0\n\t" \
  "v_accvgpr_write_b32 a139, 0\n\t" \
  "v_accvgpr_write_b32 a140, 0\n\t" \
  "v_accvgpr_write_b32 a141, 0\n\t" \
  "v_accvgpr_write_b32 a142, 0\n\t" \
  "v_accvgpr_write_b32 a143, 0\n\t" \
  "v_accvgpr_write_b32 a144, 0\n\t" \
  "v_accvgpr_write_b32 a145, 0\n\t" \
  "v_accvgpr_write_b32 a146, 0\n\t" \
  "v_accvgpr_write_b32 a147, 0\n\t" \
  "v_accvgpr_write_b32 a148, 0\n\t" \
  "v_accvgpr_write_b32 a149, 0\n\t" \
  "v_accvgpr_write_b32 a150, 0\n\t" \
  "v_accvgpr_write_b32 a151, 0\n\t" \
  "v_accvgpr_write_b32 a152, 0\n\t" \
  "v_accvgpr_write_b32 a153, 0\n\t" \
  "v_accvgpr_write_b32 a154, 0\n\t" \
  "v_accvgpr_write_b32 a155, 0\n\t" \
  "v_accvgpr_write_b32 a156, 0\n\t" \
  "v_accvgpr_write_b32 a157, 0\n\t" \
  "v_accvgpr_write_b32 a158, 0\n\t" \
  "v_accvgpr_write_b32 a159, 0\n\t" \
  "v_accvgpr_write_b32 a160, 0\n\t" \
  "v_accvgpr_write_b32 a161, 0\n\t" \
  "v_accvgpr_write_b32 a162, 0\n\t" \
  "v_accvgpr_write_b32 a163, 0\n\t" \
  "v_accvgpr_write_b32 a164, 0\n\t" \
  "v_accvgpr_write_b32 a165, 0\n\t" \
  "v_accvgpr_write_b32 a166, 0\n\t" \
  "v_accvgpr_write_b32 a167, 0\n\t" \
  "v_accvgpr_write_b32 a168, 0\n\t" \
  "v_accvgpr_write_b32 a169, 0\n\t" \
  "v_accvgpr_write_b32 a170, 0\n\t" \
  "v_accvgpr_write_b32 a171, 0\n\t" \
  "v_accvgpr_write_b32 a172, 0\n\t" \
  "v_accvgpr_write_b32 a173, 0\n\t" \
  "v_accvgpr_write_b32 a174, 0\n\t" \
  "v_accvgpr_write_b32 a175, 0\n\t" \
  "v_accvgpr_write_b32 a176, 0\n\t" \
  "v_accvgpr_write_b32 a177, 0\n\t" \
  "v_accvgpr_write_b32 a178, 0\n\t" \
  "v_accvgpr_write_b32 a179, 0\n\t" \
  "v_accvgpr_write_b32 a180, 0\n\t" \
  "v_accvgpr_write_b32 a181, 0\n\t" \
  "v_accvgpr_write_b32 a182, 0\n\t" \
  "v_accvgpr_write_b32 a183, 0\n\t" \
  "v_accvgpr_write_b32 a184, 0\n\t" \
  "v_accvgpr_write_b32 a185, 0\n\t" \
  "v_accvgpr_write_b32 a186, 0\n\t" \
  "v_accvgpr_write_b32 a187, 0\n\t" \
  "v_accvgpr_write_b32 a188, 0\n\t" \
  "v_accvgpr_write_b32 a189, 0\n\t" \
  "v_accvgpr_write_b32 a190, 0\n\t" \
  "v_accvgpr_write_b32 a191, 0\n\t" \
  "v_accvgpr_write_b32 a192, 0\n\t" \
  "v_accvgpr_write_b32 a193, 0\n\t" \
  "v_accvgpr_write_b32 a194, 0\n\t" \
  "v_accvgpr_write_b32 a195, 0\n\t" \
  "v_accvgpr_write_b32 a196, 0\n\t" \
  "v_accvgpr_write_b32 a197, 0\n\t" \
  "v_accvgpr_write_b32 a198, 0\n\t" \
  "v_accvgpr_write_b32 a199, 0\n\t" \
  "v_accvgpr_write_b32 a200, 0\n\t" \
  "v_accvgpr_write_b32 a201, 0\n\t" \
  "v_accvgpr_write_b32 a202, 0\n\t" \
  "v_accvgpr_write_b32 a203, 0\n\t" \
  "v_accvgpr_write_b32 a204, 0\n\t" \
  "v_accvgpr_write_b32 a205, 0\n\t" \
  "v_accvgpr_write_b32 a206, 0\n\t" \
  "v_accvgpr_write_b32 a207, 0\n\t" \
  "v_accvgpr_write_b32 a208, 0\n\t" \
  "v_accvgpr_write_b32 a209, 0\n\t" \
  "v_accvgpr_write_b32 a210, 0\n\t" \
  "v_accvgpr_write_b32 a211, 0\n\t" \
  "v_accvgpr_write_b32 a212, 0\n\t" \
  "v_accvgpr_write_b32 a213, 0\n\t" \
  "v_accvgpr_write_b32 a214, 0\n\t" \
  "v_accvgpr_write_b32 a215, 0\n\t" \
  "v_accvgpr_write_b32 a216, 0\n\t" \
  "v_accvgpr_write_b32 a217, 0\n\t" \
  "v_accvgpr_write_b32 a218, 0\n\t" \
  "v_accvgpr_write_b32 a219, 0\n\t" \
  "v_accvgpr_write_b32 a220, 0\n\t" \
  "v_accvgpr_write_b32 a221, 0\n\t" \
  "v_accvgpr_write_b32 a222, 0\n\t" \
  "v_accvgpr_write_b32 a223, 0\n\t" \
  "v_accvgpr_write_b32 a224, 0\n\t" \
  "v_accvgpr_write_b32 a225, 0\n\t" \
  "v_accvgpr_write_b32 a226, 0\n\t" \
  "v_accvgpr_write_b32 a227, 0\n\t" \
  "v_accvgpr_write_b32 a228, 0\n\t" \
  "v_accvgpr_write_b32 a229, 0\n\t" \
  "v_accvgpr_write_b32 a230, 0\n\t" \
  "v_accvgpr_write_b32 a231, 0\n\t" \
  "v_accvgpr_write_b32 a232, 0\n\t" \
  "v_accvgpr_write_b32 a233, 0\n\t" \
  "v_accvgpr_write_b32 a234, 0\n\t" \
  "v_accvgpr_write_b32 a235, 0\n\t" \
  "v_accvgpr_write_b32 a236, 0\n\t" \
  "v_accvgpr_write_b32 a237, 0\n\t" \
  "v_accvgpr_write_b32 a238, 0\n\t" \
  "v_accvgpr_write_b32 a239, 0\n\t" \
  "v_accvgpr_write_b32 a240, 0\n\t" \
  "v_accvgpr_write_b32 a241, 0\n\t" \
  "v_accvgpr_write_b32 a242, 0\n\t" \
  "v_accvgpr_write_b32 a243, 0\n\t" \
  "v_accvgpr_write_b32 a244, 0\n\t" \
  "v_accvgpr_write_b32 a245, 0\n\t" \
  "v_accvgpr_write_b32 a246, 0\n\t" \
  "v_accvgpr_write_b32 a247, 0\n\t" \
  "v_accvgpr_write_b32 a248, 0\n\t" \
  "v_accvgpr_write_b32 a249, 0\n\t" \
  "v_accvgpr_write_b32 a250, 0\n\t" \
  "v_accvgpr_write_b32 a251, 0\n\t" \
  "v_accvgpr_write_b32 a252, 0\n\t" \
  "v_accvgpr_write_b32 a253, 0\n\t" \
  "v_accvgpr_write_b32 a254, 0\n\t" \
  "v_accvgpr_write_b32 a255, 0\n\t" \
  "s_mov_b32 s80, 0\n\t" \
  "s_xor_b32 s86, %[lds], 0x10000\n\t" \
  "s_add_u32 s81, %[ga0], %[kas]\n\t" \
  "s_add_u32 s82, %[gb0], %[kbs]\n\t" \
  "s_add_u32 s87, s80, 1\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "v_or_b32 v120, s84, %[voa]\n\t" \
  "v_or_b32 v121, s84, %[vob]\n\t" \
  "v_or_b32 v122, s84, %[vob1]\n\t" \
  "v_or_b32 v123, s84, %[voa1]\n\t" \
  "s_waitcnt vmcnt(8)\n\t" \
  "s_barrier\n\t" \
  "ds_read_b64_tr_b16 v[128:129], %[rat0] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[130:131], %[rat0] offset:2048\n\t" \
  "ds_read_b64_tr_b16 v[160:161], %[rbt0] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[162:163], %[rbt0] offset:2048\n\t" \
  "ds_read_b64_tr_b16 v[164:165], %[rbt1] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[166:167], %[rbt1] offset:2048\n\t" \
  "ds_read_b64_tr_b16 v[168:169], %[rbt2] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[170:171], %[rbt2] offset:2048\n\t" \
  "ds_read_b64_tr_b16 v[172:173], %[rbt3] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[174:175], %[rbt3] offset:2048\n\t" \
  "ds_read_b64_tr_b16 v[132:133], %[rat1] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[134:135], %[rat1] offset:2048\n\t" \
  "ds_read_b64_tr_b16 v[136:137], %[rat2] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[138:139], %[rat2] offset:2048\n\t" \
  "ds_read_b64_tr_b16 v[140:141], %[rat3] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[142:143], %[rat3] offset:2048\n\t" \
  "s_nop 7\n\t" \
  "L_sk_loop%=:\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  MF " a[0:3], v[160:163], v[128:131], a[0:3]\n\t" \
  "ds_read_b64_tr_b16 v[176:177], %[rbt4] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[178:179], %[rbt4] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  MF " a[4:7], v[164:167], v[128:131], a[4:7]\n\t" \
  "ds_read_b64_tr_b16 v[180:181], %[rbt5] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[182:183], %[rbt5] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  MF " a[8:11], v[168:171], v[128:131], a[8:11]\n\t" \
  "ds_read_b64_tr_b16 v[184:185], %[rbt6] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[186:187], %[rbt6] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  MF " a[12:15], v[172:175], v[128:131], a[12:15]\n\t" \
  "ds_read_b64_tr_b16 v[188:189], %[rbt7] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[190:191], %[rbt7] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  MF " a[44:47], v[172:175], v[132:135], a[44:47]\n\t" \
  "ds_read_b64_tr_b16 v[144:145], %[rat4] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[146:147], %[rat4] offset:2048\n\t" \
  MF " a[40:43], v[168:171], v[132:135], a[40:43]\n\t" \
  "ds_read_b64_tr_b16 v[148:149], %[rat5] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[150:151], %[rat5] offset:2048\n\t" \
  MF " a[36:39], v[164:167], v[132:135], a[36:39]\n\t" \
  "ds_read_b64_tr_b16 v[152:153], %[rat6] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[154:155], %[rat6] offset:2048\n\t" \
  MF " a[32:35], v[160:163], v[132:135], a[32:35]\n\t" \
  "ds_read_b64_tr_b16 v[156:157], %[rat7] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[158:159], %[rat7] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(15)\n\t" \
  MF " a[64:67], v[160:163], v[136:139], a[64:67]\n\t" \
  "s_add_u32 s83, s81, %[gas4]\n\t" \
  "s_add_u32 m0, s86, 16384\n\t" \
  MF " a[68:71], v[164:167], v[136:139], a[68:71]\n\t" \
  "ds_read_b64_tr_b16 v[192:193], %[rat0] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[194:195], %[rat0] offset:18432\n\t" \
  MF " a[72:75], v[168:171], v[136:139], a[72:75]\n\t" \
  MF " a[76:79], v[172:175], v[136:139], a[76:79]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[108:111], v[172:175], v[140:143], a[108:111]\n\t" \
  MF " a[104:107], v[168:171], v[140:143], a[104:107]\n\t" \
  MF " a[100:103], v[164:167], v[140:143], a[100:103]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 20480\n\t" \
  MF " a[96:99], v[160:163], v[140:143], a[96:99]\n\t" \
  "ds_read_b64_tr_b16 v[224:225], %[rbt0] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[226:227], %[rbt0] offset:18432\n\t" \
  "s_waitcnt lgkmcnt(15)\n\t" \
  MF " a[112:115], v[176:179], v[140:143], a[112:115]\n\t" \
  MF " a[116:119], v[180:183], v[140:143], a[116:119]\n\t" \
  "s_waitcnt lgkmcnt(14)\n\t" \
  MF " a[120:123], v[184:187], v[140:143], a[120:123]\n\t" \
  "buffer_load_dwordx4 v123, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  MF " a[124:127], v[188:191], v[140:143], a[124:127]\n\t" \
  MF " a[92:95], v[188:191], v[136:139], a[92:95]\n\t" \
  "ds_read_b64_tr_b16 v[228:229], %[rbt1] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[230:231], %[rbt1] offset:18432\n\t" \
  MF " a[88:91], v[184:187], v[136:139], a[88:91]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 24576\n\t" \
  MF " a[84:87], v[180:183], v[136:139], a[84:87]\n\t" \
  MF " a[80:83], v[176:179], v[136:139], a[80:83]\n\t" \
  MF " a[48:51], v[176:179], v[132:135], a[48:51]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[52:55], v[180:183], v[132:135], a[52:55]\n\t" \
  MF " a[56:59], v[184:187], v[132:135], a[56:59]\n\t" \
  "ds_read_b64_tr_b16 v[232:233], %[rbt2] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[234:235], %[rbt2] offset:18432\n\t" \
  MF " a[60:63], v[188:191], v[132:135], a[60:63]\n\t" \
  MF " a[28:31], v[188:191], v[128:131], a[28:31]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 28672\n\t" \
  MF " a[24:27], v[184:187], v[128:131], a[24:27]\n\t" \
  MF " a[20:23], v[180:183], v[128:131], a[20:23]\n\t" \
  MF " a[16:19], v[176:179], v[128:131], a[16:19]\n\t" \
  "buffer_load_dwordx4 v123, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(14)\n\t" \
  MF " a[144:147], v[176:179], v[144:147], a[144:147]\n\t" \
  "ds_read_b64_tr_b16 v[236:237], %[rbt3] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[238:239], %[rbt3] offset:18432\n\t" \
  MF " a[148:151], v[180:183], v[144:147], a[148:151]\n\t" \
  MF " a[152:155], v[184:187], v[144:147], a[152:155]\n\t" \
  MF " a[156:159], v[188:191], v[144:147], a[156:159]\n\t" \
  "s_add_u32 s83, s82, %[gbs4]\n\t" \
  "s_add_u32 m0, s86, 49152\n\t" \
  "s_waitcnt lgkmcnt(14)\n\t" \
  MF " a[188:191], v[188:191], v[148:151], a[188:191]\n\t" \
  MF " a[184:187], v[184:187], v[148:151], a[184:187]\n\t" \
  "ds_read_b64_tr_b16 v[196:197], %[rat1] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[198:199], %[rat1] offset:18432\n\t" \
  MF " a[180:183], v[180:183], v[148:151], a[180:183]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[176:179], v[176:179], v[148:151], a[176:179]\n\t" \
  "s_waitcnt lgkmcnt(14)\n\t" \
  MF " a[208:211], v[176:179], v[152:155], a[208:211]\n\t" \
  MF " a[212:215], v[180:183], v[152:155], a[212:215]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 53248\n\t" \
  MF " a[216:219], v[184:187], v[152:155], a[216:219]\n\t" \
  MF " a[220:223], v[188:191], v[152:155], a[220:223]\n\t" \
  "ds_read_b64_tr_b16 v[200:201], %[rat2] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[202:203], %[rat2] offset:18432\n\t" \
  "s_waitcnt lgkmcnt(14)\n\t" \
  MF " a[252:255], v[188:191], v[156:159], a[252:255]\n\t" \
  MF " a[248:251], v[184:187], v[156:159], a[248:251]\n\t" \
  "buffer_load_dwordx4 v122, %[rsb], s83 offen lds\n\t" \
  MF " a[244:247], v[180:183], v[156:159], a[244:247]\n\t" \
  MF " a[240:243], v[176:179], v[156:159], a[240:243]\n\t" \
  MF " a[236:239], v[172:175], v[156:159], a[236:239]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 57344\n\t" \
  MF " a[232:235], v[168:171], v[156:159], a[232:235]\n\t" \
  "ds_read_b64_tr_b16 v[204:205], %[rat3] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[206:207], %[rat3] offset:18432\n\t" \
  MF " a[228:231], v[164:167], v[156:159], a[228:231]\n\t" \
  MF " a[224:227], v[160:163], v[156:159], a[224:227]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[192:195], v[160:163], v[152:155], a[192:195]\n\t" \
  MF " a[196:199], v[164:167], v[152:155], a[196:199]\n\t" \
  MF " a[200:203], v[168:171], v[152:155], a[200:203]\n\t" \
  MF " a[204:207], v[172:175], v[152:155], a[204:207]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 61440\n\t" \
  MF " a[172:175], v[172:175], v[148:151], a[172:175]\n\t" \
  MF " a[168:171], v[168:171], v[148:151], a[168:171]\n\t" \
  MF " a[164:167], v[164:167], v[148:151], a[164:167]\n\t" \
  "buffer_load_dwordx4 v122, %[rsb], s83 offen lds\n\t" \
  MF " a[160:163], v[160:163], v[148:151], a[160:163]\n\t" \
  MF " a[128:131], v[160:163], v[144:147], a[128:131]\n\t" \
  MF " a[132:135], v[164:167], v[144:147], a[132:135]\n\t" \
  MF " a[136:139], v[168:171], v[144:147], a[136:139]\n\t" \
  MF " a[140:143], v[172:175], v[144:147], a[140:143]\n\t" \
  "s_waitcnt vmcnt(8) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  MF " a[0:3], v[224:227], v[192:195], a[0:3]\n\t" \
  "ds_read_b64_tr_b16 v[240:241], %[rbt4] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[242:243], %[rbt4] offset:18432\n\t" \
  MF " a[4:7], v[228:231], v[192:195], a[4:7]\n\t" \
  "ds_read_b64_tr_b16 v[244:245], %[rbt5] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[246:247], %[rbt5] offset:18432\n\t" \
  MF " a[8:11], v[232:235], v[192:195], a[8:11]\n\t" \
  "ds_read_b64_tr_b16 v[248:249], %[rbt6] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[250:251], %[rbt6] offset:18432\n\t" \
  MF " a[12:15], v[236:239], v[192:195], a[12:15]\n\t" \
  "ds_read_b64_tr_b16 v[252:253], %[rbt7] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[254:255], %[rbt7] offset:18432\n\t" \
  MF " a[44:47], v[236:239], v[196:199], a[44:47]\n\t" \
  "ds_read_b64_tr_b16 v[208:209], %[rat4] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[210:211], %[rat4] offset:18432\n\t" \
  MF " a[40:43], v[232:235], v[196:199], a[40:43]\n\t" \
  "ds_read_b64_tr_b16 v[212:213], %[rat5] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[214:215], %[rat5] offset:18432\n\t" \
  MF " a[36:39], v[228:231], v[196:199], a[36:39]\n\t" \
  "ds_read_b64_tr_b16 v[216:217], %[rat6] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[218:219], %[rat6] offset:18432\n\t" \
  MF " a[32:35], v[224:227], v[196:199], a[32:35]\n\t" \
  "ds_read_b64_tr_b16 v[220:221], %[rat7] offset:16384\n\t" \
  "ds_read_b64_tr_b16 v[222:223], %[rat7] offset:18432\n\t" \
  MF " a[64:67], v[224:227], v[200:203], a[64:67]\n\t" \
  "s_add_u32 s81, s81, %[kas]\n\t" \
  "s_add_u32 s82, s82, %[kbs]\n\t" \
  MF " a[68:71], v[228:231], v[200:203], a[68:71]\n\t" \
  "s_xor_b32 s86, s86, 0x10000\n\t" \
  "s_add_u32 s87, s80, 2\n\t" \
  MF " a[72:75], v[232:235], v[200:203], a[72:75]\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  MF " a[76:79], v[236:239], v[200:203], a[76:79]\n\t" \
  "v_or_b32 v120, s84, %[voa]\n\t" \
  MF " a[108:111], v[236:239], v[204:207], a[108:111]\n\t" \
  "v_or_b32 v121, s84, %[vob]\n\t" \
  MF " a[104:107], v[232:235], v[204:207], a[104:107]\n\t" \
  "v_or_b32 v122, s84, %[vob1]\n\t" \
  MF " a[100:103], v[228:231], v[204:207], a[100:103]\n\t" \
  "v_or_b32 v123, s84, %[voa1]\n\t" \
  MF " a[96:99], v[224:227], v[204:207], a[96:99]\n\t" \
  "v_xor_b32 %[rbt0], 0x10000, %[rbt0]\n\t" \
  "s_waitcnt lgkmcnt(14)\n\t" \
  MF " a[112:115], v[240:243], v[204:207], a[112:115]\n\t" \
  "v_xor_b32 %[rbt1], 0x10000, %[rbt1]\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  MF " a[116:119], v[244:247], v[204:207], a[116:119]\n\t" \
  "v_xor_b32 %[rbt2], 0x10000, %[rbt2]\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  MF " a[120:123], v[248:251], v[204:207], a[120:123]\n\t" \
  "v_xor_b32 %[rbt3], 0x10000, %[rbt3]\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  MF " a[124:127], v[252:255], v[204:207], a[124:127]\n\t" \
  "v_xor_b32 %[rat0], 0x10000, %[rat0]\n\t" \
  MF " a[92:95], v[252:255], v[200:203], a[92:95]\n\t" \
  "v_xor_b32 %[rat1], 0x10000, %[rat1]\n\t" \
  MF " a[88:91], v[248:251], v[200:203], a[88:91]\n\t" \
  "v_xor_b32 %[rat2], 0x10000, %[rat2]\n\t" \
  MF " a[84:87], v[244:247], v[200:203], a[84:87]\n\t" \
  "v_xor_b32 %[rat3], 0x10000, %[rat3]\n\t" \
  MF " a[80:83], v[240:243], v[200:203], a[80:83]\n\t" \
  "s_mov_b32 s83, s81\n\t" \
  "s_add_u32 m0, s86, 0\n\t" \
  MF " a[48:51], v[240:243], v[196:199], a[48:51]\n\t" \
  "ds_read_b64_tr_b16 v[128:129], %[rat0] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[130:131], %[rat0] offset:2048\n\t" \
  MF " a[52:55], v[244:247], v[196:199], a[52:55]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[56:59], v[248:251], v[196:199], a[56:59]\n\t" \
  "v_xor_b32 %[rat4], 0x10000, %[rat4]\n\t" \
  MF " a[60:63], v[252:255], v[196:199], a[60:63]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 4096\n\t" \
  MF " a[28:31], v[252:255], v[192:195], a[28:31]\n\t" \
  "ds_read_b64_tr_b16 v[160:161], %[rbt0] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[162:163], %[rbt0] offset:2048\n\t" \
  MF " a[24:27], v[248:251], v[192:195], a[24:27]\n\t" \
  MF " a[20:23], v[244:247], v[192:195], a[20:23]\n\t" \
  "buffer_load_dwordx4 v123, %[rsa], s83 offen lds\n\t" \
  MF " a[16:19], v[240:243], v[192:195], a[16:19]\n\t" \
  "ds_read_b64_tr_b16 v[164:165], %[rbt1] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[166:167], %[rbt1] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  MF " a[144:147], v[240:243], v[208:211], a[144:147]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 8192\n\t" \
  MF " a[148:151], v[244:247], v[208:211], a[148:151]\n\t" \
  "v_xor_b32 %[rat5], 0x10000, %[rat5]\n\t" \
  MF " a[152:155], v[248:251], v[208:211], a[152:155]\n\t" \
  "ds_read_b64_tr_b16 v[168:169], %[rbt2] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[170:171], %[rbt2] offset:2048\n\t" \
  MF " a[156:159], v[252:255], v[208:211], a[156:159]\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  MF " a[188:191], v[252:255], v[212:215], a[188:191]\n\t" \
  MF " a[184:187], v[248:251], v[212:215], a[184:187]\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 12288\n\t" \
  MF " a[180:183], v[244:247], v[212:215], a[180:183]\n\t" \
  "v_xor_b32 %[rat6], 0x10000, %[rat6]\n\t" \
  MF " a[176:179], v[240:243], v[212:215], a[176:179]\n\t" \
  "ds_read_b64_tr_b16 v[172:173], %[rbt3] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[174:175], %[rbt3] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  MF " a[208:211], v[240:243], v[216:219], a[208:211]\n\t" \
  "buffer_load_dwordx4 v123, %[rsa], s83 offen lds\n\t" \
  MF " a[212:215], v[244:247], v[216:219], a[212:215]\n\t" \
  MF " a[216:219], v[248:251], v[216:219], a[216:219]\n\t" \
  "s_mov_b32 s83, s82\n\t" \
  "s_add_u32 m0, s86, 32768\n\t" \
  MF " a[220:223], v[252:255], v[216:219], a[220:223]\n\t" \
  "ds_read_b64_tr_b16 v[132:133], %[rat1] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[134:135], %[rat1] offset:2048\n\t" \
  "s_waitcnt lgkmcnt(12)\n\t" \
  MF " a[252:255], v[252:255], v[220:223], a[252:255]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[248:251], v[248:251], v[220:223], a[248:251]\n\t" \
  "v_xor_b32 %[rat7], 0x10000, %[rat7]\n\t" \
  MF " a[244:247], v[244:247], v[220:223], a[244:247]\n\t" \
  "ds_read_b64_tr_b16 v[136:137], %[rat2] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[138:139], %[rat2] offset:2048\n\t" \
  MF " a[240:243], v[240:243], v[220:223], a[240:243]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 36864\n\t" \
  MF " a[236:239], v[236:239], v[220:223], a[236:239]\n\t" \
  MF " a[232:235], v[232:235], v[220:223], a[232:235]\n\t" \
  "buffer_load_dwordx4 v122, %[rsb], s83 offen lds\n\t" \
  MF " a[228:231], v[228:231], v[220:223], a[228:231]\n\t" \
  "ds_read_b64_tr_b16 v[140:141], %[rat3] offset:0\n\t" \
  "ds_read_b64_tr_b16 v[142:143], %[rat3] offset:2048\n\t" \
  MF " a[224:227], v[224:227], v[220:223], a[224:227]\n\t" \
  "v_xor_b32 %[rbt4], 0x10000, %[rbt4]\n\t" \
  MF " a[192:195], v[224:227], v[216:219], a[192:195]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 40960\n\t" \
  MF " a[196:199], v[228:231], v[216:219], a[196:199]\n\t" \
  MF " a[200:203], v[232:235], v[216:219], a[200:203]\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[204:207], v[236:239], v[216:219], a[204:207]\n\t" \
  "v_xor_b32 %[rbt5], 0x10000, %[rbt5]\n\t" \
  MF " a[172:175], v[236:239], v[212:215], a[172:175]\n\t" \
  MF " a[168:171], v[232:235], v[212:215], a[168:171]\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 45056\n\t" \
  MF " a[164:167], v[228:231], v[212:215], a[164:167]\n\t" \
  "v_xor_b32 %[rbt6], 0x10000, %[rbt6]\n\t" \
  MF " a[160:163], v[224:227], v[212:215], a[160:163]\n\t" \
  "buffer_load_dwordx4 v122, %[rsb], s83 offen lds\n\t" \
  MF " a[128:131], v[224:227], v[208:211], a[128:131]\n\t" \
  MF " a[132:135], v[228:231], v[208:211], a[132:135]\n\t" \
  "v_xor_b32 %[rbt7], 0x10000, %[rbt7]\n\t" \
  MF " a[136:139], v[232:235], v[208:211], a[136:139]\n\t" \
  MF " a[140:143], v[236:239], v[208:211], a[140:143]\n\t" \
  "s_add_u32 s80, s80, 1\n\t" \
  "s_waitcnt vmcnt(8) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "s_cmp_lt_u32 s80, %[n]\n\t" \
  "s_cbranch_scc1 L_sk_loop%=\n\t" \
  "s_waitcnt vmcnt(0) lgkmcnt(0)\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  ""
#define SK_TILE_ASM_LOOP_F8(MF, MOD) \
  "v_accvgpr_write_b32 a0, 0\n\t" \
  "v_accvgpr_write_b32 a1, 0\n\t" \
  "v_accvgpr_write_b32 a2, 0\n\t" \
  "v_accvgpr_write_b32 a3, 0\n\t" \
  "v_accvgpr_write_b32 a4, 0\n\t" \
  "v_accvgpr_write_b32 a5, 0\n\t" \
  "v_accvgpr_write_b32 a6, 0\n\t" \
  "v_accvgpr_write_b32 a7, 0\n\t" \
  "v_accvgpr_write_b32 a8, 0\n\t" \
  "v_accvgpr_write_b32 a9, 0\n\t" \
  "v_accvgpr_write_b32 a10, 0\n\t" \
  "v_accvgpr_write_b32 a11, 0\n\t" \
  "v_accvgpr_write_b32 a12, 0\n\t" \
  "v_accvgpr_write_b32 a13, 0\n\t" \
  "v_accvgpr_write_b32 a14, 0\n\t" \
  "v_accvgpr_write_b32 a15, 0\n\t" \
  "v_accvgpr_write_b32 a16, 0\n\t" \
  "v_accvgpr_write_b32 a17, 0\n\t" \
  "v_accvgpr_write_b32 a18, 0\n\t" \
  "v_accvgpr_write_b32 a19, 0\n\t" \
  "v_accvgpr_write_b32 a20, 0\n\t" \
  "v_accvgpr_write_b32 a21, 0\n\t" \
  "v_accvgpr_write_b32 a22, 0\n\t" \
  "v_accvgpr_write_b32 a23, 0\n\t" \
  "v_accvgpr_write_b32 a24, 0\n\t" \
  "v_accvgpr_write_b32 a25, 0\n\t" \
  "v_accvgpr_write_b32 a26, 0\n\t" \
  "v_accvgpr_write_b32 a27, 0\n\t" \
  "v_accvgpr_write_b32 a28, 0\n\t" \
  "v_accvgpr_write_b32 a29, 0\n\t" \
  "v_accvgpr_write_b32 a30, 0\n\t" \
  "v_accvgpr_write_b32 a31, 0\n\t" \
  "v_accvgpr_write_b32 a32, 0\n\t" \
  "v_accvgpr_write_b32 a33, 0\n\t" \
  "v_accvgpr_write_b32 a34, 0\n\t" \
  "v_accvgpr_write_b32 a35, 0\n\t" \
  "v_accvgpr_write_b32 a36, 0\n\t" \
  "v_accvgpr_write_b32 a37, 0\n\t" \
  "v_accvgpr_write_b32 a38, 0\n\t" \
  "v_accvgpr_write_b32 a39, 0\n\t" \
  "v_accvgpr_write_b32 a40, 0\n\t" \
  "v_accvgpr_write_b32 a41, 0\n\t" \
  "v_accvgpr_write_b32 a42, 0\n\t" \
  "v_accvgpr_write_b32 a43, 0\n\t" \
  "v_accvgpr_write_b32 a44, 0\n\t" \
  "v_accvgpr_write_b32 a45, 0\n\t" \
  "v_accvgpr_write_b32 a46, 0\n\t" \
  "v_accvgpr_write_b32 a47, 0\n\t" \
  "v_accvgpr_write_b32 a48, 0\n\t" \
  "v_accvgpr_write_b32 a49, 0\n\t" \
  "v_accvgpr_write_b32 a50, 0\n\t" \
  "v_accvgpr_write_b32 a51, 0\n\t" \
  "v_accvgpr_write_b32 a52, 0\n\t" \
  "v_accvgpr_write_b32 a53, 0\n\t" \
  "v_accvgpr_write_b32 a54, 0\n\t" \
  "v_accvgpr_write_b32 a55, 0\n\t" \
  "v_accvgpr_write_b32 a56, 0\n\t" \
  "v_accvgpr_write_b32 a57, 0\n\t" \
  "v_accvgpr_write_b32 a58, 0\n\t" \
  "v_accvgpr_write_b32 a59, 0\n\t" \
  "v_accvgpr_write_b32 a60, 0\n\t" \
  "v_accvgpr_write_b32 a61, 0\n\t" \
  "v_accvgpr_write_b32 a62, 0\n\t" \
  "v_accvgpr_write_b32 a63, 0\n\t" \
  "v_accvgpr_write_b32 a64, 0\n\t" \
  "v_accvgpr_write_b32 a65, 0\n\t" \
  "v_accvgpr_write_b32 a66, 0\n\t" \
  "v_accvgpr_write_b32 a67, 0\n\t" \
  "v_accvgpr_write_b32 a68, 0\n\t" \
  "v_accvgpr_write_b32 a69, 0\n\t" \
  "v_accvgpr_write_b32 a70, 0\n\t" \
  "v_accvgpr_write_b32 a71, 0\n\t" \
  "v_accvgpr_write_b32 a72, 0\n\t" \
  "v_accvgpr_write_b32 a73, 0\n\t" \
  "v_accvgpr_write_b32 a74, 0\n\t" \
  "v_accvgpr_write_b32 a75, 0\n\t" \
  "v_accvgpr_write_b32 a76, 0\n\t" \
  "v_accvgpr_write_b32 a77, 0\n\t" \
  "v_accvgpr_write_b32 a78, 0\n\t" \
  "v_accvgpr_write_b32 a79, 0\n\t" \
  "v_accvgpr_write_b32 a80, 0\n\t" \
  "v_accvgpr_write_b32 a81, 0\n\t" \
  "v_accvgpr_write_b32 a82, 0\n\t" \
  "v_accvgpr_write_b32 a83, 0\n\t" \
  "v_accvgpr_write_b32 a84, 0\n\t" \
  "v_accvgpr_write_b32 a85, 0\n\t" \
  "v_accvgpr_write_b32 a86, 0\n\t" \
  "v_accvgpr_write_b32 a87, 0\n\t" \
  "v_accvgpr_write_b32 a88, 0\n\t" \
  "v_accvgpr_write_b32 a89, 0\n\t" \
  "v_accvgpr_write_b32 a90, 0\n\t" \
  "v_accvgpr_write_b32 a91, 0\n\t" \
  "v_accvgpr_write_b32 a92, 0\n\t" \
  "v_accvgpr_write_b32 a93, 0\n\t" \
  "v_accvgpr_write_b32 a94, 0\n\t" \
  "v_accvgpr_write_b32 a95, 0\n\t" \
  "v_accvgpr_write_b32 a96, 0\n\t" \
  "v_accvgpr_write_b32 a97, 0\n\t" \
  "v_accvgpr_write_b32 a98, 0\n\t" \
  "v_accvgpr_write_b32 a99, 0\n\t" \
  "v_accvgpr_write_b32 a100, 0\n\t" \
  "v_accvgpr_write_b32 a101, 0\n\t" \
  "v_accvgpr_write_b32 a102, 0\n\t" \
  "v_accvgpr_write_b32 a103, 0\n\t" \
  "v_accvgpr_write_b32 a104, 0\n\t" \
  "v_accvgpr_write_b32 a105, 0\n\t" \
  "v_accvgpr_write_b32 a106, 0\n\t" \
  "v_accvgpr_write_b32 a107, 0\n\t" \
  "v_accvgpr_write_b32 a108, 0\n\t" \
  "v_accvgpr_write_b32 a109, 0\n\t" \
  "v_accvgpr_write_b32 a110, 0\n\t" \
  "v_accvgpr_write_b32 a111, 0\n\t" \
  "v_accvgpr_write_b32 a112, 0\n\t" \
  "v_accvgpr_write_b32 a113, 0\n\t" \
  "v_accvgpr_write_b32 a114, 0\n\t" \
  "v_accvgpr_write_b32 a115, 0\n\t" \
  "v_accvgpr_write_b32 a116, 0\n\t" \
  "v_accvgpr_write_b32 a117, 0\n\t" \
  "v_accvgpr_write_b32 a118, 0\n\t" \
  "v_accvgpr_write_b32 a119, 0\n\t" \
  "v_accvgpr_write_b32 a120, 0\n\t" \
  "v_accvgpr_write_b32 a121, 0\n\t" \
  "v_accvgpr_write_b32 a122, 0\n\t" \
  "v_accvgpr_write_b32 a123, 0\n\t" \
  "v_accvgpr_write_b32 a124, 0\n\t" \
  "v_accvgpr_write_b32 a125, 0\n\t" \
  "v_accvgpr_write_b32 a126, 0\n\t" \
  "v_accvgpr_write_b32 a127, 0\n\t" \
  "v_accvgpr_write_b32 a128, 0\n\t" \
  "v_accvgpr_write_b32 a129, 0\n\t" \
  "v_accvgpr_write_b32 a130, 0\n\t" \
  "v_accvgpr_write_b32 a131, 0\n\t" \
  "v_accvgpr_write_b32 a132, 0\n\t" \
  "v_accvgpr_write_b32 a133, 0\n\t" \
  "v_accvgpr_write_b32 a134, 0\n\t" \
  "v_accvgpr_write_b32 a135, 0\n\t" \
  "v_accvgpr_write_b32 a136, 0\n\t" \
  "v_accvgpr_write_b32 a137, 0\n\t" \
  "v_accvgpr_write_b32 a138, 0\n\t" \
  "v_accvgpr_write_b32 a139, 0\n\t" \
  "v_accvgpr_write_b32 a140, 0\n\t" \
  "v_accvgpr_write_b32 a141, 0\n\t" \
  "v_accvgpr_write_b32 a142, 0\n\t" \
  "v_accvgpr_write_b32 a143, 0\n\t" \
  "v_accvgpr_write_b32 a144, 0\n\t" \
  "v_accvgpr_write_b32 a145, 0\n\t" \
  "v_accvgpr_write_b32 a146, 0\n\t" \
  "v_accvgpr_write_b32 a147, 0\n\t" \
  "v_accvgpr_write_b32 a148, 0\n\t" \
  "v_accvgpr_write_b32 a149, 0\n\t" \
  "v_accvgpr_write_b32 a150, 0\n\t" \
  "v_accvgpr_write_b32 a151, 0\n\t" \
  "v_accvgpr_write_b32 a152, 0\n\t" \
  "v_accvgpr_write_b32 a153, 0\n\t" \
  "v_accvgpr_write_b32 a154, 0\n\t" \
  "v_accvgpr_write_b32 a155, 0\n\t" \
  "v_accvgpr_write_b32 a156, 0\n\t" \
  "v_accvgpr_write_b32 a157, 0\n\t" \
  "v_accvgpr_write_b32 a158, 0\n\t" \
  "v_accvgpr_write_b32 a159, 0\n\t" \
  "v_accvgpr_write_b32 a160, 0\n\t" \
  "v_accvgpr_write_b32 a161, 0\n\t" \
  "v_accvgpr_write_b32 a162, 0\n\t" \
  "v_accvgpr_write_b32 a163, 0\n\t" \
  "v_accvgpr_write_b32 a164, 0\n\t" \
  "v_accvgpr_write_b32 a165, 0\n\t" \
  "v_accvgpr_write_b32 a166, 0\n\t" \
  "v_accvgpr_write_b32 a167, 0\n\t" \
  "v_accvgpr_write_b32 a168, 0\n\t" \
  "v_accvgpr_write_b32 a169, 0\n\t" \
  "v_accvgpr_write_b32 a170, 0\n\t" \
  "v_accvgpr_write_b32 a171, 0\n\t" \
  "v_accvgpr_write_b32 a172, 0\n\t" \
  "v_accvgpr_write_b32 a173, 0\n\t" \
  "v_accvgpr_write_b32 a174, 0\n\t" \
  "v_accvgpr_write_b32 a175, 0\n\t" \
  "v_accvgpr_write_b32 a176, 0\n\t" \
  "v_accvgpr_write_b32 a177, 0\n\t" \
  "v_accvgpr_write_b32 a178, 0\n\t" \
  "v_accvgpr_write_b32 a179, 0\n\t" \
  "v_accvgpr_write_b32 a180, 0\n\t" \
  "v_accvgpr_write_b32 a181, 0\n\t" \
  "v_accvgpr_write_b32 a182, 0\n\t" \
  "v_accvgpr_write_b32 a183, 0\n\t" \
  "v_accvgpr_write_b32 a184, 0\n\t" \
  "v_accvgpr_write_b32 a185, 0\n\t" \
  "v_accvgpr_write_b32 a186, 0\n\t" \
  "v_accvgpr_write_b32 a187, 0\n\t" \
  "v_accvgpr_write_b32 a188, 0\n\t" \
  "v_accvgpr_write_b32 a189, 0\n\t" \
  "v_accvgpr_write_b32 a190, 0\n\t" \
  "v_accvgpr_write_b32 a191, 0\n\t" \
  "v_accvgpr_write_b32 a192, 0\n\t" \
  "v_accvgpr_write_b32 a193, 0\n\t" \
  "v_accvgpr_write_b32 a194, 0\n\t" \
  "v_accvgpr_write_b32 a195, 0\n\t" \
  "v_accvgpr_write_b32 a196, 0\n\t" \
  "v_accvgpr_write_b32 a197, 0\n\t" \
  "v_accvgpr_write_b32 a198, 0\n\t" \
  "v_accvgpr_write_b32 a199, 0\n\t" \
  "v_accvgpr_write_b32 a200, 0\n\t" \
  "v_accvgpr_write_b32 a201, 0\n\t" \
  "v_accvgpr_write_b32 a202, 0\n\t" \
  "v_accvgpr_write_b32 a203, 0\n\t" \
  "v_accvgpr_write_b32 a204, 0\n\t" \
  "v_accvgpr_write_b32 a205, 0\n\t" \
  "v_accvgpr_write_b32 a206, 0\n\t" \
  "v_accvgpr_write_b32 a207, 0\n\t" \
  "v_accvgpr_write_b32 a208, 0\n\t" \
  "v_accvgpr_write_b32 a209, 0\n\t" \
  "v_accvgpr_write_b32 a210, 0\n\t" \
  "v_accvgpr_write_b32 a211, 0\n\t" \
  "v_accvgpr_write_b32 a212, 0\n\t" \
  "v_accvgpr_write_b32 a213, 0\n\t" \
  "v_accvgpr_write_b32 a214, 0\n\t" \
  "v_accvgpr_write_b32 a215, 0\n\t" \
  "v_accvgpr_write_b32 a216, 0\n\t" \
  "v_accvgpr_write_b32 a217, 0\n\t" \
  "v_accvgpr_write_b32 a218, 0\n\t" \
  "v_accvgpr_write_b32 a219, 0\n\t" \
  "v_accvgpr_write_b32 a220, 0\n\t" \
  "v_accvgpr_write_b32 a221, 0\n\t" \
  "v_accvgpr_write_b32 a222, 0\n\t" \
  "v_accvgpr_write_b32 a223, 0\n\t" \
  "v_accvgpr_write_b32 a224, 0\n\t" \
  "v_accvgpr_write_b32 a225, 0\n\t" \
  "v_accvgpr_write_b32 a226, 0\n\t" \
  "v_accvgpr_write_b32 a227, 0\n\t" \
  "v_accvgpr_write_b32 a228, 0\n\t" \
  "v_accvgpr_write_b32 a229, 0\n\t" \
  "v_accvgpr_write_b32 a230, 0\n\t" \
  "v_accvgpr_write_b32 a231, 0\n\t" \
  "v_accvgpr_write_b32 a232, 0\n\t" \
  "v_accvgpr_write_b32 a233, 0\n\t" \
  "v_accvgpr_write_b32 a234, 0\n\t" \
  "v_accvgpr_write_b32 a235, 0\n\t" \
  "v_accvgpr_write_b32 a236, 0\n\t" \
  "v_accvgpr_write_b32 a237, 0\n\t" \
  "v_accvgpr_write_b32 a238, 0\n\t" \
  "v_accvgpr_write_b32 a239, 0\n\t" \
  "v_accvgpr_write_b32 a240, 0\n\t" \
  "v_accvgpr_write_b32 a241, 0\n\t" \
  "v_accvgpr_write_b32 a242, 0\n\t" \
  "v_accvgpr_write_b32 a243, 0\n\t" \
  "v_accvgpr_write_b32 a244, 0\n\t" \
  "v_accvgpr_write_b32 a245, 0\n\t" \
  "v_accvgpr_write_b32 a246, 0\n\t" \
  "v_accvgpr_write_b32 a247, 0\n\t" \
  "v_accvgpr_write_b32 a248, 0\n\t" \
  "v_accvgpr_write_b32 a249, 0\n\t" \
  "v_accvgpr_write_b32 a250, 0\n\t" \
  "v_accvgpr_write_b32 a251, 0\n\t" \
  "v_accvgpr_write_b32 a252, 0\n\t" \
  "v_accvgpr_write_b32 a253, 0\n\t" \
  "v_accvgpr_write_b32 a254, 0\n\t" \
  "v_accvgpr_write_b32 a255, 0\n\t" \
  "s_mov_b32 s80, 0\n\t" \
  "s_mov_b32 s86, %[lds]\n\t" \
  "s_add_u32 s81, %[ga0], 256\n\t" \
  "s_add_u32 s82, %[gb0], 256\n\t" \
  "s_waitcnt vmcnt(16)\n\t" \
  "s_barrier\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  "ds_read_b128 v[132:135], %[ra1] offset:0\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:2048\n\t" \
  "ds_read_b128 v[140:143], %[ra1] offset:2048\n\t" \
  "ds_read_b128 v[144:147], %[ra0] offset:4096\n\t" \
  "ds_read_b128 v[148:151], %[ra1] offset:4096\n\t" \
  "ds_read_b128 v[152:155], %[ra0] offset:6144\n\t" \
  "ds_read_b128 v[156:159], %[ra1] offset:6144\n\t" \
  "ds_read_b128 v[248:251], %[rb0] offset:14336\n\t" \
  "ds_read_b128 v[252:255], %[rb1] offset:14336\n\t" \
  "ds_read_b128 v[240:243], %[rb0] offset:12288\n\t" \
  "ds_read_b128 v[244:247], %[rb1] offset:12288\n\t" \
  "ds_read_b128 v[232:235], %[rb0] offset:10240\n\t" \
  "ds_read_b128 v[236:239], %[rb1] offset:10240\n\t" \
  "ds_read_b128 v[224:227], %[rb0] offset:8192\n\t" \
  "ds_read_b128 v[228:231], %[rb1] offset:8192\n\t" \
  "ds_read_b128 v[216:219], %[rb0] offset:6144\n\t" \
  "ds_read_b128 v[220:223], %[rb1] offset:6144\n\t" \
  "ds_read_b128 v[208:211], %[rb0] offset:4096\n\t" \
  "ds_read_b128 v[212:215], %[rb1] offset:4096\n\t" \
  "ds_read_b128 v[200:203], %[rb0] offset:2048\n\t" \
  "ds_read_b128 v[204:207], %[rb1] offset:2048\n\t" \
  "ds_read_b128 v[192:195], %[rb0] offset:0\n\t" \
  "ds_read_b128 v[196:199], %[rb1] offset:0\n\t" \
  "s_nop 7\n\t" \
  "L_sk_loop%=:\n\t" \
  "s_waitcnt lgkmcnt(4)\n\t" \
  MF " a[28:31], v[248:255], v[128:135], a[28:31] " MOD "\n\t" \
  "ds_read_b128 v[160:163], %[ra0] offset:8192\n\t" \
  MF " a[60:63], v[248:255], v[136:143], a[60:63] " MOD "\n\t" \
  MF " a[92:95], v[248:255], v[144:151], a[92:95] " MOD "\n\t" \
  "ds_read_b128 v[164:167], %[ra1] offset:8192\n\t" \
  MF " a[124:127], v[248:255], v[152:159], a[124:127] " MOD "\n\t" \
  MF " a[24:27], v[240:247], v[128:135], a[24:27] " MOD "\n\t" \
  "ds_read_b128 v[168:171], %[ra0] offset:10240\n\t" \
  MF " a[56:59], v[240:247], v[136:143], a[56:59] " MOD "\n\t" \
  MF " a[88:91], v[240:247], v[144:151], a[88:91] " MOD "\n\t" \
  "ds_read_b128 v[172:175], %[ra1] offset:10240\n\t" \
  MF " a[120:123], v[240:247], v[152:159], a[120:123] " MOD "\n\t" \
  MF " a[20:23], v[232:239], v[128:135], a[20:23] " MOD "\n\t" \
  "ds_read_b128 v[176:179], %[ra0] offset:12288\n\t" \
  MF " a[52:55], v[232:239], v[136:143], a[52:55] " MOD "\n\t" \
  MF " a[84:87], v[232:239], v[144:151], a[84:87] " MOD "\n\t" \
  "ds_read_b128 v[180:183], %[ra1] offset:12288\n\t" \
  MF " a[116:119], v[232:239], v[152:159], a[116:119] " MOD "\n\t" \
  MF " a[16:19], v[224:231], v[128:135], a[16:19] " MOD "\n\t" \
  "ds_read_b128 v[184:187], %[ra0] offset:14336\n\t" \
  MF " a[48:51], v[224:231], v[136:143], a[48:51] " MOD "\n\t" \
  MF " a[80:83], v[224:231], v[144:151], a[80:83] " MOD "\n\t" \
  "ds_read_b128 v[188:191], %[ra1] offset:14336\n\t" \
  MF " a[112:115], v[224:231], v[152:159], a[112:115] " MOD "\n\t" \
  MF " a[12:15], v[216:223], v[128:135], a[12:15] " MOD "\n\t" \
  MF " a[44:47], v[216:223], v[136:143], a[44:47] " MOD "\n\t" \
  MF " a[76:79], v[216:223], v[144:151], a[76:79] " MOD "\n\t" \
  MF " a[108:111], v[216:223], v[152:159], a[108:111] " MOD "\n\t" \
  MF " a[8:11], v[208:215], v[128:135], a[8:11] " MOD "\n\t" \
  MF " a[40:43], v[208:215], v[136:143], a[40:43] " MOD "\n\t" \
  MF " a[72:75], v[208:215], v[144:151], a[72:75] " MOD "\n\t" \
  MF " a[104:107], v[208:215], v[152:159], a[104:107] " MOD "\n\t" \
  "s_waitcnt lgkmcnt(10)\n\t" \
  MF " a[4:7], v[200:207], v[128:135], a[4:7] " MOD "\n\t" \
  MF " a[36:39], v[200:207], v[136:143], a[36:39] " MOD "\n\t" \
  MF " a[68:71], v[200:207], v[144:151], a[68:71] " MOD "\n\t" \
  MF " a[100:103], v[200:207], v[152:159], a[100:103] " MOD "\n\t" \
  "s_waitcnt lgkmcnt(8)\n\t" \
  MF " a[0:3], v[192:199], v[128:135], a[0:3] " MOD "\n\t" \
  MF " a[32:35], v[192:199], v[136:143], a[32:35] " MOD "\n\t" \
  MF " a[64:67], v[192:199], v[144:151], a[64:67] " MOD "\n\t" \
  MF " a[96:99], v[192:199], v[152:159], a[96:99] " MOD "\n\t" \
  "s_waitcnt vmcnt(0) lgkmcnt(0)\n\t" \
  "s_barrier\n\t" \
  "s_add_u32 s87, s80, 2\n\t" \
  "s_cmp_lt_u32 s87, %[n]\n\t" \
  "s_cselect_b32 s84, 0, 0x80000000\n\t" \
  "v_or_b32 v120, s84, %[voa]\n\t" \
  "v_or_b32 v121, s84, %[vob]\n\t" \
  "v_xor_b32 %[ra0], 0x10000, %[ra0]\n\t" \
  "v_xor_b32 %[ra1], 0x10000, %[ra1]\n\t" \
  "v_xor_b32 %[rb0], 0x10000, %[rb0]\n\t" \
  "v_xor_b32 %[rb1], 0x10000, %[rb1]\n\t" \
  MF " a[156:159], v[248:255], v[160:167], a[156:159] " MOD "\n\t" \
  "ds_read_b128 v[128:131], %[ra0] offset:0\n\t" \
  MF " a[188:191], v[248:255], v[168:175], a[188:191] " MOD "\n\t" \
  "s_mov_b32 s83, s81\n\t" \
  "s_add_u32 m0, s86, 0\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[220:223], v[248:255], v[176:183], a[220:223] " MOD "\n\t" \
  "ds_read_b128 v[132:135], %[ra1] offset:0\n\t" \
  MF " a[252:255], v[248:255], v[184:191], a[252:255] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 4096\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[152:155], v[240:247], v[160:167], a[152:155] " MOD "\n\t" \
  "ds_read_b128 v[136:139], %[ra0] offset:2048\n\t" \
  MF " a[184:187], v[240:247], v[168:175], a[184:187] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 8192\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "ds_read_b128 v[248:251], %[rb0] offset:14336\n\t" \
  MF " a[216:219], v[240:247], v[176:183], a[216:219] " MOD "\n\t" \
  "ds_read_b128 v[140:143], %[ra1] offset:2048\n\t" \
  "ds_read_b128 v[252:255], %[rb1] offset:14336\n\t" \
  MF " a[248:251], v[240:247], v[184:191], a[248:251] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 12288\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[148:151], v[232:239], v[160:167], a[148:151] " MOD "\n\t" \
  "ds_read_b128 v[144:147], %[ra0] offset:4096\n\t" \
  MF " a[180:183], v[232:239], v[168:175], a[180:183] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 16384\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "ds_read_b128 v[240:243], %[rb0] offset:12288\n\t" \
  MF " a[212:215], v[232:239], v[176:183], a[212:215] " MOD "\n\t" \
  "ds_read_b128 v[148:151], %[ra1] offset:4096\n\t" \
  "ds_read_b128 v[244:247], %[rb1] offset:12288\n\t" \
  MF " a[244:247], v[232:239], v[184:191], a[244:247] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 20480\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[144:147], v[224:231], v[160:167], a[144:147] " MOD "\n\t" \
  "ds_read_b128 v[152:155], %[ra0] offset:6144\n\t" \
  MF " a[176:179], v[224:231], v[168:175], a[176:179] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 24576\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  "ds_read_b128 v[232:235], %[rb0] offset:10240\n\t" \
  MF " a[208:211], v[224:231], v[176:183], a[208:211] " MOD "\n\t" \
  "ds_read_b128 v[156:159], %[ra1] offset:6144\n\t" \
  "ds_read_b128 v[236:239], %[rb1] offset:10240\n\t" \
  MF " a[240:243], v[224:231], v[184:191], a[240:243] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gas]\n\t" \
  "s_add_u32 m0, s86, 28672\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v120, %[rsa], s83 offen lds\n\t" \
  MF " a[140:143], v[216:223], v[160:167], a[140:143] " MOD "\n\t" \
  MF " a[172:175], v[216:223], v[168:175], a[172:175] " MOD "\n\t" \
  "s_mov_b32 s83, s82\n\t" \
  "s_add_u32 m0, s86, 32768\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "ds_read_b128 v[224:227], %[rb0] offset:8192\n\t" \
  MF " a[204:207], v[216:223], v[176:183], a[204:207] " MOD "\n\t" \
  "ds_read_b128 v[228:231], %[rb1] offset:8192\n\t" \
  MF " a[236:239], v[216:223], v[184:191], a[236:239] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 36864\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[136:139], v[208:215], v[160:167], a[136:139] " MOD "\n\t" \
  MF " a[168:171], v[208:215], v[168:175], a[168:171] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 40960\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "ds_read_b128 v[216:219], %[rb0] offset:6144\n\t" \
  MF " a[200:203], v[208:215], v[176:183], a[200:203] " MOD "\n\t" \
  "ds_read_b128 v[220:223], %[rb1] offset:6144\n\t" \
  MF " a[232:235], v[208:215], v[184:191], a[232:235] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 45056\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[132:135], v[200:207], v[160:167], a[132:135] " MOD "\n\t" \
  MF " a[164:167], v[200:207], v[168:175], a[164:167] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 49152\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "ds_read_b128 v[208:211], %[rb0] offset:4096\n\t" \
  MF " a[196:199], v[200:207], v[176:183], a[196:199] " MOD "\n\t" \
  "ds_read_b128 v[212:215], %[rb1] offset:4096\n\t" \
  MF " a[228:231], v[200:207], v[184:191], a[228:231] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 53248\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  MF " a[128:131], v[192:199], v[160:167], a[128:131] " MOD "\n\t" \
  MF " a[160:163], v[192:199], v[168:175], a[160:163] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 57344\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "ds_read_b128 v[200:203], %[rb0] offset:2048\n\t" \
  MF " a[192:195], v[192:199], v[176:183], a[192:195] " MOD "\n\t" \
  "ds_read_b128 v[204:207], %[rb1] offset:2048\n\t" \
  MF " a[224:227], v[192:199], v[184:191], a[224:227] " MOD "\n\t" \
  "s_add_u32 s83, s83, %[gbs]\n\t" \
  "s_add_u32 m0, s86, 61440\n\t" \
  "s_nop 0\n\t" \
  "buffer_load_dwordx4 v121, %[rsb], s83 offen lds\n\t" \
  "ds_read_b128 v[192:195], %[rb0] offset:0\n\t" \
  "ds_read_b128 v[196:199], %[rb1] offset:0\n\t" \
  "s_add_u32 s81, s81, 128\n\t" \
  "s_add_u32 s82, s82, 128\n\t" \
  "s_xor_b32 s86, s86, 0x10000\n\t" \
  "s_add_u32 s80, s80, 1\n\t" \
  "s_cmp_lt_u32 s80, %[n]\n\t" \
  "s_cbranch_scc1 L_sk_loop%=\n\t" \
  "s_waitcnt vmcnt(0) lgkmcnt(0)\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  "s_nop 7\n\t" \
  ""
#define SK_TILE_ASM_STORE_ALL(CVT) \
  "s_mul_i32 s83, %[rowstep], 0\n\t" \
  "s_add_u32 s84, s83, %[q1]\n\t" \
  "s_add_u32 s85, s84, %[q1]\n\t" \
  "s_add_u32 s87, s85, %[q1]\n\t" \
  "v_accvgpr_read_b32 v128, a0\n\t" \
  "v_accvgpr_read_b32 v129, a1\n\t" \
  "v_accvgpr_read_b32 v130, a2\n\t" \
  "v_accvgpr_read_b32 v131, a3\n\t" \
  "v_accvgpr_read_b32 v132, a4\n\t" \
  "v_accvgpr_read_b32 v133, a5\n\t" \
  "v_accvgpr_read_b32 v134, a6\n\t" \
  "v_accvgpr_read_b32 v135, a7\n\t" \
  "v_accvgpr_read_b32 v136, a8\n\t" \
  "v_accvgpr_read_b32 v137, a9\n\t" \
  "v_accvgpr_read_b32 v138, a10\n\t" \
  "v_accvgpr_read_b32 v139, a11\n\t" \
  "v_accvgpr_read_b32 v140, a12\n\t" \
  "v_accvgpr_read_b32 v141, a13\n\t" \
  "v_accvgpr_read_b32 v142, a14\n\t" \
  "v_accvgpr_read_b32 v143, a15\n\t" \
  "v_accvgpr_read_b32 v144, a16\n\t" \
  "v_accvgpr_read_b32 v145, a17\n\t" \
  "v_accvgpr_read_b32 v146, a18\n\t" \
  "v_accvgpr_read_b32 v147, a19\n\t" \
  "v_accvgpr_read_b32 v148, a20\n\t" \
  "v_accvgpr_read_b32 v149, a21\n\t" \
  "v_accvgpr_read_b32 v150, a22\n\t" \
  "v_accvgpr_read_b32 v151, a23\n\t" \
  "v_accvgpr_read_b32 v152, a24\n\t" \
  "v_accvgpr_read_b32 v153, a25\n\t" \
  "v_accvgpr_read_b32 v154, a26\n\t" \
  "v_accvgpr_read_b32 v155, a27\n\t" \
  "v_accvgpr_read_b32 v156, a28\n\t" \
  "v_accvgpr_read_b32 v157, a29\n\t" \
  "v_accvgpr_read_b32 v158, a30\n\t" \
  "v_accvgpr_read_b32 v159, a31\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "v_accvgpr_read_b32 v192, a32\n\t" \
  "v_accvgpr_read_b32 v193, a33\n\t" \
  "v_accvgpr_read_b32 v194, a34\n\t" \
  "v_accvgpr_read_b32 v195, a35\n\t" \
  "v_accvgpr_read_b32 v196, a36\n\t" \
  "v_accvgpr_read_b32 v197, a37\n\t" \
  "v_accvgpr_read_b32 v198, a38\n\t" \
  "v_accvgpr_read_b32 v199, a39\n\t" \
  "v_accvgpr_read_b32 v200, a40\n\t" \
  "v_accvgpr_read_b32 v201, a41\n\t" \
  "v_accvgpr_read_b32 v202, a42\n\t" \
  "v_accvgpr_read_b32 v203, a43\n\t" \
  "v_accvgpr_read_b32 v204, a44\n\t" \
  "v_accvgpr_read_b32 v205, a45\n\t" \
  "v_accvgpr_read_b32 v206, a46\n\t" \
  "v_accvgpr_read_b32 v207, a47\n\t" \
  "v_accvgpr_read_b32 v208, a48\n\t" \
  "v_accvgpr_read_b32 v209, a49\n\t" \
  "v_accvgpr_read_b32 v210, a50\n\t" \
  "v_accvgpr_read_b32 v211, a51\n\t" \
  "v_accvgpr_read_b32 v212, a52\n\t" \
  "v_accvgpr_read_b32 v213, a53\n\t" \
  "v_accvgpr_read_b32 v214, a54\n\t" \
  "v_accvgpr_read_b32 v215, a55\n\t" \
  "v_accvgpr_read_b32 v216, a56\n\t" \
  "v_accvgpr_read_b32 v217, a57\n\t" \
  "v_accvgpr_read_b32 v218, a58\n\t" \
  "v_accvgpr_read_b32 v219, a59\n\t" \
  "v_accvgpr_read_b32 v220, a60\n\t" \
  "v_accvgpr_read_b32 v221, a61\n\t" \
  "v_accvgpr_read_b32 v222, a62\n\t" \
  "v_accvgpr_read_b32 v223, a63\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a64\n\t" \
  "v_accvgpr_read_b32 v129, a65\n\t" \
  "v_accvgpr_read_b32 v130, a66\n\t" \
  "v_accvgpr_read_b32 v131, a67\n\t" \
  "v_accvgpr_read_b32 v132, a68\n\t" \
  "v_accvgpr_read_b32 v133, a69\n\t" \
  "v_accvgpr_read_b32 v134, a70\n\t" \
  "v_accvgpr_read_b32 v135, a71\n\t" \
  "v_accvgpr_read_b32 v136, a72\n\t" \
  "v_accvgpr_read_b32 v137, a73\n\t" \
  "v_accvgpr_read_b32 v138, a74\n\t" \
  "v_accvgpr_read_b32 v139, a75\n\t" \
  "v_accvgpr_read_b32 v140, a76\n\t" \
  "v_accvgpr_read_b32 v141, a77\n\t" \
  "v_accvgpr_read_b32 v142, a78\n\t" \
  "v_accvgpr_read_b32 v143, a79\n\t" \
  "v_accvgpr_read_b32 v144, a80\n\t" \
  "v_accvgpr_read_b32 v145, a81\n\t" \
  "v_accvgpr_read_b32 v146, a82\n\t" \
  "v_accvgpr_read_b32 v147, a83\n\t" \
  "v_accvgpr_read_b32 v148, a84\n\t" \
  "v_accvgpr_read_b32 v149, a85\n\t" \
  "v_accvgpr_read_b32 v150, a86\n\t" \
  "v_accvgpr_read_b32 v151, a87\n\t" \
  "v_accvgpr_read_b32 v152, a88\n\t" \
  "v_accvgpr_read_b32 v153, a89\n\t" \
  "v_accvgpr_read_b32 v154, a90\n\t" \
  "v_accvgpr_read_b32 v155, a91\n\t" \
  "v_accvgpr_read_b32 v156, a92\n\t" \
  "v_accvgpr_read_b32 v157, a93\n\t" \
  "v_accvgpr_read_b32 v158, a94\n\t" \
  "v_accvgpr_read_b32 v159, a95\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a96\n\t" \
  "v_accvgpr_read_b32 v193, a97\n\t" \
  "v_accvgpr_read_b32 v194, a98\n\t" \
  "v_accvgpr_read_b32 v195, a99\n\t" \
  "v_accvgpr_read_b32 v196, a100\n\t" \
  "v_accvgpr_read_b32 v197, a101\n\t" \
  "v_accvgpr_read_b32 v198, a102\n\t" \
  "v_accvgpr_read_b32 v199, a103\n\t" \
  "v_accvgpr_read_b32 v200, a104\n\t" \
  "v_accvgpr_read_b32 v201, a105\n\t" \
  "v_accvgpr_read_b32 v202, a106\n\t" \
  "v_accvgpr_read_b32 v203, a107\n\t" \
  "v_accvgpr_read_b32 v204, a108\n\t" \
  "v_accvgpr_read_b32 v205, a109\n\t" \
  "v_accvgpr_read_b32 v206, a110\n\t" \
  "v_accvgpr_read_b32 v207, a111\n\t" \
  "v_accvgpr_read_b32 v208, a112\n\t" \
  "v_accvgpr_read_b32 v209, a113\n\t" \
  "v_accvgpr_read_b32 v210, a114\n\t" \
  "v_accvgpr_read_b32 v211, a115\n\t" \
  "v_accvgpr_read_b32 v212, a116\n\t" \
  "v_accvgpr_read_b32 v213, a117\n\t" \
  "v_accvgpr_read_b32 v214, a118\n\t" \
  "v_accvgpr_read_b32 v215, a119\n\t" \
  "v_accvgpr_read_b32 v216, a120\n\t" \
  "v_accvgpr_read_b32 v217, a121\n\t" \
  "v_accvgpr_read_b32 v218, a122\n\t" \
  "v_accvgpr_read_b32 v219, a123\n\t" \
  "v_accvgpr_read_b32 v220, a124\n\t" \
  "v_accvgpr_read_b32 v221, a125\n\t" \
  "v_accvgpr_read_b32 v222, a126\n\t" \
  "v_accvgpr_read_b32 v223, a127\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a128\n\t" \
  "v_accvgpr_read_b32 v129, a129\n\t" \
  "v_accvgpr_read_b32 v130, a130\n\t" \
  "v_accvgpr_read_b32 v131, a131\n\t" \
  "v_accvgpr_read_b32 v132, a132\n\t" \
  "v_accvgpr_read_b32 v133, a133\n\t" \
  "v_accvgpr_read_b32 v134, a134\n\t" \
  "v_accvgpr_read_b32 v135, a135\n\t" \
  "v_accvgpr_read_b32 v136, a136\n\t" \
  "v_accvgpr_read_b32 v137, a137\n\t" \
  "v_accvgpr_read_b32 v138, a138\n\t" \
  "v_accvgpr_read_b32 v139, a139\n\t" \
  "v_accvgpr_read_b32 v140, a140\n\t" \
  "v_accvgpr_read_b32 v141, a141\n\t" \
  "v_accvgpr_read_b32 v142, a142\n\t" \
  "v_accvgpr_read_b32 v143, a143\n\t" \
  "v_accvgpr_read_b32 v144, a144\n\t" \
  "v_accvgpr_read_b32 v145, a145\n\t" \
  "v_accvgpr_read_b32 v146, a146\n\t" \
  "v_accvgpr_read_b32 v147, a147\n\t" \
  "v_accvgpr_read_b32 v148, a148\n\t" \
  "v_accvgpr_read_b32 v149, a149\n\t" \
  "v_accvgpr_read_b32 v150, a150\n\t" \
  "v_accvgpr_read_b32 v151, a151\n\t" \
  "v_accvgpr_read_b32 v152, a152\n\t" \
  "v_accvgpr_read_b32 v153, a153\n\t" \
  "v_accvgpr_read_b32 v154, a154\n\t" \
  "v_accvgpr_read_b32 v155, a155\n\t" \
  "v_accvgpr_read_b32 v156, a156\n\t" \
  "v_accvgpr_read_b32 v157, a157\n\t" \
  "v_accvgpr_read_b32 v158, a158\n\t" \
  "v_accvgpr_read_b32 v159, a159\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a160\n\t" \
  "v_accvgpr_read_b32 v193, a161\n\t" \
  "v_accvgpr_read_b32 v194, a162\n\t" \
  "v_accvgpr_read_b32 v195, a163\n\t" \
  "v_accvgpr_read_b32 v196, a164\n\t" \
  "v_accvgpr_read_b32 v197, a165\n\t" \
  "v_accvgpr_read_b32 v198, a166\n\t" \
  "v_accvgpr_read_b32 v199, a167\n\t" \
  "v_accvgpr_read_b32 v200, a168\n\t" \
  "v_accvgpr_read_b32 v201, a169\n\t" \
  "v_accvgpr_read_b32 v202, a170\n\t" \
  "v_accvgpr_read_b32 v203, a171\n\t" \
  "v_accvgpr_read_b32 v204, a172\n\t" \
  "v_accvgpr_read_b32 v205, a173\n\t" \
  "v_accvgpr_read_b32 v206, a174\n\t" \
  "v_accvgpr_read_b32 v207, a175\n\t" \
  "v_accvgpr_read_b32 v208, a176\n\t" \
  "v_accvgpr_read_b32 v209, a177\n\t" \
  "v_accvgpr_read_b32 v210, a178\n\t" \
  "v_accvgpr_read_b32 v211, a179\n\t" \
  "v_accvgpr_read_b32 v212, a180\n\t" \
  "v_accvgpr_read_b32 v213, a181\n\t" \
  "v_accvgpr_read_b32 v214, a182\n\t" \
  "v_accvgpr_read_b32 v215, a183\n\t" \
  "v_accvgpr_read_b32 v216, a184\n\t" \
  "v_accvgpr_read_b32 v217, a185\n\t" \
  "v_accvgpr_read_b32 v218, a186\n\t" \
  "v_accvgpr_read_b32 v219, a187\n\t" \
  "v_accvgpr_read_b32 v220, a188\n\t" \
  "v_accvgpr_read_b32 v221, a189\n\t" \
  "v_accvgpr_read_b32 v222, a190\n\t" \
  "v_accvgpr_read_b32 v223, a191\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a192\n\t" \
  "v_accvgpr_read_b32 v129, a193\n\t" \
  "v_accvgpr_read_b32 v130, a194\n\t" \
  "v_accvgpr_read_b32 v131, a195\n\t" \
  "v_accvgpr_read_b32 v132, a196\n\t" \
  "v_accvgpr_read_b32 v133, a197\n\t" \
  "v_accvgpr_read_b32 v134, a198\n\t" \
  "v_accvgpr_read_b32 v135, a199\n\t" \
  "v_accvgpr_read_b32 v136, a200\n\t" \
  "v_accvgpr_read_b32 v137, a201\n\t" \
  "v_accvgpr_read_b32 v138, a202\n\t" \
  "v_accvgpr_read_b32 v139, a203\n\t" \
  "v_accvgpr_read_b32 v140, a204\n\t" \
  "v_accvgpr_read_b32 v141, a205\n\t" \
  "v_accvgpr_read_b32 v142, a206\n\t" \
  "v_accvgpr_read_b32 v143, a207\n\t" \
  "v_accvgpr_read_b32 v144, a208\n\t" \
  "v_accvgpr_read_b32 v145, a209\n\t" \
  "v_accvgpr_read_b32 v146, a210\n\t" \
  "v_accvgpr_read_b32 v147, a211\n\t" \
  "v_accvgpr_read_b32 v148, a212\n\t" \
  "v_accvgpr_read_b32 v149, a213\n\t" \
  "v_accvgpr_read_b32 v150, a214\n\t" \
  "v_accvgpr_read_b32 v151, a215\n\t" \
  "v_accvgpr_read_b32 v152, a216\n\t" \
  "v_accvgpr_read_b32 v153, a217\n\t" \
  "v_accvgpr_read_b32 v154, a218\n\t" \
  "v_accvgpr_read_b32 v155, a219\n\t" \
  "v_accvgpr_read_b32 v156, a220\n\t" \
  "v_accvgpr_read_b32 v157, a221\n\t" \
  "v_accvgpr_read_b32 v158, a222\n\t" \
  "v_accvgpr_read_b32 v159, a223\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a224\n\t" \
  "v_accvgpr_read_b32 v193, a225\n\t" \
  "v_accvgpr_read_b32 v194, a226\n\t" \
  "v_accvgpr_read_b32 v195, a227\n\t" \
  "v_accvgpr_read_b32 v196, a228\n\t" \
  "v_accvgpr_read_b32 v197, a229\n\t" \
  "v_accvgpr_read_b32 v198, a230\n\t" \
  "v_accvgpr_read_b32 v199, a231\n\t" \
  "v_accvgpr_read_b32 v200, a232\n\t" \
  "v_accvgpr_read_b32 v201, a233\n\t" \
  "v_accvgpr_read_b32 v202, a234\n\t" \
  "v_accvgpr_read_b32 v203, a235\n\t" \
  "v_accvgpr_read_b32 v204, a236\n\t" \
  "v_accvgpr_read_b32 v205, a237\n\t" \
  "v_accvgpr_read_b32 v206, a238\n\t" \
  "v_accvgpr_read_b32 v207, a239\n\t" \
  "v_accvgpr_read_b32 v208, a240\n\t" \
  "v_accvgpr_read_b32 v209, a241\n\t" \
  "v_accvgpr_read_b32 v210, a242\n\t" \
  "v_accvgpr_read_b32 v211, a243\n\t" \
  "v_accvgpr_read_b32 v212, a244\n\t" \
  "v_accvgpr_read_b32 v213, a245\n\t" \
  "v_accvgpr_read_b32 v214, a246\n\t" \
  "v_accvgpr_read_b32 v215, a247\n\t" \
  "v_accvgpr_read_b32 v216, a248\n\t" \
  "v_accvgpr_read_b32 v217, a249\n\t" \
  "v_accvgpr_read_b32 v218, a250\n\t" \
  "v_accvgpr_read_b32 v219, a251\n\t" \
  "v_accvgpr_read_b32 v220, a252\n\t" \
  "v_accvgpr_read_b32 v221, a253\n\t" \
  "v_accvgpr_read_b32 v222, a254\n\t" \
  "v_accvgpr_read_b32 v223, a255\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  ""
#define SK_TILE_ASM_STORE_ALL_SCALED(CVT) \
  "s_mul_i32 s83, %[rowstep], 0\n\t" \
  "s_add_u32 s84, s83, %[q1]\n\t" \
  "s_add_u32 s85, s84, %[q1]\n\t" \
  "s_add_u32 s87, s85, %[q1]\n\t" \
  "v_accvgpr_read_b32 v128, a0\n\t" \
  "v_accvgpr_read_b32 v129, a1\n\t" \
  "v_accvgpr_read_b32 v130, a2\n\t" \
  "v_accvgpr_read_b32 v131, a3\n\t" \
  "v_accvgpr_read_b32 v132, a4\n\t" \
  "v_accvgpr_read_b32 v133, a5\n\t" \
  "v_accvgpr_read_b32 v134, a6\n\t" \
  "v_accvgpr_read_b32 v135, a7\n\t" \
  "v_accvgpr_read_b32 v136, a8\n\t" \
  "v_accvgpr_read_b32 v137, a9\n\t" \
  "v_accvgpr_read_b32 v138, a10\n\t" \
  "v_accvgpr_read_b32 v139, a11\n\t" \
  "v_accvgpr_read_b32 v140, a12\n\t" \
  "v_accvgpr_read_b32 v141, a13\n\t" \
  "v_accvgpr_read_b32 v142, a14\n\t" \
  "v_accvgpr_read_b32 v143, a15\n\t" \
  "v_accvgpr_read_b32 v144, a16\n\t" \
  "v_accvgpr_read_b32 v145, a17\n\t" \
  "v_accvgpr_read_b32 v146, a18\n\t" \
  "v_accvgpr_read_b32 v147, a19\n\t" \
  "v_accvgpr_read_b32 v148, a20\n\t" \
  "v_accvgpr_read_b32 v149, a21\n\t" \
  "v_accvgpr_read_b32 v150, a22\n\t" \
  "v_accvgpr_read_b32 v151, a23\n\t" \
  "v_accvgpr_read_b32 v152, a24\n\t" \
  "v_accvgpr_read_b32 v153, a25\n\t" \
  "v_accvgpr_read_b32 v154, a26\n\t" \
  "v_accvgpr_read_b32 v155, a27\n\t" \
  "v_accvgpr_read_b32 v156, a28\n\t" \
  "v_accvgpr_read_b32 v157, a29\n\t" \
  "v_accvgpr_read_b32 v158, a30\n\t" \
  "v_accvgpr_read_b32 v159, a31\n\t" \
  "v_mul_f32 v128, %[alpha], v128\n\t" \
  "v_mul_f32 v129, %[alpha], v129\n\t" \
  "v_mul_f32 v130, %[alpha], v130\n\t" \
  "v_mul_f32 v131, %[alpha], v131\n\t" \
  "v_mul_f32 v132, %[alpha], v132\n\t" \
  "v_mul_f32 v133, %[alpha], v133\n\t" \
  "v_mul_f32 v134, %[alpha], v134\n\t" \
  "v_mul_f32 v135, %[alpha], v135\n\t" \
  "v_mul_f32 v136, %[alpha], v136\n\t" \
  "v_mul_f32 v137, %[alpha], v137\n\t" \
  "v_mul_f32 v138, %[alpha], v138\n\t" \
  "v_mul_f32 v139, %[alpha], v139\n\t" \
  "v_mul_f32 v140, %[alpha], v140\n\t" \
  "v_mul_f32 v141, %[alpha], v141\n\t" \
  "v_mul_f32 v142, %[alpha], v142\n\t" \
  "v_mul_f32 v143, %[alpha], v143\n\t" \
  "v_mul_f32 v144, %[alpha], v144\n\t" \
  "v_mul_f32 v145, %[alpha], v145\n\t" \
  "v_mul_f32 v146, %[alpha], v146\n\t" \
  "v_mul_f32 v147, %[alpha], v147\n\t" \
  "v_mul_f32 v148, %[alpha], v148\n\t" \
  "v_mul_f32 v149, %[alpha], v149\n\t" \
  "v_mul_f32 v150, %[alpha], v150\n\t" \
  "v_mul_f32 v151, %[alpha], v151\n\t" \
  "v_mul_f32 v152, %[alpha], v152\n\t" \
  "v_mul_f32 v153, %[alpha], v153\n\t" \
  "v_mul_f32 v154, %[alpha], v154\n\t" \
  "v_mul_f32 v155, %[alpha], v155\n\t" \
  "v_mul_f32 v156, %[alpha], v156\n\t" \
  "v_mul_f32 v157, %[alpha], v157\n\t" \
  "v_mul_f32 v158, %[alpha], v158\n\t" \
  "v_mul_f32 v159, %[alpha], v159\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "v_accvgpr_read_b32 v192, a32\n\t" \
  "v_accvgpr_read_b32 v193, a33\n\t" \
  "v_accvgpr_read_b32 v194, a34\n\t" \
  "v_accvgpr_read_b32 v195, a35\n\t" \
  "v_accvgpr_read_b32 v196, a36\n\t" \
  "v_accvgpr_read_b32 v197, a37\n\t" \
  "v_accvgpr_read_b32 v198, a38\n\t" \
  "v_accvgpr_read_b32 v199, a39\n\t" \
  "v_accvgpr_read_b32 v200, a40\n\t" \
  "v_accvgpr_read_b32 v201, a41\n\t" \
  "v_accvgpr_read_b32 v202, a42\n\t" \
  "v_accvgpr_read_b32 v203, a43\n\t" \
  "v_accvgpr_read_b32 v204, a44\n\t" \
  "v_accvgpr_read_b32 v205, a45\n\t" \
  "v_accvgpr_read_b32 v206, a46\n\t" \
  "v_accvgpr_read_b32 v207, a47\n\t" \
  "v_accvgpr_read_b32 v208, a48\n\t" \
  "v_accvgpr_read_b32 v209, a49\n\t" \
  "v_accvgpr_read_b32 v210, a50\n\t" \
  "v_accvgpr_read_b32 v211, a51\n\t" \
  "v_accvgpr_read_b32 v212, a52\n\t" \
  "v_accvgpr_read_b32 v213, a53\n\t" \
  "v_accvgpr_read_b32 v214, a54\n\t" \
  "v_accvgpr_read_b32 v215, a55\n\t" \
  "v_accvgpr_read_b32 v216, a56\n\t" \
  "v_accvgpr_read_b32 v217, a57\n\t" \
  "v_accvgpr_read_b32 v218, a58\n\t" \
  "v_accvgpr_read_b32 v219, a59\n\t" \
  "v_accvgpr_read_b32 v220, a60\n\t" \
  "v_accvgpr_read_b32 v221, a61\n\t" \
  "v_accvgpr_read_b32 v222, a62\n\t" \
  "v_accvgpr_read_b32 v223, a63\n\t" \
  "v_mul_f32 v192, %[alpha], v192\n\t" \
  "v_mul_f32 v193, %[alpha], v193\n\t" \
  "v_mul_f32 v194, %[alpha], v194\n\t" \
  "v_mul_f32 v195, %[alpha], v195\n\t" \
  "v_mul_f32 v196, %[alpha], v196\n\t" \
  "v_mul_f32 v197, %[alpha], v197\n\t" \
  "v_mul_f32 v198, %[alpha], v198\n\t" \
  "v_mul_f32 v199, %[alpha], v199\n\t" \
  "v_mul_f32 v200, %[alpha], v200\n\t" \
  "v_mul_f32 v201, %[alpha], v201\n\t" \
  "v_mul_f32 v202, %[alpha], v202\n\t" \
  "v_mul_f32 v203, %[alpha], v203\n\t" \
  "v_mul_f32 v204, %[alpha], v204\n\t" \
  "v_mul_f32 v205, %[alpha], v205\n\t" \
  "v_mul_f32 v206, %[alpha], v206\n\t" \
  "v_mul_f32 v207, %[alpha], v207\n\t" \
  "v_mul_f32 v208, %[alpha], v208\n\t" \
  "v_mul_f32 v209, %[alpha], v209\n\t" \
  "v_mul_f32 v210, %[alpha], v210\n\t" \
  "v_mul_f32 v211, %[alpha], v211\n\t" \
  "v_mul_f32 v212, %[alpha], v212\n\t" \
  "v_mul_f32 v213, %[alpha], v213\n\t" \
  "v_mul_f32 v214, %[alpha], v214\n\t" \
  "v_mul_f32 v215, %[alpha], v215\n\t" \
  "v_mul_f32 v216, %[alpha], v216\n\t" \
  "v_mul_f32 v217, %[alpha], v217\n\t" \
  "v_mul_f32 v218, %[alpha], v218\n\t" \
  "v_mul_f32 v219, %[alpha], v219\n\t" \
  "v_mul_f32 v220, %[alpha], v220\n\t" \
  "v_mul_f32 v221, %[alpha], v221\n\t" \
  "v_mul_f32 v222, %[alpha], v222\n\t" \
  "v_mul_f32 v223, %[alpha], v223\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a64\n\t" \
  "v_accvgpr_read_b32 v129, a65\n\t" \
  "v_accvgpr_read_b32 v130, a66\n\t" \
  "v_accvgpr_read_b32 v131, a67\n\t" \
  "v_accvgpr_read_b32 v132, a68\n\t" \
  "v_accvgpr_read_b32 v133, a69\n\t" \
  "v_accvgpr_read_b32 v134, a70\n\t" \
  "v_accvgpr_read_b32 v135, a71\n\t" \
  "v_accvgpr_read_b32 v136, a72\n\t" \
  "v_accvgpr_read_b32 v137, a73\n\t" \
  "v_accvgpr_read_b32 v138, a74\n\t" \
  "v_accvgpr_read_b32 v139, a75\n\t" \
  "v_accvgpr_read_b32 v140, a76\n\t" \
  "v_accvgpr_read_b32 v141, a77\n\t" \
  "v_accvgpr_read_b32 v142, a78\n\t" \
  "v_accvgpr_read_b32 v143, a79\n\t" \
  "v_accvgpr_read_b32 v144, a80\n\t" \
  "v_accvgpr_read_b32 v145, a81\n\t" \
  "v_accvgpr_read_b32 v146, a82\n\t" \
  "v_accvgpr_read_b32 v147, a83\n\t" \
  "v_accvgpr_read_b32 v148, a84\n\t" \
  "v_accvgpr_read_b32 v149, a85\n\t" \
  "v_accvgpr_read_b32 v150, a86\n\t" \
  "v_accvgpr_read_b32 v151, a87\n\t" \
  "v_accvgpr_read_b32 v152, a88\n\t" \
  "v_accvgpr_read_b32 v153, a89\n\t" \
  "v_accvgpr_read_b32 v154, a90\n\t" \
  "v_accvgpr_read_b32 v155, a91\n\t" \
  "v_accvgpr_read_b32 v156, a92\n\t" \
  "v_accvgpr_read_b32 v157, a93\n\t" \
  "v_accvgpr_read_b32 v158, a94\n\t" \
  "v_accvgpr_read_b32 v159, a95\n\t" \
  "v_mul_f32 v128, %[alpha], v128\n\t" \
  "v_mul_f32 v129, %[alpha], v129\n\t" \
  "v_mul_f32 v130, %[alpha], v130\n\t" \
  "v_mul_f32 v131, %[alpha], v131\n\t" \
  "v_mul_f32 v132, %[alpha], v132\n\t" \
  "v_mul_f32 v133, %[alpha], v133\n\t" \
  "v_mul_f32 v134, %[alpha], v134\n\t" \
  "v_mul_f32 v135, %[alpha], v135\n\t" \
  "v_mul_f32 v136, %[alpha], v136\n\t" \
  "v_mul_f32 v137, %[alpha], v137\n\t" \
  "v_mul_f32 v138, %[alpha], v138\n\t" \
  "v_mul_f32 v139, %[alpha], v139\n\t" \
  "v_mul_f32 v140, %[alpha], v140\n\t" \
  "v_mul_f32 v141, %[alpha], v141\n\t" \
  "v_mul_f32 v142, %[alpha], v142\n\t" \
  "v_mul_f32 v143, %[alpha], v143\n\t" \
  "v_mul_f32 v144, %[alpha], v144\n\t" \
  "v_mul_f32 v145, %[alpha], v145\n\t" \
  "v_mul_f32 v146, %[alpha], v146\n\t" \
  "v_mul_f32 v147, %[alpha], v147\n\t" \
  "v_mul_f32 v148, %[alpha], v148\n\t" \
  "v_mul_f32 v149, %[alpha], v149\n\t" \
  "v_mul_f32 v150, %[alpha], v150\n\t" \
  "v_mul_f32 v151, %[alpha], v151\n\t" \
  "v_mul_f32 v152, %[alpha], v152\n\t" \
  "v_mul_f32 v153, %[alpha], v153\n\t" \
  "v_mul_f32 v154, %[alpha], v154\n\t" \
  "v_mul_f32 v155, %[alpha], v155\n\t" \
  "v_mul_f32 v156, %[alpha], v156\n\t" \
  "v_mul_f32 v157, %[alpha], v157\n\t" \
  "v_mul_f32 v158, %[alpha], v158\n\t" \
  "v_mul_f32 v159, %[alpha], v159\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a96\n\t" \
  "v_accvgpr_read_b32 v193, a97\n\t" \
  "v_accvgpr_read_b32 v194, a98\n\t" \
  "v_accvgpr_read_b32 v195, a99\n\t" \
  "v_accvgpr_read_b32 v196, a100\n\t" \
  "v_accvgpr_read_b32 v197, a101\n\t" \
  "v_accvgpr_read_b32 v198, a102\n\t" \
  "v_accvgpr_read_b32 v199, a103\n\t" \
  "v_accvgpr_read_b32 v200, a104\n\t" \
  "v_accvgpr_read_b32 v201, a105\n\t" \
  "v_accvgpr_read_b32 v202, a106\n\t" \
  "v_accvgpr_read_b32 v203, a107\n\t" \
  "v_accvgpr_read_b32 v204, a108\n\t" \
  "v_accvgpr_read_b32 v205, a109\n\t" \
  "v_accvgpr_read_b32 v206, a110\n\t" \
  "v_accvgpr_read_b32 v207, a111\n\t" \
  "v_accvgpr_read_b32 v208, a112\n\t" \
  "v_accvgpr_read_b32 v209, a113\n\t" \
  "v_accvgpr_read_b32 v210, a114\n\t" \
  "v_accvgpr_read_b32 v211, a115\n\t" \
  "v_accvgpr_read_b32 v212, a116\n\t" \
  "v_accvgpr_read_b32 v213, a117\n\t" \
  "v_accvgpr_read_b32 v214, a118\n\t" \
  "v_accvgpr_read_b32 v215, a119\n\t" \
  "v_accvgpr_read_b32 v216, a120\n\t" \
  "v_accvgpr_read_b32 v217, a121\n\t" \
  "v_accvgpr_read_b32 v218, a122\n\t" \
  "v_accvgpr_read_b32 v219, a123\n\t" \
  "v_accvgpr_read_b32 v220, a124\n\t" \
  "v_accvgpr_read_b32 v221, a125\n\t" \
  "v_accvgpr_read_b32 v222, a126\n\t" \
  "v_accvgpr_read_b32 v223, a127\n\t" \
  "v_mul_f32 v192, %[alpha], v192\n\t" \
  "v_mul_f32 v193, %[alpha], v193\n\t" \
  "v_mul_f32 v194, %[alpha], v194\n\t" \
  "v_mul_f32 v195, %[alpha], v195\n\t" \
  "v_mul_f32 v196, %[alpha], v196\n\t" \
  "v_mul_f32 v197, %[alpha], v197\n\t" \
  "v_mul_f32 v198, %[alpha], v198\n\t" \
  "v_mul_f32 v199, %[alpha], v199\n\t" \
  "v_mul_f32 v200, %[alpha], v200\n\t" \
  "v_mul_f32 v201, %[alpha], v201\n\t" \
  "v_mul_f32 v202, %[alpha], v202\n\t" \
  "v_mul_f32 v203, %[alpha], v203\n\t" \
  "v_mul_f32 v204, %[alpha], v204\n\t" \
  "v_mul_f32 v205, %[alpha], v205\n\t" \
  "v_mul_f32 v206, %[alpha], v206\n\t" \
  "v_mul_f32 v207, %[alpha], v207\n\t" \
  "v_mul_f32 v208, %[alpha], v208\n\t" \
  "v_mul_f32 v209, %[alpha], v209\n\t" \
  "v_mul_f32 v210, %[alpha], v210\n\t" \
  "v_mul_f32 v211, %[alpha], v211\n\t" \
  "v_mul_f32 v212, %[alpha], v212\n\t" \
  "v_mul_f32 v213, %[alpha], v213\n\t" \
  "v_mul_f32 v214, %[alpha], v214\n\t" \
  "v_mul_f32 v215, %[alpha], v215\n\t" \
  "v_mul_f32 v216, %[alpha], v216\n\t" \
  "v_mul_f32 v217, %[alpha], v217\n\t" \
  "v_mul_f32 v218, %[alpha], v218\n\t" \
  "v_mul_f32 v219, %[alpha], v219\n\t" \
  "v_mul_f32 v220, %[alpha], v220\n\t" \
  "v_mul_f32 v221, %[alpha], v221\n\t" \
  "v_mul_f32 v222, %[alpha], v222\n\t" \
  "v_mul_f32 v223, %[alpha], v223\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a128\n\t" \
  "v_accvgpr_read_b32 v129, a129\n\t" \
  "v_accvgpr_read_b32 v130, a130\n\t" \
  "v_accvgpr_read_b32 v131, a131\n\t" \
  "v_accvgpr_read_b32 v132, a132\n\t" \
  "v_accvgpr_read_b32 v133, a133\n\t" \
  "v_accvgpr_read_b32 v134, a134\n\t" \
  "v_accvgpr_read_b32 v135, a135\n\t" \
  "v_accvgpr_read_b32 v136, a136\n\t" \
  "v_accvgpr_read_b32 v137, a137\n\t" \
  "v_accvgpr_read_b32 v138, a138\n\t" \
  "v_accvgpr_read_b32 v139, a139\n\t" \
  "v_accvgpr_read_b32 v140, a140\n\t" \
  "v_accvgpr_read_b32 v141, a141\n\t" \
  "v_accvgpr_read_b32 v142, a142\n\t" \
  "v_accvgpr_read_b32 v143, a143\n\t" \
  "v_accvgpr_read_b32 v144, a144\n\t" \
  "v_accvgpr_read_b32 v145, a145\n\t" \
  "v_accvgpr_read_b32 v146, a146\n\t" \
  "v_accvgpr_read_b32 v147, a147\n\t" \
  "v_accvgpr_read_b32 v148, a148\n\t" \
  "v_accvgpr_read_b32 v149, a149\n\t" \
  "v_accvgpr_read_b32 v150, a150\n\t" \
  "v_accvgpr_read_b32 v151, a151\n\t" \
  "v_accvgpr_read_b32 v152, a152\n\t" \
  "v_accvgpr_read_b32 v153, a153\n\t" \
  "v_accvgpr_read_b32 v154, a154\n\t" \
  "v_accvgpr_read_b32 v155, a155\n\t" \
  "v_accvgpr_read_b32 v156, a156\n\t" \
  "v_accvgpr_read_b32 v157, a157\n\t" \
  "v_accvgpr_read_b32 v158, a158\n\t" \
  "v_accvgpr_read_b32 v159, a159\n\t" \
  "v_mul_f32 v128, %[alpha], v128\n\t" \
  "v_mul_f32 v129, %[alpha], v129\n\t" \
  "v_mul_f32 v130, %[alpha], v130\n\t" \
  "v_mul_f32 v131, %[alpha], v131\n\t" \
  "v_mul_f32 v132, %[alpha], v132\n\t" \
  "v_mul_f32 v133, %[alpha], v133\n\t" \
  "v_mul_f32 v134, %[alpha], v134\n\t" \
  "v_mul_f32 v135, %[alpha], v135\n\t" \
  "v_mul_f32 v136, %[alpha], v136\n\t" \
  "v_mul_f32 v137, %[alpha], v137\n\t" \
  "v_mul_f32 v138, %[alpha], v138\n\t" \
  "v_mul_f32 v139, %[alpha], v139\n\t" \
  "v_mul_f32 v140, %[alpha], v140\n\t" \
  "v_mul_f32 v141, %[alpha], v141\n\t" \
  "v_mul_f32 v142, %[alpha], v142\n\t" \
  "v_mul_f32 v143, %[alpha], v143\n\t" \
  "v_mul_f32 v144, %[alpha], v144\n\t" \
  "v_mul_f32 v145, %[alpha], v145\n\t" \
  "v_mul_f32 v146, %[alpha], v146\n\t" \
  "v_mul_f32 v147, %[alpha], v147\n\t" \
  "v_mul_f32 v148, %[alpha], v148\n\t" \
  "v_mul_f32 v149, %[alpha], v149\n\t" \
  "v_mul_f32 v150, %[alpha], v150\n\t" \
  "v_mul_f32 v151, %[alpha], v151\n\t" \
  "v_mul_f32 v152, %[alpha], v152\n\t" \
  "v_mul_f32 v153, %[alpha], v153\n\t" \
  "v_mul_f32 v154, %[alpha], v154\n\t" \
  "v_mul_f32 v155, %[alpha], v155\n\t" \
  "v_mul_f32 v156, %[alpha], v156\n\t" \
  "v_mul_f32 v157, %[alpha], v157\n\t" \
  "v_mul_f32 v158, %[alpha], v158\n\t" \
  "v_mul_f32 v159, %[alpha], v159\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a160\n\t" \
  "v_accvgpr_read_b32 v193, a161\n\t" \
  "v_accvgpr_read_b32 v194, a162\n\t" \
  "v_accvgpr_read_b32 v195, a163\n\t" \
  "v_accvgpr_read_b32 v196, a164\n\t" \
  "v_accvgpr_read_b32 v197, a165\n\t" \
  "v_accvgpr_read_b32 v198, a166\n\t" \
  "v_accvgpr_read_b32 v199, a167\n\t" \
  "v_accvgpr_read_b32 v200, a168\n\t" \
  "v_accvgpr_read_b32 v201, a169\n\t" \
  "v_accvgpr_read_b32 v202, a170\n\t" \
  "v_accvgpr_read_b32 v203, a171\n\t" \
  "v_accvgpr_read_b32 v204, a172\n\t" \
  "v_accvgpr_read_b32 v205, a173\n\t" \
  "v_accvgpr_read_b32 v206, a174\n\t" \
  "v_accvgpr_read_b32 v207, a175\n\t" \
  "v_accvgpr_read_b32 v208, a176\n\t" \
  "v_accvgpr_read_b32 v209, a177\n\t" \
  "v_accvgpr_read_b32 v210, a178\n\t" \
  "v_accvgpr_read_b32 v211, a179\n\t" \
  "v_accvgpr_read_b32 v212, a180\n\t" \
  "v_accvgpr_read_b32 v213, a181\n\t" \
  "v_accvgpr_read_b32 v214, a182\n\t" \
  "v_accvgpr_read_b32 v215, a183\n\t" \
  "v_accvgpr_read_b32 v216, a184\n\t" \
  "v_accvgpr_read_b32 v217, a185\n\t" \
  "v_accvgpr_read_b32 v218, a186\n\t" \
  "v_accvgpr_read_b32 v219, a187\n\t" \
  "v_accvgpr_read_b32 v220, a188\n\t" \
  "v_accvgpr_read_b32 v221, a189\n\t" \
  "v_accvgpr_read_b32 v222, a190\n\t" \
  "v_accvgpr_read_b32 v223, a191\n\t" \
  "v_mul_f32 v192, %[alpha], v192\n\t" \
  "v_mul_f32 v193, %[alpha], v193\n\t" \
  "v_mul_f32 v194, %[alpha], v194\n\t" \
  "v_mul_f32 v195, %[alpha], v195\n\t" \
  "v_mul_f32 v196, %[alpha], v196\n\t" \
  "v_mul_f32 v197, %[alpha], v197\n\t" \
  "v_mul_f32 v198, %[alpha], v198\n\t" \
  "v_mul_f32 v199, %[alpha], v199\n\t" \
  "v_mul_f32 v200, %[alpha], v200\n\t" \
  "v_mul_f32 v201, %[alpha], v201\n\t" \
  "v_mul_f32 v202, %[alpha], v202\n\t" \
  "v_mul_f32 v203, %[alpha], v203\n\t" \
  "v_mul_f32 v204, %[alpha], v204\n\t" \
  "v_mul_f32 v205, %[alpha], v205\n\t" \
  "v_mul_f32 v206, %[alpha], v206\n\t" \
  "v_mul_f32 v207, %[alpha], v207\n\t" \
  "v_mul_f32 v208, %[alpha], v208\n\t" \
  "v_mul_f32 v209, %[alpha], v209\n\t" \
  "v_mul_f32 v210, %[alpha], v210\n\t" \
  "v_mul_f32 v211, %[alpha], v211\n\t" \
  "v_mul_f32 v212, %[alpha], v212\n\t" \
  "v_mul_f32 v213, %[alpha], v213\n\t" \
  "v_mul_f32 v214, %[alpha], v214\n\t" \
  "v_mul_f32 v215, %[alpha], v215\n\t" \
  "v_mul_f32 v216, %[alpha], v216\n\t" \
  "v_mul_f32 v217, %[alpha], v217\n\t" \
  "v_mul_f32 v218, %[alpha], v218\n\t" \
  "v_mul_f32 v219, %[alpha], v219\n\t" \
  "v_mul_f32 v220, %[alpha], v220\n\t" \
  "v_mul_f32 v221, %[alpha], v221\n\t" \
  "v_mul_f32 v222, %[alpha], v222\n\t" \
  "v_mul_f32 v223, %[alpha], v223\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a192\n\t" \
  "v_accvgpr_read_b32 v129, a193\n\t" \
  "v_accvgpr_read_b32 v130, a194\n\t" \
  "v_accvgpr_read_b32 v131, a195\n\t" \
  "v_accvgpr_read_b32 v132, a196\n\t" \
  "v_accvgpr_read_b32 v133, a197\n\t" \
  "v_accvgpr_read_b32 v134, a198\n\t" \
  "v_accvgpr_read_b32 v135, a199\n\t" \
  "v_accvgpr_read_b32 v136, a200\n\t" \
  "v_accvgpr_read_b32 v137, a201\n\t" \
  "v_accvgpr_read_b32 v138, a202\n\t" \
  "v_accvgpr_read_b32 v139, a203\n\t" \
  "v_accvgpr_read_b32 v140, a204\n\t" \
  "v_accvgpr_read_b32 v141, a205\n\t" \
  "v_accvgpr_read_b32 v142, a206\n\t" \
  "v_accvgpr_read_b32 v143, a207\n\t" \
  "v_accvgpr_read_b32 v144, a208\n\t" \
  "v_accvgpr_read_b32 v145, a209\n\t" \
  "v_accvgpr_read_b32 v146, a210\n\t" \
  "v_accvgpr_read_b32 v147, a211\n\t" \
  "v_accvgpr_read_b32 v148, a212\n\t" \
  "v_accvgpr_read_b32 v149, a213\n\t" \
  "v_accvgpr_read_b32 v150, a214\n\t" \
  "v_accvgpr_read_b32 v151, a215\n\t" \
  "v_accvgpr_read_b32 v152, a216\n\t" \
  "v_accvgpr_read_b32 v153, a217\n\t" \
  "v_accvgpr_read_b32 v154, a218\n\t" \
  "v_accvgpr_read_b32 v155, a219\n\t" \
  "v_accvgpr_read_b32 v156, a220\n\t" \
  "v_accvgpr_read_b32 v157, a221\n\t" \
  "v_accvgpr_read_b32 v158, a222\n\t" \
  "v_accvgpr_read_b32 v159, a223\n\t" \
  "v_mul_f32 v128, %[alpha], v128\n\t" \
  "v_mul_f32 v129, %[alpha], v129\n\t" \
  "v_mul_f32 v130, %[alpha], v130\n\t" \
  "v_mul_f32 v131, %[alpha], v131\n\t" \
  "v_mul_f32 v132, %[alpha], v132\n\t" \
  "v_mul_f32 v133, %[alpha], v133\n\t" \
  "v_mul_f32 v134, %[alpha], v134\n\t" \
  "v_mul_f32 v135, %[alpha], v135\n\t" \
  "v_mul_f32 v136, %[alpha], v136\n\t" \
  "v_mul_f32 v137, %[alpha], v137\n\t" \
  "v_mul_f32 v138, %[alpha], v138\n\t" \
  "v_mul_f32 v139, %[alpha], v139\n\t" \
  "v_mul_f32 v140, %[alpha], v140\n\t" \
  "v_mul_f32 v141, %[alpha], v141\n\t" \
  "v_mul_f32 v142, %[alpha], v142\n\t" \
  "v_mul_f32 v143, %[alpha], v143\n\t" \
  "v_mul_f32 v144, %[alpha], v144\n\t" \
  "v_mul_f32 v145, %[alpha], v145\n\t" \
  "v_mul_f32 v146, %[alpha], v146\n\t" \
  "v_mul_f32 v147, %[alpha], v147\n\t" \
  "v_mul_f32 v148, %[alpha], v148\n\t" \
  "v_mul_f32 v149, %[alpha], v149\n\t" \
  "v_mul_f32 v150, %[alpha], v150\n\t" \
  "v_mul_f32 v151, %[alpha], v151\n\t" \
  "v_mul_f32 v152, %[alpha], v152\n\t" \
  "v_mul_f32 v153, %[alpha], v153\n\t" \
  "v_mul_f32 v154, %[alpha], v154\n\t" \
  "v_mul_f32 v155, %[alpha], v155\n\t" \
  "v_mul_f32 v156, %[alpha], v156\n\t" \
  "v_mul_f32 v157, %[alpha], v157\n\t" \
  "v_mul_f32 v158, %[alpha], v158\n\t" \
  "v_mul_f32 v159, %[alpha], v159\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a224\n\t" \
  "v_accvgpr_read_b32 v193, a225\n\t" \
  "v_accvgpr_read_b32 v194, a226\n\t" \
  "v_accvgpr_read_b32 v195, a227\n\t" \
  "v_accvgpr_read_b32 v196, a228\n\t" \
  "v_accvgpr_read_b32 v197, a229\n\t" \
  "v_accvgpr_read_b32 v198, a230\n\t" \
  "v_accvgpr_read_b32 v199, a231\n\t" \
  "v_accvgpr_read_b32 v200, a232\n\t" \
  "v_accvgpr_read_b32 v201, a233\n\t" \
  "v_accvgpr_read_b32 v202, a234\n\t" \
  "v_accvgpr_read_b32 v203, a235\n\t" \
  "v_accvgpr_read_b32 v204, a236\n\t" \
  "v_accvgpr_read_b32 v205, a237\n\t" \
  "v_accvgpr_read_b32 v206, a238\n\t" \
  "v_accvgpr_read_b32 v207, a239\n\t" \
  "v_accvgpr_read_b32 v208, a240\n\t" \
  "v_accvgpr_read_b32 v209, a241\n\t" \
  "v_accvgpr_read_b32 v210, a242\n\t" \
  "v_accvgpr_read_b32 v211, a243\n\t" \
  "v_accvgpr_read_b32 v212, a244\n\t" \
  "v_accvgpr_read_b32 v213, a245\n\t" \
  "v_accvgpr_read_b32 v214, a246\n\t" \
  "v_accvgpr_read_b32 v215, a247\n\t" \
  "v_accvgpr_read_b32 v216, a248\n\t" \
  "v_accvgpr_read_b32 v217, a249\n\t" \
  "v_accvgpr_read_b32 v218, a250\n\t" \
  "v_accvgpr_read_b32 v219, a251\n\t" \
  "v_accvgpr_read_b32 v220, a252\n\t" \
  "v_accvgpr_read_b32 v221, a253\n\t" \
  "v_accvgpr_read_b32 v222, a254\n\t" \
  "v_accvgpr_read_b32 v223, a255\n\t" \
  "v_mul_f32 v192, %[alpha], v192\n\t" \
  "v_mul_f32 v193, %[alpha], v193\n\t" \
  "v_mul_f32 v194, %[alpha], v194\n\t" \
  "v_mul_f32 v195, %[alpha], v195\n\t" \
  "v_mul_f32 v196, %[alpha], v196\n\t" \
  "v_mul_f32 v197, %[alpha], v197\n\t" \
  "v_mul_f32 v198, %[alpha], v198\n\t" \
  "v_mul_f32 v199, %[alpha], v199\n\t" \
  "v_mul_f32 v200, %[alpha], v200\n\t" \
  "v_mul_f32 v201, %[alpha], v201\n\t" \
  "v_mul_f32 v202, %[alpha], v202\n\t" \
  "v_mul_f32 v203, %[alpha], v203\n\t" \
  "v_mul_f32 v204, %[alpha], v204\n\t" \
  "v_mul_f32 v205, %[alpha], v205\n\t" \
  "v_mul_f32 v206, %[alpha], v206\n\t" \
  "v_mul_f32 v207, %[alpha], v207\n\t" \
  "v_mul_f32 v208, %[alpha], v208\n\t" \
  "v_mul_f32 v209, %[alpha], v209\n\t" \
  "v_mul_f32 v210, %[alpha], v210\n\t" \
  "v_mul_f32 v211, %[alpha], v211\n\t" \
  "v_mul_f32 v212, %[alpha], v212\n\t" \
  "v_mul_f32 v213, %[alpha], v213\n\t" \
  "v_mul_f32 v214, %[alpha], v214\n\t" \
  "v_mul_f32 v215, %[alpha], v215\n\t" \
  "v_mul_f32 v216, %[alpha], v216\n\t" \
  "v_mul_f32 v217, %[alpha], v217\n\t" \
  "v_mul_f32 v218, %[alpha], v218\n\t" \
  "v_mul_f32 v219, %[alpha], v219\n\t" \
  "v_mul_f32 v220, %[alpha], v220\n\t" \
  "v_mul_f32 v221, %[alpha], v221\n\t" \
  "v_mul_f32 v222, %[alpha], v222\n\t" \
  "v_mul_f32 v223, %[alpha], v223\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  ""
#define SK_TILE_ASM_STORE_ALL_NT(CVT) \
  "s_mul_i32 s83, %[rowstep], 0\n\t" \
  "s_add_u32 s84, s83, %[q1]\n\t" \
  "s_add_u32 s85, s84, %[q1]\n\t" \
  "s_add_u32 s87, s85, %[q1]\n\t" \
  "v_accvgpr_read_b32 v128, a0\n\t" \
  "v_accvgpr_read_b32 v129, a1\n\t" \
  "v_accvgpr_read_b32 v130, a2\n\t" \
  "v_accvgpr_read_b32 v131, a3\n\t" \
  "v_accvgpr_read_b32 v132, a4\n\t" \
  "v_accvgpr_read_b32 v133, a5\n\t" \
  "v_accvgpr_read_b32 v134, a6\n\t" \
  "v_accvgpr_read_b32 v135, a7\n\t" \
  "v_accvgpr_read_b32 v136, a8\n\t" \
  "v_accvgpr_read_b32 v137, a9\n\t" \
  "v_accvgpr_read_b32 v138, a10\n\t" \
  "v_accvgpr_read_b32 v139, a11\n\t" \
  "v_accvgpr_read_b32 v140, a12\n\t" \
  "v_accvgpr_read_b32 v141, a13\n\t" \
  "v_accvgpr_read_b32 v142, a14\n\t" \
  "v_accvgpr_read_b32 v143, a15\n\t" \
  "v_accvgpr_read_b32 v144, a16\n\t" \
  "v_accvgpr_read_b32 v145, a17\n\t" \
  "v_accvgpr_read_b32 v146, a18\n\t" \
  "v_accvgpr_read_b32 v147, a19\n\t" \
  "v_accvgpr_read_b32 v148, a20\n\t" \
  "v_accvgpr_read_b32 v149, a21\n\t" \
  "v_accvgpr_read_b32 v150, a22\n\t" \
  "v_accvgpr_read_b32 v151, a23\n\t" \
  "v_accvgpr_read_b32 v152, a24\n\t" \
  "v_accvgpr_read_b32 v153, a25\n\t" \
  "v_accvgpr_read_b32 v154, a26\n\t" \
  "v_accvgpr_read_b32 v155, a27\n\t" \
  "v_accvgpr_read_b32 v156, a28\n\t" \
  "v_accvgpr_read_b32 v157, a29\n\t" \
  "v_accvgpr_read_b32 v158, a30\n\t" \
  "v_accvgpr_read_b32 v159, a31\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "v_accvgpr_read_b32 v192, a32\n\t" \
  "v_accvgpr_read_b32 v193, a33\n\t" \
  "v_accvgpr_read_b32 v194, a34\n\t" \
  "v_accvgpr_read_b32 v195, a35\n\t" \
  "v_accvgpr_read_b32 v196, a36\n\t" \
  "v_accvgpr_read_b32 v197, a37\n\t" \
  "v_accvgpr_read_b32 v198, a38\n\t" \
  "v_accvgpr_read_b32 v199, a39\n\t" \
  "v_accvgpr_read_b32 v200, a40\n\t" \
  "v_accvgpr_read_b32 v201, a41\n\t" \
  "v_accvgpr_read_b32 v202, a42\n\t" \
  "v_accvgpr_read_b32 v203, a43\n\t" \
  "v_accvgpr_read_b32 v204, a44\n\t" \
  "v_accvgpr_read_b32 v205, a45\n\t" \
  "v_accvgpr_read_b32 v206, a46\n\t" \
  "v_accvgpr_read_b32 v207, a47\n\t" \
  "v_accvgpr_read_b32 v208, a48\n\t" \
  "v_accvgpr_read_b32 v209, a49\n\t" \
  "v_accvgpr_read_b32 v210, a50\n\t" \
  "v_accvgpr_read_b32 v211, a51\n\t" \
  "v_accvgpr_read_b32 v212, a52\n\t" \
  "v_accvgpr_read_b32 v213, a53\n\t" \
  "v_accvgpr_read_b32 v214, a54\n\t" \
  "v_accvgpr_read_b32 v215, a55\n\t" \
  "v_accvgpr_read_b32 v216, a56\n\t" \
  "v_accvgpr_read_b32 v217, a57\n\t" \
  "v_accvgpr_read_b32 v218, a58\n\t" \
  "v_accvgpr_read_b32 v219, a59\n\t" \
  "v_accvgpr_read_b32 v220, a60\n\t" \
  "v_accvgpr_read_b32 v221, a61\n\t" \
  "v_accvgpr_read_b32 v222, a62\n\t" \
  "v_accvgpr_read_b32 v223, a63\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a64\n\t" \
  "v_accvgpr_read_b32 v129, a65\n\t" \
  "v_accvgpr_read_b32 v130, a66\n\t" \
  "v_accvgpr_read_b32 v131, a67\n\t" \
  "v_accvgpr_read_b32 v132, a68\n\t" \
  "v_accvgpr_read_b32 v133, a69\n\t" \
  "v_accvgpr_read_b32 v134, a70\n\t" \
  "v_accvgpr_read_b32 v135, a71\n\t" \
  "v_accvgpr_read_b32 v136, a72\n\t" \
  "v_accvgpr_read_b32 v137, a73\n\t" \
  "v_accvgpr_read_b32 v138, a74\n\t" \
  "v_accvgpr_read_b32 v139, a75\n\t" \
  "v_accvgpr_read_b32 v140, a76\n\t" \
  "v_accvgpr_read_b32 v141, a77\n\t" \
  "v_accvgpr_read_b32 v142, a78\n\t" \
  "v_accvgpr_read_b32 v143, a79\n\t" \
  "v_accvgpr_read_b32 v144, a80\n\t" \
  "v_accvgpr_read_b32 v145, a81\n\t" \
  "v_accvgpr_read_b32 v146, a82\n\t" \
  "v_accvgpr_read_b32 v147, a83\n\t" \
  "v_accvgpr_read_b32 v148, a84\n\t" \
  "v_accvgpr_read_b32 v149, a85\n\t" \
  "v_accvgpr_read_b32 v150, a86\n\t" \
  "v_accvgpr_read_b32 v151, a87\n\t" \
  "v_accvgpr_read_b32 v152, a88\n\t" \
  "v_accvgpr_read_b32 v153, a89\n\t" \
  "v_accvgpr_read_b32 v154, a90\n\t" \
  "v_accvgpr_read_b32 v155, a91\n\t" \
  "v_accvgpr_read_b32 v156, a92\n\t" \
  "v_accvgpr_read_b32 v157, a93\n\t" \
  "v_accvgpr_read_b32 v158, a94\n\t" \
  "v_accvgpr_read_b32 v159, a95\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a96\n\t" \
  "v_accvgpr_read_b32 v193, a97\n\t" \
  "v_accvgpr_read_b32 v194, a98\n\t" \
  "v_accvgpr_read_b32 v195, a99\n\t" \
  "v_accvgpr_read_b32 v196, a100\n\t" \
  "v_accvgpr_read_b32 v197, a101\n\t" \
  "v_accvgpr_read_b32 v198, a102\n\t" \
  "v_accvgpr_read_b32 v199, a103\n\t" \
  "v_accvgpr_read_b32 v200, a104\n\t" \
  "v_accvgpr_read_b32 v201, a105\n\t" \
  "v_accvgpr_read_b32 v202, a106\n\t" \
  "v_accvgpr_read_b32 v203, a107\n\t" \
  "v_accvgpr_read_b32 v204, a108\n\t" \
  "v_accvgpr_read_b32 v205, a109\n\t" \
  "v_accvgpr_read_b32 v206, a110\n\t" \
  "v_accvgpr_read_b32 v207, a111\n\t" \
  "v_accvgpr_read_b32 v208, a112\n\t" \
  "v_accvgpr_read_b32 v209, a113\n\t" \
  "v_accvgpr_read_b32 v210, a114\n\t" \
  "v_accvgpr_read_b32 v211, a115\n\t" \
  "v_accvgpr_read_b32 v212, a116\n\t" \
  "v_accvgpr_read_b32 v213, a117\n\t" \
  "v_accvgpr_read_b32 v214, a118\n\t" \
  "v_accvgpr_read_b32 v215, a119\n\t" \
  "v_accvgpr_read_b32 v216, a120\n\t" \
  "v_accvgpr_read_b32 v217, a121\n\t" \
  "v_accvgpr_read_b32 v218, a122\n\t" \
  "v_accvgpr_read_b32 v219, a123\n\t" \
  "v_accvgpr_read_b32 v220, a124\n\t" \
  "v_accvgpr_read_b32 v221, a125\n\t" \
  "v_accvgpr_read_b32 v222, a126\n\t" \
  "v_accvgpr_read_b32 v223, a127\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a128\n\t" \
  "v_accvgpr_read_b32 v129, a129\n\t" \
  "v_accvgpr_read_b32 v130, a130\n\t" \
  "v_accvgpr_read_b32 v131, a131\n\t" \
  "v_accvgpr_read_b32 v132, a132\n\t" \
  "v_accvgpr_read_b32 v133, a133\n\t" \
  "v_accvgpr_read_b32 v134, a134\n\t" \
  "v_accvgpr_read_b32 v135, a135\n\t" \
  "v_accvgpr_read_b32 v136, a136\n\t" \
  "v_accvgpr_read_b32 v137, a137\n\t" \
  "v_accvgpr_read_b32 v138, a138\n\t" \
  "v_accvgpr_read_b32 v139, a139\n\t" \
  "v_accvgpr_read_b32 v140, a140\n\t" \
  "v_accvgpr_read_b32 v141, a141\n\t" \
  "v_accvgpr_read_b32 v142, a142\n\t" \
  "v_accvgpr_read_b32 v143, a143\n\t" \
  "v_accvgpr_read_b32 v144, a144\n\t" \
  "v_accvgpr_read_b32 v145, a145\n\t" \
  "v_accvgpr_read_b32 v146, a146\n\t" \
  "v_accvgpr_read_b32 v147, a147\n\t" \
  "v_accvgpr_read_b32 v148, a148\n\t" \
  "v_accvgpr_read_b32 v149, a149\n\t" \
  "v_accvgpr_read_b32 v150, a150\n\t" \
  "v_accvgpr_read_b32 v151, a151\n\t" \
  "v_accvgpr_read_b32 v152, a152\n\t" \
  "v_accvgpr_read_b32 v153, a153\n\t" \
  "v_accvgpr_read_b32 v154, a154\n\t" \
  "v_accvgpr_read_b32 v155, a155\n\t" \
  "v_accvgpr_read_b32 v156, a156\n\t" \
  "v_accvgpr_read_b32 v157, a157\n\t" \
  "v_accvgpr_read_b32 v158, a158\n\t" \
  "v_accvgpr_read_b32 v159, a159\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a160\n\t" \
  "v_accvgpr_read_b32 v193, a161\n\t" \
  "v_accvgpr_read_b32 v194, a162\n\t" \
  "v_accvgpr_read_b32 v195, a163\n\t" \
  "v_accvgpr_read_b32 v196, a164\n\t" \
  "v_accvgpr_read_b32 v197, a165\n\t" \
  "v_accvgpr_read_b32 v198, a166\n\t" \
  "v_accvgpr_read_b32 v199, a167\n\t" \
  "v_accvgpr_read_b32 v200, a168\n\t" \
  "v_accvgpr_read_b32 v201, a169\n\t" \
  "v_accvgpr_read_b32 v202, a170\n\t" \
  "v_accvgpr_read_b32 v203, a171\n\t" \
  "v_accvgpr_read_b32 v204, a172\n\t" \
  "v_accvgpr_read_b32 v205, a173\n\t" \
  "v_accvgpr_read_b32 v206, a174\n\t" \
  "v_accvgpr_read_b32 v207, a175\n\t" \
  "v_accvgpr_read_b32 v208, a176\n\t" \
  "v_accvgpr_read_b32 v209, a177\n\t" \
  "v_accvgpr_read_b32 v210, a178\n\t" \
  "v_accvgpr_read_b32 v211, a179\n\t" \
  "v_accvgpr_read_b32 v212, a180\n\t" \
  "v_accvgpr_read_b32 v213, a181\n\t" \
  "v_accvgpr_read_b32 v214, a182\n\t" \
  "v_accvgpr_read_b32 v215, a183\n\t" \
  "v_accvgpr_read_b32 v216, a184\n\t" \
  "v_accvgpr_read_b32 v217, a185\n\t" \
  "v_accvgpr_read_b32 v218, a186\n\t" \
  "v_accvgpr_read_b32 v219, a187\n\t" \
  "v_accvgpr_read_b32 v220, a188\n\t" \
  "v_accvgpr_read_b32 v221, a189\n\t" \
  "v_accvgpr_read_b32 v222, a190\n\t" \
  "v_accvgpr_read_b32 v223, a191\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a192\n\t" \
  "v_accvgpr_read_b32 v129, a193\n\t" \
  "v_accvgpr_read_b32 v130, a194\n\t" \
  "v_accvgpr_read_b32 v131, a195\n\t" \
  "v_accvgpr_read_b32 v132, a196\n\t" \
  "v_accvgpr_read_b32 v133, a197\n\t" \
  "v_accvgpr_read_b32 v134, a198\n\t" \
  "v_accvgpr_read_b32 v135, a199\n\t" \
  "v_accvgpr_read_b32 v136, a200\n\t" \
  "v_accvgpr_read_b32 v137, a201\n\t" \
  "v_accvgpr_read_b32 v138, a202\n\t" \
  "v_accvgpr_read_b32 v139, a203\n\t" \
  "v_accvgpr_read_b32 v140, a204\n\t" \
  "v_accvgpr_read_b32 v141, a205\n\t" \
  "v_accvgpr_read_b32 v142, a206\n\t" \
  "v_accvgpr_read_b32 v143, a207\n\t" \
  "v_accvgpr_read_b32 v144, a208\n\t" \
  "v_accvgpr_read_b32 v145, a209\n\t" \
  "v_accvgpr_read_b32 v146, a210\n\t" \
  "v_accvgpr_read_b32 v147, a211\n\t" \
  "v_accvgpr_read_b32 v148, a212\n\t" \
  "v_accvgpr_read_b32 v149, a213\n\t" \
  "v_accvgpr_read_b32 v150, a214\n\t" \
  "v_accvgpr_read_b32 v151, a215\n\t" \
  "v_accvgpr_read_b32 v152, a216\n\t" \
  "v_accvgpr_read_b32 v153, a217\n\t" \
  "v_accvgpr_read_b32 v154, a218\n\t" \
  "v_accvgpr_read_b32 v155, a219\n\t" \
  "v_accvgpr_read_b32 v156, a220\n\t" \
  "v_accvgpr_read_b32 v157, a221\n\t" \
  "v_accvgpr_read_b32 v158, a222\n\t" \
  "v_accvgpr_read_b32 v159, a223\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a224\n\t" \
  "v_accvgpr_read_b32 v193, a225\n\t" \
  "v_accvgpr_read_b32 v194, a226\n\t" \
  "v_accvgpr_read_b32 v195, a227\n\t" \
  "v_accvgpr_read_b32 v196, a228\n\t" \
  "v_accvgpr_read_b32 v197, a229\n\t" \
  "v_accvgpr_read_b32 v198, a230\n\t" \
  "v_accvgpr_read_b32 v199, a231\n\t" \
  "v_accvgpr_read_b32 v200, a232\n\t" \
  "v_accvgpr_read_b32 v201, a233\n\t" \
  "v_accvgpr_read_b32 v202, a234\n\t" \
  "v_accvgpr_read_b32 v203, a235\n\t" \
  "v_accvgpr_read_b32 v204, a236\n\t" \
  "v_accvgpr_read_b32 v205, a237\n\t" \
  "v_accvgpr_read_b32 v206, a238\n\t" \
  "v_accvgpr_read_b32 v207, a239\n\t" \
  "v_accvgpr_read_b32 v208, a240\n\t" \
  "v_accvgpr_read_b32 v209, a241\n\t" \
  "v_accvgpr_read_b32 v210, a242\n\t" \
  "v_accvgpr_read_b32 v211, a243\n\t" \
  "v_accvgpr_read_b32 v212, a244\n\t" \
  "v_accvgpr_read_b32 v213, a245\n\t" \
  "v_accvgpr_read_b32 v214, a246\n\t" \
  "v_accvgpr_read_b32 v215, a247\n\t" \
  "v_accvgpr_read_b32 v216, a248\n\t" \
  "v_accvgpr_read_b32 v217, a249\n\t" \
  "v_accvgpr_read_b32 v218, a250\n\t" \
  "v_accvgpr_read_b32 v219, a251\n\t" \
  "v_accvgpr_read_b32 v220, a252\n\t" \
  "v_accvgpr_read_b32 v221, a253\n\t" \
  "v_accvgpr_read_b32 v222, a254\n\t" \
  "v_accvgpr_read_b32 v223, a255\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  ""
#define SK_TILE_ASM_STORE_HALF0(CVT) \
  "s_mul_i32 s83, %[rowstep], 0\n\t" \
  "s_add_u32 s84, s83, %[q1]\n\t" \
  "s_add_u32 s85, s84, %[q1]\n\t" \
  "s_add_u32 s87, s85, %[q1]\n\t" \
  "v_accvgpr_read_b32 v128, a0\n\t" \
  "v_accvgpr_read_b32 v129, a1\n\t" \
  "v_accvgpr_read_b32 v130, a2\n\t" \
  "v_accvgpr_read_b32 v131, a3\n\t" \
  "v_accvgpr_read_b32 v132, a4\n\t" \
  "v_accvgpr_read_b32 v133, a5\n\t" \
  "v_accvgpr_read_b32 v134, a6\n\t" \
  "v_accvgpr_read_b32 v135, a7\n\t" \
  "v_accvgpr_read_b32 v136, a8\n\t" \
  "v_accvgpr_read_b32 v137, a9\n\t" \
  "v_accvgpr_read_b32 v138, a10\n\t" \
  "v_accvgpr_read_b32 v139, a11\n\t" \
  "v_accvgpr_read_b32 v140, a12\n\t" \
  "v_accvgpr_read_b32 v141, a13\n\t" \
  "v_accvgpr_read_b32 v142, a14\n\t" \
  "v_accvgpr_read_b32 v143, a15\n\t" \
  "v_accvgpr_read_b32 v144, a16\n\t" \
  "v_accvgpr_read_b32 v145, a17\n\t" \
  "v_accvgpr_read_b32 v146, a18\n\t" \
  "v_accvgpr_read_b32 v147, a19\n\t" \
  "v_accvgpr_read_b32 v148, a20\n\t" \
  "v_accvgpr_read_b32 v149, a21\n\t" \
  "v_accvgpr_read_b32 v150, a22\n\t" \
  "v_accvgpr_read_b32 v151, a23\n\t" \
  "v_accvgpr_read_b32 v152, a24\n\t" \
  "v_accvgpr_read_b32 v153, a25\n\t" \
  "v_accvgpr_read_b32 v154, a26\n\t" \
  "v_accvgpr_read_b32 v155, a27\n\t" \
  "v_accvgpr_read_b32 v156, a28\n\t" \
  "v_accvgpr_read_b32 v157, a29\n\t" \
  "v_accvgpr_read_b32 v158, a30\n\t" \
  "v_accvgpr_read_b32 v159, a31\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "v_accvgpr_read_b32 v192, a32\n\t" \
  "v_accvgpr_read_b32 v193, a33\n\t" \
  "v_accvgpr_read_b32 v194, a34\n\t" \
  "v_accvgpr_read_b32 v195, a35\n\t" \
  "v_accvgpr_read_b32 v196, a36\n\t" \
  "v_accvgpr_read_b32 v197, a37\n\t" \
  "v_accvgpr_read_b32 v198, a38\n\t" \
  "v_accvgpr_read_b32 v199, a39\n\t" \
  "v_accvgpr_read_b32 v200, a40\n\t" \
  "v_accvgpr_read_b32 v201, a41\n\t" \
  "v_accvgpr_read_b32 v202, a42\n\t" \
  "v_accvgpr_read_b32 v203, a43\n\t" \
  "v_accvgpr_read_b32 v204, a44\n\t" \
  "v_accvgpr_read_b32 v205, a45\n\t" \
  "v_accvgpr_read_b32 v206, a46\n\t" \
  "v_accvgpr_read_b32 v207, a47\n\t" \
  "v_accvgpr_read_b32 v208, a48\n\t" \
  "v_accvgpr_read_b32 v209, a49\n\t" \
  "v_accvgpr_read_b32 v210, a50\n\t" \
  "v_accvgpr_read_b32 v211, a51\n\t" \
  "v_accvgpr_read_b32 v212, a52\n\t" \
  "v_accvgpr_read_b32 v213, a53\n\t" \
  "v_accvgpr_read_b32 v214, a54\n\t" \
  "v_accvgpr_read_b32 v215, a55\n\t" \
  "v_accvgpr_read_b32 v216, a56\n\t" \
  "v_accvgpr_read_b32 v217, a57\n\t" \
  "v_accvgpr_read_b32 v218, a58\n\t" \
  "v_accvgpr_read_b32 v219, a59\n\t" \
  "v_accvgpr_read_b32 v220, a60\n\t" \
  "v_accvgpr_read_b32 v221, a61\n\t" \
  "v_accvgpr_read_b32 v222, a62\n\t" \
  "v_accvgpr_read_b32 v223, a63\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a64\n\t" \
  "v_accvgpr_read_b32 v129, a65\n\t" \
  "v_accvgpr_read_b32 v130, a66\n\t" \
  "v_accvgpr_read_b32 v131, a67\n\t" \
  "v_accvgpr_read_b32 v132, a68\n\t" \
  "v_accvgpr_read_b32 v133, a69\n\t" \
  "v_accvgpr_read_b32 v134, a70\n\t" \
  "v_accvgpr_read_b32 v135, a71\n\t" \
  "v_accvgpr_read_b32 v136, a72\n\t" \
  "v_accvgpr_read_b32 v137, a73\n\t" \
  "v_accvgpr_read_b32 v138, a74\n\t" \
  "v_accvgpr_read_b32 v139, a75\n\t" \
  "v_accvgpr_read_b32 v140, a76\n\t" \
  "v_accvgpr_read_b32 v141, a77\n\t" \
  "v_accvgpr_read_b32 v142, a78\n\t" \
  "v_accvgpr_read_b32 v143, a79\n\t" \
  "v_accvgpr_read_b32 v144, a80\n\t" \
  "v_accvgpr_read_b32 v145, a81\n\t" \
  "v_accvgpr_read_b32 v146, a82\n\t" \
  "v_accvgpr_read_b32 v147, a83\n\t" \
  "v_accvgpr_read_b32 v148, a84\n\t" \
  "v_accvgpr_read_b32 v149, a85\n\t" \
  "v_accvgpr_read_b32 v150, a86\n\t" \
  "v_accvgpr_read_b32 v151, a87\n\t" \
  "v_accvgpr_read_b32 v152, a88\n\t" \
  "v_accvgpr_read_b32 v153, a89\n\t" \
  "v_accvgpr_read_b32 v154, a90\n\t" \
  "v_accvgpr_read_b32 v155, a91\n\t" \
  "v_accvgpr_read_b32 v156, a92\n\t" \
  "v_accvgpr_read_b32 v157, a93\n\t" \
  "v_accvgpr_read_b32 v158, a94\n\t" \
  "v_accvgpr_read_b32 v159, a95\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a96\n\t" \
  "v_accvgpr_read_b32 v193, a97\n\t" \
  "v_accvgpr_read_b32 v194, a98\n\t" \
  "v_accvgpr_read_b32 v195, a99\n\t" \
  "v_accvgpr_read_b32 v196, a100\n\t" \
  "v_accvgpr_read_b32 v197, a101\n\t" \
  "v_accvgpr_read_b32 v198, a102\n\t" \
  "v_accvgpr_read_b32 v199, a103\n\t" \
  "v_accvgpr_read_b32 v200, a104\n\t" \
  "v_accvgpr_read_b32 v201, a105\n\t" \
  "v_accvgpr_read_b32 v202, a106\n\t" \
  "v_accvgpr_read_b32 v203, a107\n\t" \
  "v_accvgpr_read_b32 v204, a108\n\t" \
  "v_accvgpr_read_b32 v205, a109\n\t" \
  "v_accvgpr_read_b32 v206, a110\n\t" \
  "v_accvgpr_read_b32 v207, a111\n\t" \
  "v_accvgpr_read_b32 v208, a112\n\t" \
  "v_accvgpr_read_b32 v209, a113\n\t" \
  "v_accvgpr_read_b32 v210, a114\n\t" \
  "v_accvgpr_read_b32 v211, a115\n\t" \
  "v_accvgpr_read_b32 v212, a116\n\t" \
  "v_accvgpr_read_b32 v213, a117\n\t" \
  "v_accvgpr_read_b32 v214, a118\n\t" \
  "v_accvgpr_read_b32 v215, a119\n\t" \
  "v_accvgpr_read_b32 v216, a120\n\t" \
  "v_accvgpr_read_b32 v217, a121\n\t" \
  "v_accvgpr_read_b32 v218, a122\n\t" \
  "v_accvgpr_read_b32 v219, a123\n\t" \
  "v_accvgpr_read_b32 v220, a124\n\t" \
  "v_accvgpr_read_b32 v221, a125\n\t" \
  "v_accvgpr_read_b32 v222, a126\n\t" \
  "v_accvgpr_read_b32 v223, a127\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  ""
#define SK_TILE_ASM_STORE_HALF0_SCALED(CVT) \
  "s_mul_i32 s83, %[rowstep], 0\n\t" \
  "s_add_u32 s84, s83, %[q1]\n\t" \
  "s_add_u32 s85, s84, %[q1]\n\t" \
  "s_add_u32 s87, s85, %[q1]\n\t" \
  "v_accvgpr_read_b32 v128, a0\n\t" \
  "v_accvgpr_read_b32 v129, a1\n\t" \
  "v_accvgpr_read_b32 v130, a2\n\t" \
  "v_accvgpr_read_b32 v131, a3\n\t" \
  "v_accvgpr_read_b32 v132, a4\n\t" \
  "v_accvgpr_read_b32 v133, a5\n\t" \
  "v_accvgpr_read_b32 v134, a6\n\t" \
  "v_accvgpr_read_b32 v135, a7\n\t" \
  "v_accvgpr_read_b32 v136, a8\n\t" \
  "v_accvgpr_read_b32 v137, a9\n\t" \
  "v_accvgpr_read_b32 v138, a10\n\t" \
  "v_accvgpr_read_b32 v139, a11\n\t" \
  "v_accvgpr_read_b32 v140, a12\n\t" \
  "v_accvgpr_read_b32 v141, a13\n\t" \
  "v_accvgpr_read_b32 v142, a14\n\t" \
  "v_accvgpr_read_b32 v143, a15\n\t" \
  "v_accvgpr_read_b32 v144, a16\n\t" \
  "v_accvgpr_read_b32 v145, a17\n\t" \
  "v_accvgpr_read_b32 v146, a18\n\t" \
  "v_accvgpr_read_b32 v147, a19\n\t" \
  "v_accvgpr_read_b32 v148, a20\n\t" \
  "v_accvgpr_read_b32 v149, a21\n\t" \
  "v_accvgpr_read_b32 v150, a22\n\t" \
  "v_accvgpr_read_b32 v151, a23\n\t" \
  "v_accvgpr_read_b32 v152, a24\n\t" \
  "v_accvgpr_read_b32 v153, a25\n\t" \
  "v_accvgpr_read_b32 v154, a26\n\t" \
  "v_accvgpr_read_b32 v155, a27\n\t" \
  "v_accvgpr_read_b32 v156, a28\n\t" \
  "v_accvgpr_read_b32 v157, a29\n\t" \
  "v_accvgpr_read_b32 v158, a30\n\t" \
  "v_accvgpr_read_b32 v159, a31\n\t" \
  "v_mul_f32 v128, %[alpha], v128\n\t" \
  "v_mul_f32 v129, %[alpha], v129\n\t" \
  "v_mul_f32 v130, %[alpha], v130\n\t" \
  "v_mul_f32 v131, %[alpha], v131\n\t" \
  "v_mul_f32 v132, %[alpha], v132\n\t" \
  "v_mul_f32 v133, %[alpha], v133\n\t" \
  "v_mul_f32 v134, %[alpha], v134\n\t" \
  "v_mul_f32 v135, %[alpha], v135\n\t" \
  "v_mul_f32 v136, %[alpha], v136\n\t" \
  "v_mul_f32 v137, %[alpha], v137\n\t" \
  "v_mul_f32 v138, %[alpha], v138\n\t" \
  "v_mul_f32 v139, %[alpha], v139\n\t" \
  "v_mul_f32 v140, %[alpha], v140\n\t" \
  "v_mul_f32 v141, %[alpha], v141\n\t" \
  "v_mul_f32 v142, %[alpha], v142\n\t" \
  "v_mul_f32 v143, %[alpha], v143\n\t" \
  "v_mul_f32 v144, %[alpha], v144\n\t" \
  "v_mul_f32 v145, %[alpha], v145\n\t" \
  "v_mul_f32 v146, %[alpha], v146\n\t" \
  "v_mul_f32 v147, %[alpha], v147\n\t" \
  "v_mul_f32 v148, %[alpha], v148\n\t" \
  "v_mul_f32 v149, %[alpha], v149\n\t" \
  "v_mul_f32 v150, %[alpha], v150\n\t" \
  "v_mul_f32 v151, %[alpha], v151\n\t" \
  "v_mul_f32 v152, %[alpha], v152\n\t" \
  "v_mul_f32 v153, %[alpha], v153\n\t" \
  "v_mul_f32 v154, %[alpha], v154\n\t" \
  "v_mul_f32 v155, %[alpha], v155\n\t" \
  "v_mul_f32 v156, %[alpha], v156\n\t" \
  "v_mul_f32 v157, %[alpha], v157\n\t" \
  "v_mul_f32 v158, %[alpha], v158\n\t" \
  "v_mul_f32 v159, %[alpha], v159\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "v_accvgpr_read_b32 v192, a32\n\t" \
  "v_accvgpr_read_b32 v193, a33\n\t" \
  "v_accvgpr_read_b32 v194, a34\n\t" \
  "v_accvgpr_read_b32 v195, a35\n\t" \
  "v_accvgpr_read_b32 v196, a36\n\t" \
  "v_accvgpr_read_b32 v197, a37\n\t" \
  "v_accvgpr_read_b32 v198, a38\n\t" \
  "v_accvgpr_read_b32 v199, a39\n\t" \
  "v_accvgpr_read_b32 v200, a40\n\t" \
  "v_accvgpr_read_b32 v201, a41\n\t" \
  "v_accvgpr_read_b32 v202, a42\n\t" \
  "v_accvgpr_read_b32 v203, a43\n\t" \
  "v_accvgpr_read_b32 v204, a44\n\t" \
  "v_accvgpr_read_b32 v205, a45\n\t" \
  "v_accvgpr_read_b32 v206, a46\n\t" \
  "v_accvgpr_read_b32 v207, a47\n\t" \
  "v_accvgpr_read_b32 v208, a48\n\t" \
  "v_accvgpr_read_b32 v209, a49\n\t" \
  "v_accvgpr_read_b32 v210, a50\n\t" \
  "v_accvgpr_read_b32 v211, a51\n\t" \
  "v_accvgpr_read_b32 v212, a52\n\t" \
  "v_accvgpr_read_b32 v213, a53\n\t" \
  "v_accvgpr_read_b32 v214, a54\n\t" \
  "v_accvgpr_read_b32 v215, a55\n\t" \
  "v_accvgpr_read_b32 v216, a56\n\t" \
  "v_accvgpr_read_b32 v217, a57\n\t" \
  "v_accvgpr_read_b32 v218, a58\n\t" \
  "v_accvgpr_read_b32 v219, a59\n\t" \
  "v_accvgpr_read_b32 v220, a60\n\t" \
  "v_accvgpr_read_b32 v221, a61\n\t" \
  "v_accvgpr_read_b32 v222, a62\n\t" \
  "v_accvgpr_read_b32 v223, a63\n\t" \
  "v_mul_f32 v192, %[alpha], v192\n\t" \
  "v_mul_f32 v193, %[alpha], v193\n\t" \
  "v_mul_f32 v194, %[alpha], v194\n\t" \
  "v_mul_f32 v195, %[alpha], v195\n\t" \
  "v_mul_f32 v196, %[alpha], v196\n\t" \
  "v_mul_f32 v197, %[alpha], v197\n\t" \
  "v_mul_f32 v198, %[alpha], v198\n\t" \
  "v_mul_f32 v199, %[alpha], v199\n\t" \
  "v_mul_f32 v200, %[alpha], v200\n\t" \
  "v_mul_f32 v201, %[alpha], v201\n\t" \
  "v_mul_f32 v202, %[alpha], v202\n\t" \
  "v_mul_f32 v203, %[alpha], v203\n\t" \
  "v_mul_f32 v204, %[alpha], v204\n\t" \
  "v_mul_f32 v205, %[alpha], v205\n\t" \
  "v_mul_f32 v206, %[alpha], v206\n\t" \
  "v_mul_f32 v207, %[alpha], v207\n\t" \
  "v_mul_f32 v208, %[alpha], v208\n\t" \
  "v_mul_f32 v209, %[alpha], v209\n\t" \
  "v_mul_f32 v210, %[alpha], v210\n\t" \
  "v_mul_f32 v211, %[alpha], v211\n\t" \
  "v_mul_f32 v212, %[alpha], v212\n\t" \
  "v_mul_f32 v213, %[alpha], v213\n\t" \
  "v_mul_f32 v214, %[alpha], v214\n\t" \
  "v_mul_f32 v215, %[alpha], v215\n\t" \
  "v_mul_f32 v216, %[alpha], v216\n\t" \
  "v_mul_f32 v217, %[alpha], v217\n\t" \
  "v_mul_f32 v218, %[alpha], v218\n\t" \
  "v_mul_f32 v219, %[alpha], v219\n\t" \
  "v_mul_f32 v220, %[alpha], v220\n\t" \
  "v_mul_f32 v221, %[alpha], v221\n\t" \
  "v_mul_f32 v222, %[alpha], v222\n\t" \
  "v_mul_f32 v223, %[alpha], v223\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a64\n\t" \
  "v_accvgpr_read_b32 v129, a65\n\t" \
  "v_accvgpr_read_b32 v130, a66\n\t" \
  "v_accvgpr_read_b32 v131, a67\n\t" \
  "v_accvgpr_read_b32 v132, a68\n\t" \
  "v_accvgpr_read_b32 v133, a69\n\t" \
  "v_accvgpr_read_b32 v134, a70\n\t" \
  "v_accvgpr_read_b32 v135, a71\n\t" \
  "v_accvgpr_read_b32 v136, a72\n\t" \
  "v_accvgpr_read_b32 v137, a73\n\t" \
  "v_accvgpr_read_b32 v138, a74\n\t" \
  "v_accvgpr_read_b32 v139, a75\n\t" \
  "v_accvgpr_read_b32 v140, a76\n\t" \
  "v_accvgpr_read_b32 v141, a77\n\t" \
  "v_accvgpr_read_b32 v142, a78\n\t" \
  "v_accvgpr_read_b32 v143, a79\n\t" \
  "v_accvgpr_read_b32 v144, a80\n\t" \
  "v_accvgpr_read_b32 v145, a81\n\t" \
  "v_accvgpr_read_b32 v146, a82\n\t" \
  "v_accvgpr_read_b32 v147, a83\n\t" \
  "v_accvgpr_read_b32 v148, a84\n\t" \
  "v_accvgpr_read_b32 v149, a85\n\t" \
  "v_accvgpr_read_b32 v150, a86\n\t" \
  "v_accvgpr_read_b32 v151, a87\n\t" \
  "v_accvgpr_read_b32 v152, a88\n\t" \
  "v_accvgpr_read_b32 v153, a89\n\t" \
  "v_accvgpr_read_b32 v154, a90\n\t" \
  "v_accvgpr_read_b32 v155, a91\n\t" \
  "v_accvgpr_read_b32 v156, a92\n\t" \
  "v_accvgpr_read_b32 v157, a93\n\t" \
  "v_accvgpr_read_b32 v158, a94\n\t" \
  "v_accvgpr_read_b32 v159, a95\n\t" \
  "v_mul_f32 v128, %[alpha], v128\n\t" \
  "v_mul_f32 v129, %[alpha], v129\n\t" \
  "v_mul_f32 v130, %[alpha], v130\n\t" \
  "v_mul_f32 v131, %[alpha], v131\n\t" \
  "v_mul_f32 v132, %[alpha], v132\n\t" \
  "v_mul_f32 v133, %[alpha], v133\n\t" \
  "v_mul_f32 v134, %[alpha], v134\n\t" \
  "v_mul_f32 v135, %[alpha], v135\n\t" \
  "v_mul_f32 v136, %[alpha], v136\n\t" \
  "v_mul_f32 v137, %[alpha], v137\n\t" \
  "v_mul_f32 v138, %[alpha], v138\n\t" \
  "v_mul_f32 v139, %[alpha], v139\n\t" \
  "v_mul_f32 v140, %[alpha], v140\n\t" \
  "v_mul_f32 v141, %[alpha], v141\n\t" \
  "v_mul_f32 v142, %[alpha], v142\n\t" \
  "v_mul_f32 v143, %[alpha], v143\n\t" \
  "v_mul_f32 v144, %[alpha], v144\n\t" \
  "v_mul_f32 v145, %[alpha], v145\n\t" \
  "v_mul_f32 v146, %[alpha], v146\n\t" \
  "v_mul_f32 v147, %[alpha], v147\n\t" \
  "v_mul_f32 v148, %[alpha], v148\n\t" \
  "v_mul_f32 v149, %[alpha], v149\n\t" \
  "v_mul_f32 v150, %[alpha], v150\n\t" \
  "v_mul_f32 v151, %[alpha], v151\n\t" \
  "v_mul_f32 v152, %[alpha], v152\n\t" \
  "v_mul_f32 v153, %[alpha], v153\n\t" \
  "v_mul_f32 v154, %[alpha], v154\n\t" \
  "v_mul_f32 v155, %[alpha], v155\n\t" \
  "v_mul_f32 v156, %[alpha], v156\n\t" \
  "v_mul_f32 v157, %[alpha], v157\n\t" \
  "v_mul_f32 v158, %[alpha], v158\n\t" \
  "v_mul_f32 v159, %[alpha], v159\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a96\n\t" \
  "v_accvgpr_read_b32 v193, a97\n\t" \
  "v_accvgpr_read_b32 v194, a98\n\t" \
  "v_accvgpr_read_b32 v195, a99\n\t" \
  "v_accvgpr_read_b32 v196, a100\n\t" \
  "v_accvgpr_read_b32 v197, a101\n\t" \
  "v_accvgpr_read_b32 v198, a102\n\t" \
  "v_accvgpr_read_b32 v199, a103\n\t" \
  "v_accvgpr_read_b32 v200, a104\n\t" \
  "v_accvgpr_read_b32 v201, a105\n\t" \
  "v_accvgpr_read_b32 v202, a106\n\t" \
  "v_accvgpr_read_b32 v203, a107\n\t" \
  "v_accvgpr_read_b32 v204, a108\n\t" \
  "v_accvgpr_read_b32 v205, a109\n\t" \
  "v_accvgpr_read_b32 v206, a110\n\t" \
  "v_accvgpr_read_b32 v207, a111\n\t" \
  "v_accvgpr_read_b32 v208, a112\n\t" \
  "v_accvgpr_read_b32 v209, a113\n\t" \
  "v_accvgpr_read_b32 v210, a114\n\t" \
  "v_accvgpr_read_b32 v211, a115\n\t" \
  "v_accvgpr_read_b32 v212, a116\n\t" \
  "v_accvgpr_read_b32 v213, a117\n\t" \
  "v_accvgpr_read_b32 v214, a118\n\t" \
  "v_accvgpr_read_b32 v215, a119\n\t" \
  "v_accvgpr_read_b32 v216, a120\n\t" \
  "v_accvgpr_read_b32 v217, a121\n\t" \
  "v_accvgpr_read_b32 v218, a122\n\t" \
  "v_accvgpr_read_b32 v219, a123\n\t" \
  "v_accvgpr_read_b32 v220, a124\n\t" \
  "v_accvgpr_read_b32 v221, a125\n\t" \
  "v_accvgpr_read_b32 v222, a126\n\t" \
  "v_accvgpr_read_b32 v223, a127\n\t" \
  "v_mul_f32 v192, %[alpha], v192\n\t" \
  "v_mul_f32 v193, %[alpha], v193\n\t" \
  "v_mul_f32 v194, %[alpha], v194\n\t" \
  "v_mul_f32 v195, %[alpha], v195\n\t" \
  "v_mul_f32 v196, %[alpha], v196\n\t" \
  "v_mul_f32 v197, %[alpha], v197\n\t" \
  "v_mul_f32 v198, %[alpha], v198\n\t" \
  "v_mul_f32 v199, %[alpha], v199\n\t" \
  "v_mul_f32 v200, %[alpha], v200\n\t" \
  "v_mul_f32 v201, %[alpha], v201\n\t" \
  "v_mul_f32 v202, %[alpha], v202\n\t" \
  "v_mul_f32 v203, %[alpha], v203\n\t" \
  "v_mul_f32 v204, %[alpha], v204\n\t" \
  "v_mul_f32 v205, %[alpha], v205\n\t" \
  "v_mul_f32 v206, %[alpha], v206\n\t" \
  "v_mul_f32 v207, %[alpha], v207\n\t" \
  "v_mul_f32 v208, %[alpha], v208\n\t" \
  "v_mul_f32 v209, %[alpha], v209\n\t" \
  "v_mul_f32 v210, %[alpha], v210\n\t" \
  "v_mul_f32 v211, %[alpha], v211\n\t" \
  "v_mul_f32 v212, %[alpha], v212\n\t" \
  "v_mul_f32 v213, %[alpha], v213\n\t" \
  "v_mul_f32 v214, %[alpha], v214\n\t" \
  "v_mul_f32 v215, %[alpha], v215\n\t" \
  "v_mul_f32 v216, %[alpha], v216\n\t" \
  "v_mul_f32 v217, %[alpha], v217\n\t" \
  "v_mul_f32 v218, %[alpha], v218\n\t" \
  "v_mul_f32 v219, %[alpha], v219\n\t" \
  "v_mul_f32 v220, %[alpha], v220\n\t" \
  "v_mul_f32 v221, %[alpha], v221\n\t" \
  "v_mul_f32 v222, %[alpha], v222\n\t" \
  "v_mul_f32 v223, %[alpha], v223\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  ""
#define SK_TILE_ASM_STORE_HALF0_NT(CVT) \
  "s_mul_i32 s83, %[rowstep], 0\n\t" \
  "s_add_u32 s84, s83, %[q1]\n\t" \
  "s_add_u32 s85, s84, %[q1]\n\t" \
  "s_add_u32 s87, s85, %[q1]\n\t" \
  "v_accvgpr_read_b32 v128, a0\n\t" \
  "v_accvgpr_read_b32 v129, a1\n\t" \
  "v_accvgpr_read_b32 v130, a2\n\t" \
  "v_accvgpr_read_b32 v131, a3\n\t" \
  "v_accvgpr_read_b32 v132, a4\n\t" \
  "v_accvgpr_read_b32 v133, a5\n\t" \
  "v_accvgpr_read_b32 v134, a6\n\t" \
  "v_accvgpr_read_b32 v135, a7\n\t" \
  "v_accvgpr_read_b32 v136, a8\n\t" \
  "v_accvgpr_read_b32 v137, a9\n\t" \
  "v_accvgpr_read_b32 v138, a10\n\t" \
  "v_accvgpr_read_b32 v139, a11\n\t" \
  "v_accvgpr_read_b32 v140, a12\n\t" \
  "v_accvgpr_read_b32 v141, a13\n\t" \
  "v_accvgpr_read_b32 v142, a14\n\t" \
  "v_accvgpr_read_b32 v143, a15\n\t" \
  "v_accvgpr_read_b32 v144, a16\n\t" \
  "v_accvgpr_read_b32 v145, a17\n\t" \
  "v_accvgpr_read_b32 v146, a18\n\t" \
  "v_accvgpr_read_b32 v147, a19\n\t" \
  "v_accvgpr_read_b32 v148, a20\n\t" \
  "v_accvgpr_read_b32 v149, a21\n\t" \
  "v_accvgpr_read_b32 v150, a22\n\t" \
  "v_accvgpr_read_b32 v151, a23\n\t" \
  "v_accvgpr_read_b32 v152, a24\n\t" \
  "v_accvgpr_read_b32 v153, a25\n\t" \
  "v_accvgpr_read_b32 v154, a26\n\t" \
  "v_accvgpr_read_b32 v155, a27\n\t" \
  "v_accvgpr_read_b32 v156, a28\n\t" \
  "v_accvgpr_read_b32 v157, a29\n\t" \
  "v_accvgpr_read_b32 v158, a30\n\t" \
  "v_accvgpr_read_b32 v159, a31\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "v_accvgpr_read_b32 v192, a32\n\t" \
  "v_accvgpr_read_b32 v193, a33\n\t" \
  "v_accvgpr_read_b32 v194, a34\n\t" \
  "v_accvgpr_read_b32 v195, a35\n\t" \
  "v_accvgpr_read_b32 v196, a36\n\t" \
  "v_accvgpr_read_b32 v197, a37\n\t" \
  "v_accvgpr_read_b32 v198, a38\n\t" \
  "v_accvgpr_read_b32 v199, a39\n\t" \
  "v_accvgpr_read_b32 v200, a40\n\t" \
  "v_accvgpr_read_b32 v201, a41\n\t" \
  "v_accvgpr_read_b32 v202, a42\n\t" \
  "v_accvgpr_read_b32 v203, a43\n\t" \
  "v_accvgpr_read_b32 v204, a44\n\t" \
  "v_accvgpr_read_b32 v205, a45\n\t" \
  "v_accvgpr_read_b32 v206, a46\n\t" \
  "v_accvgpr_read_b32 v207, a47\n\t" \
  "v_accvgpr_read_b32 v208, a48\n\t" \
  "v_accvgpr_read_b32 v209, a49\n\t" \
  "v_accvgpr_read_b32 v210, a50\n\t" \
  "v_accvgpr_read_b32 v211, a51\n\t" \
  "v_accvgpr_read_b32 v212, a52\n\t" \
  "v_accvgpr_read_b32 v213, a53\n\t" \
  "v_accvgpr_read_b32 v214, a54\n\t" \
  "v_accvgpr_read_b32 v215, a55\n\t" \
  "v_accvgpr_read_b32 v216, a56\n\t" \
  "v_accvgpr_read_b32 v217, a57\n\t" \
  "v_accvgpr_read_b32 v218, a58\n\t" \
  "v_accvgpr_read_b32 v219, a59\n\t" \
  "v_accvgpr_read_b32 v220, a60\n\t" \
  "v_accvgpr_read_b32 v221, a61\n\t" \
  "v_accvgpr_read_b32 v222, a62\n\t" \
  "v_accvgpr_read_b32 v223, a63\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a64\n\t" \
  "v_accvgpr_read_b32 v129, a65\n\t" \
  "v_accvgpr_read_b32 v130, a66\n\t" \
  "v_accvgpr_read_b32 v131, a67\n\t" \
  "v_accvgpr_read_b32 v132, a68\n\t" \
  "v_accvgpr_read_b32 v133, a69\n\t" \
  "v_accvgpr_read_b32 v134, a70\n\t" \
  "v_accvgpr_read_b32 v135, a71\n\t" \
  "v_accvgpr_read_b32 v136, a72\n\t" \
  "v_accvgpr_read_b32 v137, a73\n\t" \
  "v_accvgpr_read_b32 v138, a74\n\t" \
  "v_accvgpr_read_b32 v139, a75\n\t" \
  "v_accvgpr_read_b32 v140, a76\n\t" \
  "v_accvgpr_read_b32 v141, a77\n\t" \
  "v_accvgpr_read_b32 v142, a78\n\t" \
  "v_accvgpr_read_b32 v143, a79\n\t" \
  "v_accvgpr_read_b32 v144, a80\n\t" \
  "v_accvgpr_read_b32 v145, a81\n\t" \
  "v_accvgpr_read_b32 v146, a82\n\t" \
  "v_accvgpr_read_b32 v147, a83\n\t" \
  "v_accvgpr_read_b32 v148, a84\n\t" \
  "v_accvgpr_read_b32 v149, a85\n\t" \
  "v_accvgpr_read_b32 v150, a86\n\t" \
  "v_accvgpr_read_b32 v151, a87\n\t" \
  "v_accvgpr_read_b32 v152, a88\n\t" \
  "v_accvgpr_read_b32 v153, a89\n\t" \
  "v_accvgpr_read_b32 v154, a90\n\t" \
  "v_accvgpr_read_b32 v155, a91\n\t" \
  "v_accvgpr_read_b32 v156, a92\n\t" \
  "v_accvgpr_read_b32 v157, a93\n\t" \
  "v_accvgpr_read_b32 v158, a94\n\t" \
  "v_accvgpr_read_b32 v159, a95\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a96\n\t" \
  "v_accvgpr_read_b32 v193, a97\n\t" \
  "v_accvgpr_read_b32 v194, a98\n\t" \
  "v_accvgpr_read_b32 v195, a99\n\t" \
  "v_accvgpr_read_b32 v196, a100\n\t" \
  "v_accvgpr_read_b32 v197, a101\n\t" \
  "v_accvgpr_read_b32 v198, a102\n\t" \
  "v_accvgpr_read_b32 v199, a103\n\t" \
  "v_accvgpr_read_b32 v200, a104\n\t" \
  "v_accvgpr_read_b32 v201, a105\n\t" \
  "v_accvgpr_read_b32 v202, a106\n\t" \
  "v_accvgpr_read_b32 v203, a107\n\t" \
  "v_accvgpr_read_b32 v204, a108\n\t" \
  "v_accvgpr_read_b32 v205, a109\n\t" \
  "v_accvgpr_read_b32 v206, a110\n\t" \
  "v_accvgpr_read_b32 v207, a111\n\t" \
  "v_accvgpr_read_b32 v208, a112\n\t" \
  "v_accvgpr_read_b32 v209, a113\n\t" \
  "v_accvgpr_read_b32 v210, a114\n\t" \
  "v_accvgpr_read_b32 v211, a115\n\t" \
  "v_accvgpr_read_b32 v212, a116\n\t" \
  "v_accvgpr_read_b32 v213, a117\n\t" \
  "v_accvgpr_read_b32 v214, a118\n\t" \
  "v_accvgpr_read_b32 v215, a119\n\t" \
  "v_accvgpr_read_b32 v216, a120\n\t" \
  "v_accvgpr_read_b32 v217, a121\n\t" \
  "v_accvgpr_read_b32 v218, a122\n\t" \
  "v_accvgpr_read_b32 v219, a123\n\t" \
  "v_accvgpr_read_b32 v220, a124\n\t" \
  "v_accvgpr_read_b32 v221, a125\n\t" \
  "v_accvgpr_read_b32 v222, a126\n\t" \
  "v_accvgpr_read_b32 v223, a127\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  ""
#define SK_TILE_ASM_STORE_HALF1(CVT) \
  "s_mul_i32 s83, %[rowstep], 4\n\t" \
  "s_add_u32 s84, s83, %[q1]\n\t" \
  "s_add_u32 s85, s84, %[q1]\n\t" \
  "s_add_u32 s87, s85, %[q1]\n\t" \
  "v_accvgpr_read_b32 v128, a128\n\t" \
  "v_accvgpr_read_b32 v129, a129\n\t" \
  "v_accvgpr_read_b32 v130, a130\n\t" \
  "v_accvgpr_read_b32 v131, a131\n\t" \
  "v_accvgpr_read_b32 v132, a132\n\t" \
  "v_accvgpr_read_b32 v133, a133\n\t" \
  "v_accvgpr_read_b32 v134, a134\n\t" \
  "v_accvgpr_read_b32 v135, a135\n\t" \
  "v_accvgpr_read_b32 v136, a136\n\t" \
  "v_accvgpr_read_b32 v137, a137\n\t" \
  "v_accvgpr_read_b32 v138, a138\n\t" \
  "v_accvgpr_read_b32 v139, a139\n\t" \
  "v_accvgpr_read_b32 v140, a140\n\t" \
  "v_accvgpr_read_b32 v141, a141\n\t" \
  "v_accvgpr_read_b32 v142, a142\n\t" \
  "v_accvgpr_read_b32 v143, a143\n\t" \
  "v_accvgpr_read_b32 v144, a144\n\t" \
  "v_accvgpr_read_b32 v145, a145\n\t" \
  "v_accvgpr_read_b32 v146, a146\n\t" \
  "v_accvgpr_read_b32 v147, a147\n\t" \
  "v_accvgpr_read_b32 v148, a148\n\t" \
  "v_accvgpr_read_b32 v149, a149\n\t" \
  "v_accvgpr_read_b32 v150, a150\n\t" \
  "v_accvgpr_read_b32 v151, a151\n\t" \
  "v_accvgpr_read_b32 v152, a152\n\t" \
  "v_accvgpr_read_b32 v153, a153\n\t" \
  "v_accvgpr_read_b32 v154, a154\n\t" \
  "v_accvgpr_read_b32 v155, a155\n\t" \
  "v_accvgpr_read_b32 v156, a156\n\t" \
  "v_accvgpr_read_b32 v157, a157\n\t" \
  "v_accvgpr_read_b32 v158, a158\n\t" \
  "v_accvgpr_read_b32 v159, a159\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "v_accvgpr_read_b32 v192, a160\n\t" \
  "v_accvgpr_read_b32 v193, a161\n\t" \
  "v_accvgpr_read_b32 v194, a162\n\t" \
  "v_accvgpr_read_b32 v195, a163\n\t" \
  "v_accvgpr_read_b32 v196, a164\n\t" \
  "v_accvgpr_read_b32 v197, a165\n\t" \
  "v_accvgpr_read_b32 v198, a166\n\t" \
  "v_accvgpr_read_b32 v199, a167\n\t" \
  "v_accvgpr_read_b32 v200, a168\n\t" \
  "v_accvgpr_read_b32 v201, a169\n\t" \
  "v_accvgpr_read_b32 v202, a170\n\t" \
  "v_accvgpr_read_b32 v203, a171\n\t" \
  "v_accvgpr_read_b32 v204, a172\n\t" \
  "v_accvgpr_read_b32 v205, a173\n\t" \
  "v_accvgpr_read_b32 v206, a174\n\t" \
  "v_accvgpr_read_b32 v207, a175\n\t" \
  "v_accvgpr_read_b32 v208, a176\n\t" \
  "v_accvgpr_read_b32 v209, a177\n\t" \
  "v_accvgpr_read_b32 v210, a178\n\t" \
  "v_accvgpr_read_b32 v211, a179\n\t" \
  "v_accvgpr_read_b32 v212, a180\n\t" \
  "v_accvgpr_read_b32 v213, a181\n\t" \
  "v_accvgpr_read_b32 v214, a182\n\t" \
  "v_accvgpr_read_b32 v215, a183\n\t" \
  "v_accvgpr_read_b32 v216, a184\n\t" \
  "v_accvgpr_read_b32 v217, a185\n\t" \
  "v_accvgpr_read_b32 v218, a186\n\t" \
  "v_accvgpr_read_b32 v219, a187\n\t" \
  "v_accvgpr_read_b32 v220, a188\n\t" \
  "v_accvgpr_read_b32 v221, a189\n\t" \
  "v_accvgpr_read_b32 v222, a190\n\t" \
  "v_accvgpr_read_b32 v223, a191\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a192\n\t" \
  "v_accvgpr_read_b32 v129, a193\n\t" \
  "v_accvgpr_read_b32 v130, a194\n\t" \
  "v_accvgpr_read_b32 v131, a195\n\t" \
  "v_accvgpr_read_b32 v132, a196\n\t" \
  "v_accvgpr_read_b32 v133, a197\n\t" \
  "v_accvgpr_read_b32 v134, a198\n\t" \
  "v_accvgpr_read_b32 v135, a199\n\t" \
  "v_accvgpr_read_b32 v136, a200\n\t" \
  "v_accvgpr_read_b32 v137, a201\n\t" \
  "v_accvgpr_read_b32 v138, a202\n\t" \
  "v_accvgpr_read_b32 v139, a203\n\t" \
  "v_accvgpr_read_b32 v140, a204\n\t" \
  "v_accvgpr_read_b32 v141, a205\n\t" \
  "v_accvgpr_read_b32 v142, a206\n\t" \
  "v_accvgpr_read_b32 v143, a207\n\t" \
  "v_accvgpr_read_b32 v144, a208\n\t" \
  "v_accvgpr_read_b32 v145, a209\n\t" \
  "v_accvgpr_read_b32 v146, a210\n\t" \
  "v_accvgpr_read_b32 v147, a211\n\t" \
  "v_accvgpr_read_b32 v148, a212\n\t" \
  "v_accvgpr_read_b32 v149, a213\n\t" \
  "v_accvgpr_read_b32 v150, a214\n\t" \
  "v_accvgpr_read_b32 v151, a215\n\t" \
  "v_accvgpr_read_b32 v152, a216\n\t" \
  "v_accvgpr_read_b32 v153, a217\n\t" \
  "v_accvgpr_read_b32 v154, a218\n\t" \
  "v_accvgpr_read_b32 v155, a219\n\t" \
  "v_accvgpr_read_b32 v156, a220\n\t" \
  "v_accvgpr_read_b32 v157, a221\n\t" \
  "v_accvgpr_read_b32 v158, a222\n\t" \
  "v_accvgpr_read_b32 v159, a223\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a224\n\t" \
  "v_accvgpr_read_b32 v193, a225\n\t" \
  "v_accvgpr_read_b32 v194, a226\n\t" \
  "v_accvgpr_read_b32 v195, a227\n\t" \
  "v_accvgpr_read_b32 v196, a228\n\t" \
  "v_accvgpr_read_b32 v197, a229\n\t" \
  "v_accvgpr_read_b32 v198, a230\n\t" \
  "v_accvgpr_read_b32 v199, a231\n\t" \
  "v_accvgpr_read_b32 v200, a232\n\t" \
  "v_accvgpr_read_b32 v201, a233\n\t" \
  "v_accvgpr_read_b32 v202, a234\n\t" \
  "v_accvgpr_read_b32 v203, a235\n\t" \
  "v_accvgpr_read_b32 v204, a236\n\t" \
  "v_accvgpr_read_b32 v205, a237\n\t" \
  "v_accvgpr_read_b32 v206, a238\n\t" \
  "v_accvgpr_read_b32 v207, a239\n\t" \
  "v_accvgpr_read_b32 v208, a240\n\t" \
  "v_accvgpr_read_b32 v209, a241\n\t" \
  "v_accvgpr_read_b32 v210, a242\n\t" \
  "v_accvgpr_read_b32 v211, a243\n\t" \
  "v_accvgpr_read_b32 v212, a244\n\t" \
  "v_accvgpr_read_b32 v213, a245\n\t" \
  "v_accvgpr_read_b32 v214, a246\n\t" \
  "v_accvgpr_read_b32 v215, a247\n\t" \
  "v_accvgpr_read_b32 v216, a248\n\t" \
  "v_accvgpr_read_b32 v217, a249\n\t" \
  "v_accvgpr_read_b32 v218, a250\n\t" \
  "v_accvgpr_read_b32 v219, a251\n\t" \
  "v_accvgpr_read_b32 v220, a252\n\t" \
  "v_accvgpr_read_b32 v221, a253\n\t" \
  "v_accvgpr_read_b32 v222, a254\n\t" \
  "v_accvgpr_read_b32 v223, a255\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  ""
#define SK_TILE_ASM_STORE_HALF1_SCALED(CVT) \
  "s_mul_i32 s83, %[rowstep], 4\n\t" \
  "s_add_u32 s84, s83, %[q1]\n\t" \
  "s_add_u32 s85, s84, %[q1]\n\t" \
  "s_add_u32 s87, s85, %[q1]\n\t" \
  "v_accvgpr_read_b32 v128, a128\n\t" \
  "v_accvgpr_read_b32 v129, a129\n\t" \
  "v_accvgpr_read_b32 v130, a130\n\t" \
  "v_accvgpr_read_b32 v131, a131\n\t" \
  "v_accvgpr_read_b32 v132, a132\n\t" \
  "v_accvgpr_read_b32 v133, a133\n\t" \
  "v_accvgpr_read_b32 v134, a134\n\t" \
  "v_accvgpr_read_b32 v135, a135\n\t" \
  "v_accvgpr_read_b32 v136, a136\n\t" \
  "v_accvgpr_read_b32 v137, a137\n\t" \
  "v_accvgpr_read_b32 v138, a138\n\t" \
  "v_accvgpr_read_b32 v139, a139\n\t" \
  "v_accvgpr_read_b32 v140, a140\n\t" \
  "v_accvgpr_read_b32 v141, a141\n\t" \
  "v_accvgpr_read_b32 v142, a142\n\t" \
  "v_accvgpr_read_b32 v143, a143\n\t" \
  "v_accvgpr_read_b32 v144, a144\n\t" \
  "v_accvgpr_read_b32 v145, a145\n\t" \
  "v_accvgpr_read_b32 v146, a146\n\t" \
  "v_accvgpr_read_b32 v147, a147\n\t" \
  "v_accvgpr_read_b32 v148, a148\n\t" \
  "v_accvgpr_read_b32 v149, a149\n\t" \
  "v_accvgpr_read_b32 v150, a150\n\t" \
  "v_accvgpr_read_b32 v151, a151\n\t" \
  "v_accvgpr_read_b32 v152, a152\n\t" \
  "v_accvgpr_read_b32 v153, a153\n\t" \
  "v_accvgpr_read_b32 v154, a154\n\t" \
  "v_accvgpr_read_b32 v155, a155\n\t" \
  "v_accvgpr_read_b32 v156, a156\n\t" \
  "v_accvgpr_read_b32 v157, a157\n\t" \
  "v_accvgpr_read_b32 v158, a158\n\t" \
  "v_accvgpr_read_b32 v159, a159\n\t" \
  "v_mul_f32 v128, %[alpha], v128\n\t" \
  "v_mul_f32 v129, %[alpha], v129\n\t" \
  "v_mul_f32 v130, %[alpha], v130\n\t" \
  "v_mul_f32 v131, %[alpha], v131\n\t" \
  "v_mul_f32 v132, %[alpha], v132\n\t" \
  "v_mul_f32 v133, %[alpha], v133\n\t" \
  "v_mul_f32 v134, %[alpha], v134\n\t" \
  "v_mul_f32 v135, %[alpha], v135\n\t" \
  "v_mul_f32 v136, %[alpha], v136\n\t" \
  "v_mul_f32 v137, %[alpha], v137\n\t" \
  "v_mul_f32 v138, %[alpha], v138\n\t" \
  "v_mul_f32 v139, %[alpha], v139\n\t" \
  "v_mul_f32 v140, %[alpha], v140\n\t" \
  "v_mul_f32 v141, %[alpha], v141\n\t" \
  "v_mul_f32 v142, %[alpha], v142\n\t" \
  "v_mul_f32 v143, %[alpha], v143\n\t" \
  "v_mul_f32 v144, %[alpha], v144\n\t" \
  "v_mul_f32 v145, %[alpha], v145\n\t" \
  "v_mul_f32 v146, %[alpha], v146\n\t" \
  "v_mul_f32 v147, %[alpha], v147\n\t" \
  "v_mul_f32 v148, %[alpha], v148\n\t" \
  "v_mul_f32 v149, %[alpha], v149\n\t" \
  "v_mul_f32 v150, %[alpha], v150\n\t" \
  "v_mul_f32 v151, %[alpha], v151\n\t" \
  "v_mul_f32 v152, %[alpha], v152\n\t" \
  "v_mul_f32 v153, %[alpha], v153\n\t" \
  "v_mul_f32 v154, %[alpha], v154\n\t" \
  "v_mul_f32 v155, %[alpha], v155\n\t" \
  "v_mul_f32 v156, %[alpha], v156\n\t" \
  "v_mul_f32 v157, %[alpha], v157\n\t" \
  "v_mul_f32 v158, %[alpha], v158\n\t" \
  "v_mul_f32 v159, %[alpha], v159\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "v_accvgpr_read_b32 v192, a160\n\t" \
  "v_accvgpr_read_b32 v193, a161\n\t" \
  "v_accvgpr_read_b32 v194, a162\n\t" \
  "v_accvgpr_read_b32 v195, a163\n\t" \
  "v_accvgpr_read_b32 v196, a164\n\t" \
  "v_accvgpr_read_b32 v197, a165\n\t" \
  "v_accvgpr_read_b32 v198, a166\n\t" \
  "v_accvgpr_read_b32 v199, a167\n\t" \
  "v_accvgpr_read_b32 v200, a168\n\t" \
  "v_accvgpr_read_b32 v201, a169\n\t" \
  "v_accvgpr_read_b32 v202, a170\n\t" \
  "v_accvgpr_read_b32 v203, a171\n\t" \
  "v_accvgpr_read_b32 v204, a172\n\t" \
  "v_accvgpr_read_b32 v205, a173\n\t" \
  "v_accvgpr_read_b32 v206, a174\n\t" \
  "v_accvgpr_read_b32 v207, a175\n\t" \
  "v_accvgpr_read_b32 v208, a176\n\t" \
  "v_accvgpr_read_b32 v209, a177\n\t" \
  "v_accvgpr_read_b32 v210, a178\n\t" \
  "v_accvgpr_read_b32 v211, a179\n\t" \
  "v_accvgpr_read_b32 v212, a180\n\t" \
  "v_accvgpr_read_b32 v213, a181\n\t" \
  "v_accvgpr_read_b32 v214, a182\n\t" \
  "v_accvgpr_read_b32 v215, a183\n\t" \
  "v_accvgpr_read_b32 v216, a184\n\t" \
  "v_accvgpr_read_b32 v217, a185\n\t" \
  "v_accvgpr_read_b32 v218, a186\n\t" \
  "v_accvgpr_read_b32 v219, a187\n\t" \
  "v_accvgpr_read_b32 v220, a188\n\t" \
  "v_accvgpr_read_b32 v221, a189\n\t" \
  "v_accvgpr_read_b32 v222, a190\n\t" \
  "v_accvgpr_read_b32 v223, a191\n\t" \
  "v_mul_f32 v192, %[alpha], v192\n\t" \
  "v_mul_f32 v193, %[alpha], v193\n\t" \
  "v_mul_f32 v194, %[alpha], v194\n\t" \
  "v_mul_f32 v195, %[alpha], v195\n\t" \
  "v_mul_f32 v196, %[alpha], v196\n\t" \
  "v_mul_f32 v197, %[alpha], v197\n\t" \
  "v_mul_f32 v198, %[alpha], v198\n\t" \
  "v_mul_f32 v199, %[alpha], v199\n\t" \
  "v_mul_f32 v200, %[alpha], v200\n\t" \
  "v_mul_f32 v201, %[alpha], v201\n\t" \
  "v_mul_f32 v202, %[alpha], v202\n\t" \
  "v_mul_f32 v203, %[alpha], v203\n\t" \
  "v_mul_f32 v204, %[alpha], v204\n\t" \
  "v_mul_f32 v205, %[alpha], v205\n\t" \
  "v_mul_f32 v206, %[alpha], v206\n\t" \
  "v_mul_f32 v207, %[alpha], v207\n\t" \
  "v_mul_f32 v208, %[alpha], v208\n\t" \
  "v_mul_f32 v209, %[alpha], v209\n\t" \
  "v_mul_f32 v210, %[alpha], v210\n\t" \
  "v_mul_f32 v211, %[alpha], v211\n\t" \
  "v_mul_f32 v212, %[alpha], v212\n\t" \
  "v_mul_f32 v213, %[alpha], v213\n\t" \
  "v_mul_f32 v214, %[alpha], v214\n\t" \
  "v_mul_f32 v215, %[alpha], v215\n\t" \
  "v_mul_f32 v216, %[alpha], v216\n\t" \
  "v_mul_f32 v217, %[alpha], v217\n\t" \
  "v_mul_f32 v218, %[alpha], v218\n\t" \
  "v_mul_f32 v219, %[alpha], v219\n\t" \
  "v_mul_f32 v220, %[alpha], v220\n\t" \
  "v_mul_f32 v221, %[alpha], v221\n\t" \
  "v_mul_f32 v222, %[alpha], v222\n\t" \
  "v_mul_f32 v223, %[alpha], v223\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a192\n\t" \
  "v_accvgpr_read_b32 v129, a193\n\t" \
  "v_accvgpr_read_b32 v130, a194\n\t" \
  "v_accvgpr_read_b32 v131, a195\n\t" \
  "v_accvgpr_read_b32 v132, a196\n\t" \
  "v_accvgpr_read_b32 v133, a197\n\t" \
  "v_accvgpr_read_b32 v134, a198\n\t" \
  "v_accvgpr_read_b32 v135, a199\n\t" \
  "v_accvgpr_read_b32 v136, a200\n\t" \
  "v_accvgpr_read_b32 v137, a201\n\t" \
  "v_accvgpr_read_b32 v138, a202\n\t" \
  "v_accvgpr_read_b32 v139, a203\n\t" \
  "v_accvgpr_read_b32 v140, a204\n\t" \
  "v_accvgpr_read_b32 v141, a205\n\t" \
  "v_accvgpr_read_b32 v142, a206\n\t" \
  "v_accvgpr_read_b32 v143, a207\n\t" \
  "v_accvgpr_read_b32 v144, a208\n\t" \
  "v_accvgpr_read_b32 v145, a209\n\t" \
  "v_accvgpr_read_b32 v146, a210\n\t" \
  "v_accvgpr_read_b32 v147, a211\n\t" \
  "v_accvgpr_read_b32 v148, a212\n\t" \
  "v_accvgpr_read_b32 v149, a213\n\t" \
  "v_accvgpr_read_b32 v150, a214\n\t" \
  "v_accvgpr_read_b32 v151, a215\n\t" \
  "v_accvgpr_read_b32 v152, a216\n\t" \
  "v_accvgpr_read_b32 v153, a217\n\t" \
  "v_accvgpr_read_b32 v154, a218\n\t" \
  "v_accvgpr_read_b32 v155, a219\n\t" \
  "v_accvgpr_read_b32 v156, a220\n\t" \
  "v_accvgpr_read_b32 v157, a221\n\t" \
  "v_accvgpr_read_b32 v158, a222\n\t" \
  "v_accvgpr_read_b32 v159, a223\n\t" \
  "v_mul_f32 v128, %[alpha], v128\n\t" \
  "v_mul_f32 v129, %[alpha], v129\n\t" \
  "v_mul_f32 v130, %[alpha], v130\n\t" \
  "v_mul_f32 v131, %[alpha], v131\n\t" \
  "v_mul_f32 v132, %[alpha], v132\n\t" \
  "v_mul_f32 v133, %[alpha], v133\n\t" \
  "v_mul_f32 v134, %[alpha], v134\n\t" \
  "v_mul_f32 v135, %[alpha], v135\n\t" \
  "v_mul_f32 v136, %[alpha], v136\n\t" \
  "v_mul_f32 v137, %[alpha], v137\n\t" \
  "v_mul_f32 v138, %[alpha], v138\n\t" \
  "v_mul_f32 v139, %[alpha], v139\n\t" \
  "v_mul_f32 v140, %[alpha], v140\n\t" \
  "v_mul_f32 v141, %[alpha], v141\n\t" \
  "v_mul_f32 v142, %[alpha], v142\n\t" \
  "v_mul_f32 v143, %[alpha], v143\n\t" \
  "v_mul_f32 v144, %[alpha], v144\n\t" \
  "v_mul_f32 v145, %[alpha], v145\n\t" \
  "v_mul_f32 v146, %[alpha], v146\n\t" \
  "v_mul_f32 v147, %[alpha], v147\n\t" \
  "v_mul_f32 v148, %[alpha], v148\n\t" \
  "v_mul_f32 v149, %[alpha], v149\n\t" \
  "v_mul_f32 v150, %[alpha], v150\n\t" \
  "v_mul_f32 v151, %[alpha], v151\n\t" \
  "v_mul_f32 v152, %[alpha], v152\n\t" \
  "v_mul_f32 v153, %[alpha], v153\n\t" \
  "v_mul_f32 v154, %[alpha], v154\n\t" \
  "v_mul_f32 v155, %[alpha], v155\n\t" \
  "v_mul_f32 v156, %[alpha], v156\n\t" \
  "v_mul_f32 v157, %[alpha], v157\n\t" \
  "v_mul_f32 v158, %[alpha], v158\n\t" \
  "v_mul_f32 v159, %[alpha], v159\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a224\n\t" \
  "v_accvgpr_read_b32 v193, a225\n\t" \
  "v_accvgpr_read_b32 v194, a226\n\t" \
  "v_accvgpr_read_b32 v195, a227\n\t" \
  "v_accvgpr_read_b32 v196, a228\n\t" \
  "v_accvgpr_read_b32 v197, a229\n\t" \
  "v_accvgpr_read_b32 v198, a230\n\t" \
  "v_accvgpr_read_b32 v199, a231\n\t" \
  "v_accvgpr_read_b32 v200, a232\n\t" \
  "v_accvgpr_read_b32 v201, a233\n\t" \
  "v_accvgpr_read_b32 v202, a234\n\t" \
  "v_accvgpr_read_b32 v203, a235\n\t" \
  "v_accvgpr_read_b32 v204, a236\n\t" \
  "v_accvgpr_read_b32 v205, a237\n\t" \
  "v_accvgpr_read_b32 v206, a238\n\t" \
  "v_accvgpr_read_b32 v207, a239\n\t" \
  "v_accvgpr_read_b32 v208, a240\n\t" \
  "v_accvgpr_read_b32 v209, a241\n\t" \
  "v_accvgpr_read_b32 v210, a242\n\t" \
  "v_accvgpr_read_b32 v211, a243\n\t" \
  "v_accvgpr_read_b32 v212, a244\n\t" \
  "v_accvgpr_read_b32 v213, a245\n\t" \
  "v_accvgpr_read_b32 v214, a246\n\t" \
  "v_accvgpr_read_b32 v215, a247\n\t" \
  "v_accvgpr_read_b32 v216, a248\n\t" \
  "v_accvgpr_read_b32 v217, a249\n\t" \
  "v_accvgpr_read_b32 v218, a250\n\t" \
  "v_accvgpr_read_b32 v219, a251\n\t" \
  "v_accvgpr_read_b32 v220, a252\n\t" \
  "v_accvgpr_read_b32 v221, a253\n\t" \
  "v_accvgpr_read_b32 v222, a254\n\t" \
  "v_accvgpr_read_b32 v223, a255\n\t" \
  "v_mul_f32 v192, %[alpha], v192\n\t" \
  "v_mul_f32 v193, %[alpha], v193\n\t" \
  "v_mul_f32 v194, %[alpha], v194\n\t" \
  "v_mul_f32 v195, %[alpha], v195\n\t" \
  "v_mul_f32 v196, %[alpha], v196\n\t" \
  "v_mul_f32 v197, %[alpha], v197\n\t" \
  "v_mul_f32 v198, %[alpha], v198\n\t" \
  "v_mul_f32 v199, %[alpha], v199\n\t" \
  "v_mul_f32 v200, %[alpha], v200\n\t" \
  "v_mul_f32 v201, %[alpha], v201\n\t" \
  "v_mul_f32 v202, %[alpha], v202\n\t" \
  "v_mul_f32 v203, %[alpha], v203\n\t" \
  "v_mul_f32 v204, %[alpha], v204\n\t" \
  "v_mul_f32 v205, %[alpha], v205\n\t" \
  "v_mul_f32 v206, %[alpha], v206\n\t" \
  "v_mul_f32 v207, %[alpha], v207\n\t" \
  "v_mul_f32 v208, %[alpha], v208\n\t" \
  "v_mul_f32 v209, %[alpha], v209\n\t" \
  "v_mul_f32 v210, %[alpha], v210\n\t" \
  "v_mul_f32 v211, %[alpha], v211\n\t" \
  "v_mul_f32 v212, %[alpha], v212\n\t" \
  "v_mul_f32 v213, %[alpha], v213\n\t" \
  "v_mul_f32 v214, %[alpha], v214\n\t" \
  "v_mul_f32 v215, %[alpha], v215\n\t" \
  "v_mul_f32 v216, %[alpha], v216\n\t" \
  "v_mul_f32 v217, %[alpha], v217\n\t" \
  "v_mul_f32 v218, %[alpha], v218\n\t" \
  "v_mul_f32 v219, %[alpha], v219\n\t" \
  "v_mul_f32 v220, %[alpha], v220\n\t" \
  "v_mul_f32 v221, %[alpha], v221\n\t" \
  "v_mul_f32 v222, %[alpha], v222\n\t" \
  "v_mul_f32 v223, %[alpha], v223\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  ""
#define SK_TILE_ASM_STORE_HALF1_NT(CVT) \
  "s_mul_i32 s83, %[rowstep], 4\n\t" \
  "s_add_u32 s84, s83, %[q1]\n\t" \
  "s_add_u32 s85, s84, %[q1]\n\t" \
  "s_add_u32 s87, s85, %[q1]\n\t" \
  "v_accvgpr_read_b32 v128, a128\n\t" \
  "v_accvgpr_read_b32 v129, a129\n\t" \
  "v_accvgpr_read_b32 v130, a130\n\t" \
  "v_accvgpr_read_b32 v131, a131\n\t" \
  "v_accvgpr_read_b32 v132, a132\n\t" \
  "v_accvgpr_read_b32 v133, a133\n\t" \
  "v_accvgpr_read_b32 v134, a134\n\t" \
  "v_accvgpr_read_b32 v135, a135\n\t" \
  "v_accvgpr_read_b32 v136, a136\n\t" \
  "v_accvgpr_read_b32 v137, a137\n\t" \
  "v_accvgpr_read_b32 v138, a138\n\t" \
  "v_accvgpr_read_b32 v139, a139\n\t" \
  "v_accvgpr_read_b32 v140, a140\n\t" \
  "v_accvgpr_read_b32 v141, a141\n\t" \
  "v_accvgpr_read_b32 v142, a142\n\t" \
  "v_accvgpr_read_b32 v143, a143\n\t" \
  "v_accvgpr_read_b32 v144, a144\n\t" \
  "v_accvgpr_read_b32 v145, a145\n\t" \
  "v_accvgpr_read_b32 v146, a146\n\t" \
  "v_accvgpr_read_b32 v147, a147\n\t" \
  "v_accvgpr_read_b32 v148, a148\n\t" \
  "v_accvgpr_read_b32 v149, a149\n\t" \
  "v_accvgpr_read_b32 v150, a150\n\t" \
  "v_accvgpr_read_b32 v151, a151\n\t" \
  "v_accvgpr_read_b32 v152, a152\n\t" \
  "v_accvgpr_read_b32 v153, a153\n\t" \
  "v_accvgpr_read_b32 v154, a154\n\t" \
  "v_accvgpr_read_b32 v155, a155\n\t" \
  "v_accvgpr_read_b32 v156, a156\n\t" \
  "v_accvgpr_read_b32 v157, a157\n\t" \
  "v_accvgpr_read_b32 v158, a158\n\t" \
  "v_accvgpr_read_b32 v159, a159\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "v_accvgpr_read_b32 v192, a160\n\t" \
  "v_accvgpr_read_b32 v193, a161\n\t" \
  "v_accvgpr_read_b32 v194, a162\n\t" \
  "v_accvgpr_read_b32 v195, a163\n\t" \
  "v_accvgpr_read_b32 v196, a164\n\t" \
  "v_accvgpr_read_b32 v197, a165\n\t" \
  "v_accvgpr_read_b32 v198, a166\n\t" \
  "v_accvgpr_read_b32 v199, a167\n\t" \
  "v_accvgpr_read_b32 v200, a168\n\t" \
  "v_accvgpr_read_b32 v201, a169\n\t" \
  "v_accvgpr_read_b32 v202, a170\n\t" \
  "v_accvgpr_read_b32 v203, a171\n\t" \
  "v_accvgpr_read_b32 v204, a172\n\t" \
  "v_accvgpr_read_b32 v205, a173\n\t" \
  "v_accvgpr_read_b32 v206, a174\n\t" \
  "v_accvgpr_read_b32 v207, a175\n\t" \
  "v_accvgpr_read_b32 v208, a176\n\t" \
  "v_accvgpr_read_b32 v209, a177\n\t" \
  "v_accvgpr_read_b32 v210, a178\n\t" \
  "v_accvgpr_read_b32 v211, a179\n\t" \
  "v_accvgpr_read_b32 v212, a180\n\t" \
  "v_accvgpr_read_b32 v213, a181\n\t" \
  "v_accvgpr_read_b32 v214, a182\n\t" \
  "v_accvgpr_read_b32 v215, a183\n\t" \
  "v_accvgpr_read_b32 v216, a184\n\t" \
  "v_accvgpr_read_b32 v217, a185\n\t" \
  "v_accvgpr_read_b32 v218, a186\n\t" \
  "v_accvgpr_read_b32 v219, a187\n\t" \
  "v_accvgpr_read_b32 v220, a188\n\t" \
  "v_accvgpr_read_b32 v221, a189\n\t" \
  "v_accvgpr_read_b32 v222, a190\n\t" \
  "v_accvgpr_read_b32 v223, a191\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v128, a192\n\t" \
  "v_accvgpr_read_b32 v129, a193\n\t" \
  "v_accvgpr_read_b32 v130, a194\n\t" \
  "v_accvgpr_read_b32 v131, a195\n\t" \
  "v_accvgpr_read_b32 v132, a196\n\t" \
  "v_accvgpr_read_b32 v133, a197\n\t" \
  "v_accvgpr_read_b32 v134, a198\n\t" \
  "v_accvgpr_read_b32 v135, a199\n\t" \
  "v_accvgpr_read_b32 v136, a200\n\t" \
  "v_accvgpr_read_b32 v137, a201\n\t" \
  "v_accvgpr_read_b32 v138, a202\n\t" \
  "v_accvgpr_read_b32 v139, a203\n\t" \
  "v_accvgpr_read_b32 v140, a204\n\t" \
  "v_accvgpr_read_b32 v141, a205\n\t" \
  "v_accvgpr_read_b32 v142, a206\n\t" \
  "v_accvgpr_read_b32 v143, a207\n\t" \
  "v_accvgpr_read_b32 v144, a208\n\t" \
  "v_accvgpr_read_b32 v145, a209\n\t" \
  "v_accvgpr_read_b32 v146, a210\n\t" \
  "v_accvgpr_read_b32 v147, a211\n\t" \
  "v_accvgpr_read_b32 v148, a212\n\t" \
  "v_accvgpr_read_b32 v149, a213\n\t" \
  "v_accvgpr_read_b32 v150, a214\n\t" \
  "v_accvgpr_read_b32 v151, a215\n\t" \
  "v_accvgpr_read_b32 v152, a216\n\t" \
  "v_accvgpr_read_b32 v153, a217\n\t" \
  "v_accvgpr_read_b32 v154, a218\n\t" \
  "v_accvgpr_read_b32 v155, a219\n\t" \
  "v_accvgpr_read_b32 v156, a220\n\t" \
  "v_accvgpr_read_b32 v157, a221\n\t" \
  "v_accvgpr_read_b32 v158, a222\n\t" \
  "v_accvgpr_read_b32 v159, a223\n\t" \
  CVT " v160, v128, v129\n\t" \
  CVT " v161, v130, v131\n\t" \
  CVT " v162, v132, v133\n\t" \
  CVT " v163, v134, v135\n\t" \
  CVT " v164, v136, v137\n\t" \
  CVT " v165, v138, v139\n\t" \
  CVT " v166, v140, v141\n\t" \
  CVT " v167, v142, v143\n\t" \
  CVT " v168, v144, v145\n\t" \
  CVT " v169, v146, v147\n\t" \
  CVT " v170, v148, v149\n\t" \
  CVT " v171, v150, v151\n\t" \
  CVT " v172, v152, v153\n\t" \
  CVT " v173, v154, v155\n\t" \
  CVT " v174, v156, v157\n\t" \
  CVT " v175, v158, v159\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[160:161] offset:0\n\t" \
  "ds_write_b64 %[wr], v[162:163] offset:32\n\t" \
  "ds_write_b64 %[wr], v[164:165] offset:64\n\t" \
  "ds_write_b64 %[wr], v[166:167] offset:96\n\t" \
  "ds_write_b64 %[wr], v[168:169] offset:128\n\t" \
  "ds_write_b64 %[wr], v[170:171] offset:160\n\t" \
  "ds_write_b64 %[wr], v[172:173] offset:192\n\t" \
  "ds_write_b64 %[wr], v[174:175] offset:224\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "v_accvgpr_read_b32 v192, a224\n\t" \
  "v_accvgpr_read_b32 v193, a225\n\t" \
  "v_accvgpr_read_b32 v194, a226\n\t" \
  "v_accvgpr_read_b32 v195, a227\n\t" \
  "v_accvgpr_read_b32 v196, a228\n\t" \
  "v_accvgpr_read_b32 v197, a229\n\t" \
  "v_accvgpr_read_b32 v198, a230\n\t" \
  "v_accvgpr_read_b32 v199, a231\n\t" \
  "v_accvgpr_read_b32 v200, a232\n\t" \
  "v_accvgpr_read_b32 v201, a233\n\t" \
  "v_accvgpr_read_b32 v202, a234\n\t" \
  "v_accvgpr_read_b32 v203, a235\n\t" \
  "v_accvgpr_read_b32 v204, a236\n\t" \
  "v_accvgpr_read_b32 v205, a237\n\t" \
  "v_accvgpr_read_b32 v206, a238\n\t" \
  "v_accvgpr_read_b32 v207, a239\n\t" \
  "v_accvgpr_read_b32 v208, a240\n\t" \
  "v_accvgpr_read_b32 v209, a241\n\t" \
  "v_accvgpr_read_b32 v210, a242\n\t" \
  "v_accvgpr_read_b32 v211, a243\n\t" \
  "v_accvgpr_read_b32 v212, a244\n\t" \
  "v_accvgpr_read_b32 v213, a245\n\t" \
  "v_accvgpr_read_b32 v214, a246\n\t" \
  "v_accvgpr_read_b32 v215, a247\n\t" \
  "v_accvgpr_read_b32 v216, a248\n\t" \
  "v_accvgpr_read_b32 v217, a249\n\t" \
  "v_accvgpr_read_b32 v218, a250\n\t" \
  "v_accvgpr_read_b32 v219, a251\n\t" \
  "v_accvgpr_read_b32 v220, a252\n\t" \
  "v_accvgpr_read_b32 v221, a253\n\t" \
  "v_accvgpr_read_b32 v222, a254\n\t" \
  "v_accvgpr_read_b32 v223, a255\n\t" \
  CVT " v224, v192, v193\n\t" \
  CVT " v225, v194, v195\n\t" \
  CVT " v226, v196, v197\n\t" \
  CVT " v227, v198, v199\n\t" \
  CVT " v228, v200, v201\n\t" \
  CVT " v229, v202, v203\n\t" \
  CVT " v230, v204, v205\n\t" \
  CVT " v231, v206, v207\n\t" \
  CVT " v232, v208, v209\n\t" \
  CVT " v233, v210, v211\n\t" \
  CVT " v234, v212, v213\n\t" \
  CVT " v235, v214, v215\n\t" \
  CVT " v236, v216, v217\n\t" \
  CVT " v237, v218, v219\n\t" \
  CVT " v238, v220, v221\n\t" \
  CVT " v239, v222, v223\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[176:179], %[rd] offset:0\n\t" \
  "ds_read_b128 v[180:183], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[184:187], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[188:191], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_write_b64 %[wr], v[224:225] offset:0\n\t" \
  "ds_write_b64 %[wr], v[226:227] offset:32\n\t" \
  "ds_write_b64 %[wr], v[228:229] offset:64\n\t" \
  "ds_write_b64 %[wr], v[230:231] offset:96\n\t" \
  "ds_write_b64 %[wr], v[232:233] offset:128\n\t" \
  "ds_write_b64 %[wr], v[234:235] offset:160\n\t" \
  "ds_write_b64 %[wr], v[236:237] offset:192\n\t" \
  "ds_write_b64 %[wr], v[238:239] offset:224\n\t" \
  "buffer_store_dwordx4 v[176:179], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[180:183], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[184:187], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[188:191], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "ds_read_b128 v[240:243], %[rd] offset:0\n\t" \
  "ds_read_b128 v[244:247], %[rd] offset:1088\n\t" \
  "ds_read_b128 v[248:251], %[rd] offset:2176\n\t" \
  "ds_read_b128 v[252:255], %[rd] offset:3264\n\t" \
  "s_waitcnt lgkmcnt(0)\n\t" \
  "buffer_store_dwordx4 v[240:243], %[voff], %[rsc], s83 offen nt\n\t" \
  "buffer_store_dwordx4 v[244:247], %[voff], %[rsc], s84 offen nt\n\t" \
  "buffer_store_dwordx4 v[248:251], %[voff], %[rsc], s85 offen nt\n\t" \
  "buffer_store_dwordx4 v[252:255], %[voff], %[rsc], s87 offen nt\n\t" \
  "s_add_u32 s83, s83, %[rowstep]\n\t" \
  "s_add_u32 s84, s84, %[rowstep]\n\t" \
  "s_add_u32 s85, s85, %[rowstep]\n\t" \
  "s_add_u32 s87, s87, %[rowstep]\n\t" \
  ""
#define SK_TILE_ASM_CLOBBERS \
  "a0", "a1", "a2", "a3", "a4", "a5", "a6", "a7", "a8", "a9", "a10", "a11", "a12", "a13", "a14", "a15", \
  "a16", "a17", "a18", "a19", "a20", "a21", "a22", "a23", "a24", "a25", "a26", "a27", "a28", "a29", "a30", "a31", \
  "a32", "a33", "a34", "a35", "a36", "a37", "a38", "a39", "a40", "a41", "a42", "a43", "a44", "a45", "a46", "a47", \
  "a48", "a49", "a50", "a51", "a52", "a53", "a54", "a55", "a56", "a57", "a58", "a59", "a60", "a61", "a62", "a63", \
  "a64", "a65", "a66", "a67", "a68", "a69", "a70", "a71", "a72", "a73", "a74", "a75", "a76", "a77", "a78", "a79", \
  "a80", "a81", "a82", "a83", "a84", "a85", "a86", "a87", "a88", "a89", "a90", "a91", "a92", "a93", "a94", "a95", \
  "a96", "a97", "a98", "a99", "a100", "a101", "a102", "a103", "a104", "a105", "a106", "a107", "a108", "a109", "a110", "a111", \
  "a112", "a113", "a114", "a115", "a116", "a117", "a118", "a119", "a120", "a121", "a122", "a123", "a124", "a125", "a126", "a127", \
  "a128", "a129", "a130", "a131", "a132", "a133", "a134", "a135", "a136", "a137", "a138", "a139", "a140", "a141", "a142", "a143", \
  "a144", "a145", "a146", "a147", "a148", "a149", "a150", "a151", "a152", "a153", "a154", "a155", "a156", "a157", "a158", "a159", \
  "a160", "a161", "a162", "a163", "a164", "a165", "a166", "a167", "a168", "a169", "a170", "a171", "a172", "a173", "a174", "a175", \
  "a176", "a177", "a178", "a179", "a180", "a181", "a182", "a183", "a184", "a185", "a186", "a187", "a188", "a189", "a190", "a191", \
  "a192", "a193", "a194", "a195", "a196", "a197", "a198", "a199", "a200", "a201", "a202", "a203", "a204", "a205", "a206", "a207", \
  "a208", "a209", "a210", "a211", "a212", "a213", "a214", "a215", "a216", "a217", "a218", "a219", "a220", "a221", "a222", "a223", \
  "a224", "a225", "a226", "a227", "a228", "a229", "a230", "a231", "a232", "a233", "a234", "a235", "a236", "a237", "a238", "a239", \
  "a240", "a241", "a242", "a243", "a244", "a245", "a246", "a247", "a248", "a249", "a250", "a251", "a252", "a253", "a254", "a255", \
  "v120", "v121", "v122", "v123", "v124", "v125", "v126", "v127", "v128", "v129", "v130", "v131", "v132", "v133", "v134", "v135", \
  "v136", "v137", "v138", "v139", "v140", "v141", "v142", "v143", "v144", "v145", "v146", "v147", "v148", "v149", "v150", "v151", \
  "v152", "v153", "v154", "v155", "v156", "v157", "v158", "v159", "v160", "v161", "v162", "v163", "v164", "v165", "v166", "v167", \
  "v168", "v169", "v170", "v171", "v172", "v173", "v174", "v175", "v176", "v177", "v178", "v179", "v180", "v181", "v182", "v183", \
  "v184", "v185", "v186", "v187", "v188", "v189", "v190", "v191", "v192", "v193", "v194", "v195", "v196", "v197", "v198", "v199", \
  "v200", "v201", "v202", "v203", "v204", "v205", "v206", "v207", "v208", "v209", "v210", "v211", "v212", "v213", "v214", "v215", \
  "v216", "v217", "v218", "v219", "v220", "v221", "v222", "v223", "v224", "v225", "v226", "v227", "v228", "v229", "v230", "v231", \
  "v232", "v233", "v234", "v235", "v236", "v237", "v238", "v239", "v240", "v241", "v242", "v243", "v244", "v245", "v246", "v247", \
  "v248", "v249", "v250", "v251", "v252", "v253", "v254", "v255", "s80", "s81", "s82", "s83", "s84", "s85", "s86", "s87"
