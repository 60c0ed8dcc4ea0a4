! paged_checks.f90 -- the paged cache (fg_paged_* of include/fgpt.h) from
! Fortran; test code, built by build() next to this file.
!
!   refusals   every entry refuses a null handle (needs no device).
!   greedy     two sequences in one cache: the prompt IDS_FILE, and a fork of
!              it at half its length; then NGEN steps over both at once, each
!              step's ids the next one's input, the even steps' by argmax,
!              the odd ones' by a draw at temperature 0. OUT_FILE gets a line
!              of NGEN ids a sequence.
!
! Usage:
!   paged_checks refusals
!   paged_checks greedy WDIR L D H KH HD V IDS_FILE NGEN OUT_FILE
program paged_checks
  use, intrinsic :: iso_c_binding
  use, intrinsic :: iso_fortran_env, only: error_unit
  use fgpt_c
  use fgpt_util
  implicit none

  character(len=512) :: mode

  if (command_argument_count() < 1) call usage()
  call get_command_argument(1, mode)
  select case (trim(mode))
  case ('refusals')
    call run_refusals()
  case ('greedy')
    call run_greedy()
  case default
    call usage()
  end select

contains

  subroutine usage()
    write (error_unit, '(A)') 'usage: paged_checks refusals'
    write (error_unit, '(A)') '       paged_checks greedy WDIR L D H KH HD V IDS NGEN OUT'
    stop 2
  end subroutine usage

  subroutine expect(what, rc, want)
    character(*), intent(in) :: what
    integer(c_int32_t), intent(in) :: rc, want
    if (rc /= want) then
      write (error_unit, '(A,A,I0,A,I0)') what, ': ', rc, ', expected ', want
      stop 1
    end if
  end subroutine expect

  subroutine ok(what, rc)
    character(*), intent(in) :: what
    integer(c_int32_t), intent(in) :: rc
    if (rc /= FG_OK) call stop_rc(what, rc)
  end subroutine ok

  subroutine run_refusals()
    type(c_ptr) :: nul, pc
    integer(c_int32_t) :: n, one(1)
    nul = c_null_ptr
    one = 1
    call expect('create', fg_paged_create(nul, 4, 16, 1, 0, 0, 0, pc), FG_EARG)
    call expect('len', fg_paged_len(nul, 0, n), FG_EARG)
    call expect('free', fg_paged_free(nul, n), FG_EARG)
    call expect('fork', fg_paged_fork(nul, 0, 1, 1), FG_EARG)
    call expect('trim', fg_paged_trim(nul, 0, 0), FG_EARG)
    call expect('compact', fg_paged_compact(nul, n), FG_EARG)
    call expect('read', fg_paged_read(nul, 0, nul, nul), FG_EARG)
    call expect('step', fg_paged_step(nul, nul, 1, one, one, one, nul, nul, nul), FG_EARG)
    write (*, '(A)') 'refusals: ok'
  end subroutine run_refusals

  subroutine run_greedy()
    character(len=512) :: wdir, ids_file, out_file
    type(fg_dims) :: dims
    type(fg_draw_cfg), target :: draw
    type(c_ptr) :: m, pc, settings
    integer :: n, ngen, half, i, u
    integer(c_int), allocatable :: ids(:), out(:, :)
    integer(c_int32_t) :: length, free0, free1, moved
    integer(c_int32_t), target :: next(2)
    real(c_float), target :: temp(2), unif(2)
    real(c_float), allocatable :: cos_b(:), sin_b(:)

    if (command_argument_count() < 11) call usage()
    wdir = sarg(2)
    dims = fg_dims(iarg(3), iarg(4), iarg(5), iarg(6), iarg(7), iarg(8), 1.0e-5_c_float)
    ids_file = sarg(9); ngen = iarg(10); out_file = sarg(11)
    call read_ids(trim(ids_file), ids, n)
    half = n/2
    allocate (out(ngen, 2))
    call ok('load', fg_model_load(dims, trim(wdir)//c_null_char, m))
    call rope_tables(n + ngen, dims%head_dim, cos_b, sin_b)
    call ok('rope', fg_set_rope(m, 0, n + ngen, cos_b, sin_b))
    call ok('create', fg_paged_create(m, 4*(n + ngen)/16 + 4, 16, 4, 0, 0, 0, pc))
    call ok('free', fg_paged_free(pc, free0))

    ! the prompt, its fork, and the id after each
    call ok('prompt', fg_paged_step(m, pc, 1, [0], [n], ids, c_null_ptr, c_null_ptr, c_loc(next)))
    out(1, 1) = next(1)
    if (half > 1) call ok('fork', fg_paged_fork(pc, 0, 2, half - 1))
    call ok('forked', fg_paged_step(m, pc, 1, [2], [1], ids(half:half), c_null_ptr, c_null_ptr, &
        c_loc(next)))
    out(1, 2) = next(1)
    temp = 0.0_c_float
    unif = 0.5_c_float
    draw%temp = c_loc(temp)
    draw%u = c_loc(unif)
    do i = 2, ngen
      settings = c_null_ptr
      if (mod(i, 2) == 1) settings = c_loc(draw)
      call ok('step', fg_paged_step(m, pc, 2, [2, 0], [1, 1], [out(i - 1, 2), out(i - 1, 1)], &
          settings, c_null_ptr, c_loc(next)))
      out(i, 2) = next(1)
      out(i, 1) = next(2)
    end do

    call ok('len', fg_paged_len(pc, 2, length))
    call expect('length', length, int(half + ngen - 1, c_int32_t))
    call ok('trim', fg_paged_trim(pc, 0, 0))
    call ok('compact', fg_paged_compact(pc, moved))
    call ok('trim', fg_paged_trim(pc, 2, 0))
    call ok('free', fg_paged_free(pc, free1))
    call expect('pages free', free1, free0)
    call ok('destroy', fg_paged_destroy(pc))
    call ok('destroy', fg_model_destroy(m))
    open (newunit=u, file=trim(out_file), status='replace', action='write')
    do i = 1, 2
      write (u, '(*(I0,1X))') out(:, i)
    end do
    close (u)
  end subroutine run_greedy
end program paged_checks
